// Attention over the 8-bit cache, row by row (single tokens of many sequences).
//
// With keys k = s_K a and values v = s_V b of whole numbers a, b and a scale per block of 16 tokens, for every query head
//     t_j = (s_K scale log2 e) q . a_j + log2 s_V        w_j = 2^(t_j - M)        out = sum_j w_j b_j / sum_j (w_j / s_V)
// The value's scale rides in the exponent, so one running maximum M bounds the weights by 1 whatever the scales are, f16 holds them with 11 bits,
// and no product needs a scale of its own. Queries are f16 with a power of two in front (kv8_cache.cuh), sums and maxima f32.
//
// A warp takes a block at a time. Keys are the rows of the matrix product, heads its columns (eight query heads of a kv head at most): S^T = K Q^T
// and O^T = V^T P^T, so that little of a matrix instruction is padding. The cache's byte order makes 16 bytes of a lane two k-steps of keys, or two
// row tiles of values. The 8 x 8 transposition between the two products is one instruction per eight tokens.
// Grid: (splits of the keys, kv head x eights of its query heads, row); four warps deal a split's blocks among them and merge through shared memory;
// several splits of a row go through scratch and a second kernel.
#include <algorithm>

#include "kv8_attention.cuh"

namespace gptrs {
namespace {

constexpr int kWarps = 4;
constexpr int kCols = 8;    // query heads of a CTA

// A row's blocks in parts of equal size, at most chunk_blocks each.
__device__ __forceinline__ void parts_of(const Kv8Attention& p, const Kv8Span& s, int* first, int* blocks, int* parts, int* per) {
    *first = s.begin / kKv8Tokens;
    *blocks = s.end > s.begin ? (s.end - 1) / kKv8Tokens + 1 - *first : 0;
    *parts = (*blocks + p.chunk_blocks - 1) / p.chunk_blocks;
    *per = *parts > 0 ? (*blocks + *parts - 1) / *parts : 1;
    *parts = (*blocks + *per - 1) / *per;
}

template <int kDim>
__global__ void __launch_bounds__(kWarps * 32) kv8_attention_kernel(const Kv8Attention p) {
    constexpr int kC = kDim / 32;      // chunks of 32 channels
    __shared__ float o_part[kWarps][kCols][kDim + 1];
    __shared__ float ml_part[kWarps][kCols][2];

    pdl_launch_dependents();
    pdl_wait();
    const int split = blockIdx.x, eights = (p.group + kCols - 1) / kCols;
    const int kv_head = blockIdx.y / eights, head0 = kv_head * p.group + (blockIdx.y % eights) * kCols;
    const int cols = min(kCols, p.group - (int)(blockIdx.y % eights) * kCols);
    const int row = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const Kv8Span span = kv8_span(p, row);
    if (span.slot < 0) return;
    int first, blocks, parts, per;
    parts_of(p, span, &first, &blocks, &parts, &per);
    if (split >= parts && !(split == 0 && parts == 0)) return;
    const int b_end = first + min((split + 1) * per, blocks);

    // ---- queries: column g of B, channels 32 c + 8 t + 4 s .. + 3 -------------------------------------------------------------------------
    uint32_t qf[kC][2][2];
    float q_scale;
    {
        uint32_t raw[kC][2][2], big = 0;
        const __nv_bfloat16* src = p.q + row * p.ldq + (long long)(head0 + min(g, cols - 1)) * kDim;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            const uint4 v = *reinterpret_cast<const uint4*>(src + 32 * c + 8 * t);
            raw[c][0][0] = v.x; raw[c][0][1] = v.y; raw[c][1][0] = v.z; raw[c][1][1] = v.w;
            big = __vmaxu2(big, __vmaxu2(abs_bits_max2(v.x, v.y), abs_bits_max2(v.z, v.w)));
        }
        uint32_t top = widest_half(big);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = pow2_exponent(top);
        const float factor = e == 128 ? 0.f : pow2(-e);
        q_scale = e == 128 ? __uint_as_float(0x7fc00000u) : pow2(e) * p.scale_log2;
#pragma unroll
        for (int c = 0; c < kC; ++c)
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) qf[c][s][i] = bf16x2_to_f16x2(raw[c][s][i], factor);
    }
    // the lane's two columns of S^T: heads 2 t, 2 t + 1
    const float qs0 = __shfl_sync(0xffffffffu, q_scale, 8 * t), qs1 = __shfl_sync(0xffffffffu, q_scale, 8 * t + 4);

    float o[2 * kC][4];
#pragma unroll
    for (int i = 0; i < 2 * kC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    for (int b = first + split * per + warp; b < b_end; b += kWarps) {
        uint32_t kf[kC][2][4], vf[2 * kC][4];
        float k_scale, v_scale;
        if ((b + 1) * kKv8Tokens <= span.length) {
            const int page = kv8_page(p.table, span.slot, p.max_pages, b, p.n_pages, p.status);
            if (page < 0) { atomicExch(p.status, 2); continue; }
            const unsigned char* src = p.pool + ((long long)page * p.kv_heads + kv_head) * kv8_block_bytes(kDim);
            const float2 scale = __ldg(reinterpret_cast<const float2*>(src + 32 * kDim));
            k_scale = scale.x; v_scale = scale.y;
            uint4 kb[kC], vb[kC];
#pragma unroll
            for (int c = 0; c < kC; ++c) kb[c] = ldg_stream_16(src + c * 512 + lane * 16);
#pragma unroll
            for (int c = 0; c < kC; ++c) vb[c] = ldg_stream_16(src + 16 * kDim + c * 512 + lane * 16);
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                kv8_widen(kb[c].x, &kf[c][0][0], &kf[c][0][2]);
                kv8_widen(kb[c].y, &kf[c][1][0], &kf[c][1][2]);
                kv8_widen(kb[c].z, &kf[c][0][1], &kf[c][0][3]);
                kv8_widen(kb[c].w, &kf[c][1][1], &kf[c][1][3]);
                kv8_widen(vb[c].x, &vf[2 * c][0], &vf[2 * c][2]);
                kv8_widen(vb[c].y, &vf[2 * c][1], &vf[2 * c][3]);
                kv8_widen(vb[c].z, &vf[2 * c + 1][0], &vf[2 * c + 1][2]);
                kv8_widen(vb[c].w, &vf[2 * c + 1][1], &vf[2 * c + 1][3]);
            }
        } else {
            // the block that is not complete: bf16 rows; what lies behind the last token may be anything and counts as zero
            const int have = span.length - b * kKv8Tokens;
            const __nv_bfloat16* ks = p.open + (long long)span.slot * kv8_open_elems(p.kv_heads, kDim) + kv8_open_at(b, p.kv_heads, kv_head, 0, kDim);
            const __nv_bfloat16* vs = ks + kKv8Tokens * kDim;
            uint4 kr[kC][2];
            uint32_t big = 0;
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    kr[c][r] = g + 8 * r < have ? *reinterpret_cast<const uint4*>(ks + (g + 8 * r) * kDim + 32 * c + 8 * t) : make_uint4(0, 0, 0, 0);
                    big = __vmaxu2(big, __vmaxu2(abs_bits_max2(kr[c][r].x, kr[c][r].y), abs_bits_max2(kr[c][r].z, kr[c][r].w)));
                }
            int e = pow2_exponent(__reduce_max_sync(0xffffffffu, widest_half(big)));
            float factor = e == 128 ? 0.f : pow2(-e);
            k_scale = e == 128 ? __uint_as_float(0x7fc00000u) : pow2(e);
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    kf[c][0][r] = bf16x2_to_f16x2(kr[c][r].x, factor);
                    kf[c][0][2 + r] = bf16x2_to_f16x2(kr[c][r].y, factor);
                    kf[c][1][r] = bf16x2_to_f16x2(kr[c][r].z, factor);
                    kf[c][1][2 + r] = bf16x2_to_f16x2(kr[c][r].w, factor);
                }
            big = 0;
            const unsigned short* vbits = reinterpret_cast<const unsigned short*>(vs);
#pragma unroll
            for (int i = 0; i < 2 * kC; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int d = 16 * i + 8 * (j & 1) + g, tok = 2 * t + 8 * (j >> 1);
                    const uint32_t lo = tok < have ? vbits[tok * kDim + d] : 0u, hi = tok + 1 < have ? vbits[(tok + 1) * kDim + d] : 0u;
                    vf[i][j] = lo | hi << 16;
                    big = __vmaxu2(big, vf[i][j] & 0x7fff7fffu);
                }
            e = pow2_exponent(__reduce_max_sync(0xffffffffu, widest_half(big)));
            factor = e == 128 ? 0.f : pow2(-e);
            v_scale = e == 128 ? __uint_as_float(0x7fc00000u) : pow2(e);
#pragma unroll
            for (int i = 0; i < 2 * kC; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) vf[i][j] = bf16x2_to_f16x2(vf[i][j], factor);
        }

        float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            mma_f16_16816(s, kf[c][0][0], kf[c][0][1], kf[c][0][2], kf[c][0][3], qf[c][0][0], qf[c][0][1]);
            mma_f16_16816(s2, kf[c][1][0], kf[c][1][1], kf[c][1][2], kf[c][1][3], qf[c][1][0], qf[c][1][1]);
        }
        // tokens g, g + 8 of the block x heads 2 t, 2 t + 1. A scale that is not a number makes the weights of the tokens that are seen none,
        // and nothing else: 1 / scale stays 1.
        const float lv = __log2f(v_scale), inv = v_scale == v_scale ? __fdividef(1.f, v_scale) : 1.f;
        const int tok = b * kKv8Tokens + g;
        const bool see_lo = tok >= span.begin && tok < span.end, see_hi = tok + 8 >= span.begin && tok + 8 < span.end;
        const float c0 = k_scale * qs0, c1 = k_scale * qs1;
        float w[4];
        w[0] = see_lo ? fmaf(s[0] + s2[0], c0, lv) : -INFINITY;
        w[1] = see_lo ? fmaf(s[1] + s2[1], c1, lv) : -INFINITY;
        w[2] = see_hi ? fmaf(s[2] + s2[2], c0, lv) : -INFINITY;
        w[3] = see_hi ? fmaf(s[3] + s2[3], c1, lv) : -INFINITY;
        float x0 = fmaxf(w[0], w[2]), x1 = fmaxf(w[1], w[3]);
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
        }
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;   // nothing seen yet (or nothing but NaN)
        const float a0 = kv8_exp2(m0 - u0), a1 = kv8_exp2(m1 - u1);
        m0 = n0; m1 = n1;
        w[0] = kv8_exp2(w[0] - u0); w[2] = kv8_exp2(w[2] - u0);
        w[1] = kv8_exp2(w[1] - u1); w[3] = kv8_exp2(w[3] - u1);
        l0 = l0 * a0 + (w[0] + w[2]) * inv;
        l1 = l1 * a1 + (w[1] + w[3]) * inv;
        if (__any_sync(0xffffffffu, a0 != 1.f || a1 != 1.f)) {
#pragma unroll
            for (int i = 0; i < 2 * kC; ++i) { o[i][0] *= a0; o[i][1] *= a1; o[i][2] *= a0; o[i][3] *= a1; }
        }
        const uint32_t p0 = movmatrix_trans(pack_f16x2(w[0], w[1])), p1 = movmatrix_trans(pack_f16x2(w[2], w[3]));
#pragma unroll
        for (int i = 0; i < 2 * kC; ++i) mma_f16_16816(o[i], vf[i][0], vf[i][1], vf[i][2], vf[i][3], p0, p1);
    }
#pragma unroll
    for (int d = 4; d < 32; d *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    // ---- the warps' parts -----------------------------------------------------------------------------------------------------------------
#pragma unroll
    for (int i = 0; i < 2 * kC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o_part[warp][2 * t + (j & 1)][16 * i + 8 * (j >> 1) + g] = o[i][j];
    if (g == 0) {
        ml_part[warp][2 * t][0] = m0; ml_part[warp][2 * t][1] = l0;
        ml_part[warp][2 * t + 1][0] = m1; ml_part[warp][2 * t + 1][1] = l1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < cols * (kDim / 2); i += kWarps * 32) {
        const int h = i / (kDim / 2), d = i % (kDim / 2) * 2;
        float top = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) top = fmaxf(top, ml_part[v][h][0]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
            const float f = kv8_exp2(ml_part[v][h][0] - ref);
            // a warp whose blocks all count for nothing but NaN has no maximum and a sum of NaN
            const float fl = ml_part[v][h][0] == -INFINITY && ml_part[v][h][1] == 0.f ? 0.f : ml_part[v][h][0] == -INFINITY ? ml_part[v][h][1] : f;
            l += ml_part[v][h][1] * fl;
            x += o_part[v][h][d] * fl;
            y += o_part[v][h][d + 1] * fl;
        }
        const long long at = (long long)row * p.q_heads + head0 + h;
        if (parts <= 1) {
            const float r = blocks == 0 ? 0.f : l == 0.f ? 0.f : __fdividef(1.f, l);
            *reinterpret_cast<uint32_t*>(p.out + at * kDim + d) = pack_bf16x2(x * r, y * r);
        } else {
            const long long part = at * p.splits + split;
            *reinterpret_cast<float2*>(p.part_o + part * kDim + d) = make_float2(x, y);
            if (d == 0) { p.part_ml[2 * part] = top; p.part_ml[2 * part + 1] = l; }
        }
    }
}

// The parts of a row's head, added up in their order.
template <int kDim>
__global__ void __launch_bounds__(kDim / 2) kv8_merge_kernel(const Kv8Attention p) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, d = threadIdx.x * 2;
    const Kv8Span span = kv8_span(p, row);
    if (span.slot < 0) return;
    int first, blocks, parts = p.splits, per;
    if (p.n_tiles == 0) parts_of(p, span, &first, &blocks, &parts, &per);   // of a tile every part has its sum
    if (parts <= 1) return;
    const long long at = (long long)row * p.q_heads + blockIdx.x;
    const float* ml = p.part_ml + 2 * at * p.splits;
    float top = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
    for (int i = 0; i < parts; ++i) top = fmaxf(top, ml[2 * i]);
    const float ref = top == -INFINITY ? 0.f : top;
    for (int i = 0; i < parts; ++i) {
        const float f = ml[2 * i] == -INFINITY ? ml[2 * i + 1] : kv8_exp2(ml[2 * i] - ref);   // no maximum: nothing (0) or nothing but NaN
        if (ml[2 * i] == -INFINITY && f == 0.f) continue;                                             // and its part of the output is not there
        const float2 v = *reinterpret_cast<const float2*>(p.part_o + (at * p.splits + i) * kDim + d);
        l += ml[2 * i + 1] * f;
        x += v.x * f;
        y += v.y * f;
    }
    const float r = l == 0.f ? 0.f : __fdividef(1.f, l);
    *reinterpret_cast<uint32_t*>(p.out + at * kDim + d) = pack_bf16x2(x * r, y * r);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int kDim>
int launch_attention(const Kv8Attention& p, cudaStream_t st) {
    const int eights = (p.group + kCols - 1) / kCols;
    const int rc = p.n_tiles ? kv8_prompt_attention(p, kDim, st)
                             : launch_kernel(kv8_attention_kernel<kDim>, dim3((unsigned)p.splits, (unsigned)(p.kv_heads * eights), (unsigned)p.rows), dim3(kWarps * 32), 0, st, 1, p);
    if (rc || p.splits == 1) return rc;
    return launch_kernel(kv8_merge_kernel<kDim>, dim3((unsigned)p.q_heads, (unsigned)p.rows), dim3(kDim / 2), 0, st, 1, p);
}

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" {

int gptrs_cuda_kv8_splits(const gptrs_kv8_cache* c, int64_t rows, int64_t n_tiles, int64_t max_ctx_len) {
    if (!c || rows < 1 || c->kv_heads < 1) return 1;
    if (n_tiles > 0) {
        // a CTA per tile and kv head has an SM to itself: parts only where many SMs would have nothing, of 512 keys at least
        const int64_t ctas = n_tiles * c->kv_heads, keys = c->window > 0 ? std::min<int64_t>(max_ctx_len, c->window + c->tile_tokens) : max_ctx_len;
        return rows > 65535 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(sm_count() / ctas, keys / 512));
    }
    const int64_t seen = c->window > 0 ? std::min<int64_t>(max_ctx_len, c->window + kKv8Tokens) : max_ctx_len;
    const int64_t blocks = (seen + kKv8Tokens - 1) / kKv8Tokens;
    const int64_t ctas = rows * c->kv_heads;
    const int64_t want = (8 * (int64_t)sm_count() + ctas - 1) / ctas;       // several CTAs per SM
    const int64_t most = (blocks + 4 * kWarps - 1) / (4 * kWarps);          // a warp takes four blocks at least
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(want, most), 256));
}

size_t gptrs_cuda_kv8_scratch_bytes(const gptrs_kv8_cache* c, int64_t rows, int64_t n_tiles, int splits) {
    if (!c || splits <= 1 || rows < 1) return 0;
    return (size_t)rows * c->q_heads * splits * (c->dim + 2) * sizeof(float);
}

int gptrs_cuda_kv8_attention(const gptrs_kv8_cache* c, const gptrs_kv8_attention_step* s, void* stream) {
    const int rc = kv8_check(c);
    if (rc) return rc;
    GPTRS_REQUIRE(s && s->d_q && s->d_pool && s->d_open && s->d_page_table && s->d_slot && s->d_ctx_len && s->d_length && s->d_out && s->d_status, "null pointer");
    GPTRS_REQUIRE(s->rows >= 0 && s->rows <= 0x3fffffff && s->n_tiles >= 0 && s->n_tiles <= 65535, "bad row count");
    GPTRS_REQUIRE(s->n_tiles == 0 || (s->d_tile_row && s->d_tile_rows), "tiles are missing");
    GPTRS_REQUIRE(s->max_pages >= 1 && s->max_pages * kKv8Tokens < ((int64_t)1 << 31) && s->n_pages >= 1 && s->n_slots >= 1 && s->n_slots <= 0x7fffffff, "bad cache sizes");
    GPTRS_REQUIRE(s->max_ctx_len >= 0 && s->max_ctx_len < ((int64_t)1 << 31), "bad max_ctx_len");
    GPTRS_REQUIRE(s->splits >= 1 && s->splits <= 65535, "bad number of splits");
    GPTRS_REQUIRE(aligned16(s->d_q) && aligned16(s->d_pool) && aligned16(s->d_open) && aligned16(s->d_out) && aligned16(s->d_scratch), "pointers must be 16-byte aligned");
    const int64_t width = (int64_t)c->q_heads * c->dim;
    Kv8Attention p = {};
    p.ldq = s->ldq ? s->ldq : width;
    GPTRS_REQUIRE(p.ldq >= width && p.ldq % 8 == 0, "rows of queries overlap, or do not start at multiples of 16 bytes");
    GPTRS_REQUIRE(s->splits == 1 || (s->d_scratch && s->scratch_bytes >= gptrs_cuda_kv8_scratch_bytes(c, s->rows, s->n_tiles, s->splits)), "scratch is too small");
    if (s->rows == 0) return GPTRS_OK;
    p.q = static_cast<const __nv_bfloat16*>(s->d_q);
    p.pool = static_cast<const unsigned char*>(s->d_pool);
    p.open = static_cast<const __nv_bfloat16*>(s->d_open);
    p.table = s->d_page_table; p.slot = s->d_slot; p.ctx_len = s->d_ctx_len; p.length = s->d_length;
    p.out = static_cast<__nv_bfloat16*>(s->d_out);
    p.status = s->d_status;
    p.n_pages = s->n_pages; p.max_pages = s->max_pages; p.n_slots = (int)s->n_slots; p.rows = (int)s->rows;
    p.q_heads = c->q_heads; p.kv_heads = c->kv_heads; p.group = c->q_heads / c->kv_heads; p.window = c->window;
    p.scale_log2 = c->scale * kKv8Log2e;
    p.splits = s->splits;
    p.max_len = (int)std::min<int64_t>(s->max_ctx_len, s->max_pages * kKv8Tokens);
    const int64_t blocks = (p.max_len + kKv8Tokens - 1) / kKv8Tokens;
    const int64_t seen = c->window > 0 ? std::min<int64_t>(blocks, c->window / kKv8Tokens + 2) : blocks;
    p.chunk_blocks = std::max(1, ceil_div(seen, s->splits));
    p.part_o = static_cast<float*>(s->d_scratch);
    p.part_ml = p.part_o + (size_t)p.rows * p.q_heads * p.splits * c->dim;
    p.tile_row = s->d_tile_row; p.tile_rows = s->d_tile_rows; p.n_tiles = (int)s->n_tiles;
    // a grid's last dimension holds 65535 rows: longer lists go in several launches over their own part of the scratch
    const int64_t most = s->n_tiles && s->splits == 1 ? s->rows : 65535;
    GPTRS_REQUIRE(s->n_tiles == 0 || s->rows <= most, "tiles of more than 65535 rows are not split along the keys");
    for (int64_t row = 0; row < s->rows; row += most) {
        Kv8Attention part = p;
        part.rows = (int)std::min<int64_t>(most, s->rows - row);
        part.q += row * p.ldq; part.slot += row; part.ctx_len += row;
        part.out += row * width;
        part.part_o += row * p.q_heads * p.splits * c->dim;
        part.part_ml += row * p.q_heads * p.splits * 2;
        const int e = c->dim == 64 ? launch_attention<64>(part, as_stream(stream)) : launch_attention<128>(part, as_stream(stream));
        if (e) return e;
    }
    return GPTRS_OK;
}

}  // extern "C"
