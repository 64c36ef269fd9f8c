// Attention over the 8-bit cache, row by row (single tokens of many sequences).
//
// With keys k = s_K a and values v = s_V b of whole numbers a, b and a scale per block of 16 tokens, for every query head
//     t_j = (s_K scale log2 e) q . a_j + log2 s_V        w_j = 2^(t_j - M)        out = sum_j w_j b_j / sum_j (w_j / s_V)
// The value's scale rides in the exponent, so one running reference M bounds the weights whatever the scales are, and no product needs a scale of its own. M is
// the maximum less 15: weights go as f16 up to 2^15, with 11 bits down to 2^-29 of the largest and off by at most 2^-40 of it below, so that the
// tokens of a long tail still count beside one that has nearly all of the weight (2^20 of them lose 2^-20 of it). Queries are f16 with a power of two in front
// (kv8_cache.cuh), sums and maxima f32.
//
// A warp takes a block at a time. Keys are the rows of the matrix product, heads its columns (eight query heads of a kv head at most): S^T = K Q^T
// and O^T = V^T P^T, so that little of a matrix instruction is padding. The cache's byte order makes 16 bytes of a lane two k-steps of keys, or two
// row tiles of values. The 8 x 8 transposition between the two products is one instruction per eight tokens.
// Four warps deal the blocks of a part of the keys among them, each with a ring of its own in shared memory that bulk copies fill (a block is one piece of
// memory, its scales included), and merge at the end. Up to eight parts of a row and kv head (of eight of its query heads) that fit into one wave
// of CTAs are a cluster that merges through distributed shared memory; others go through scratch and a second kernel. Parts are cut by the bound of the
// lengths that the caller gives, so a bound far above a row's length leaves it fewer of them: one sequence of 1500 tokens, 32 / 8 heads of 128, takes 8.1 us with a
// bound of 1504, 14.6 with 32768 and 20.0 with 131072; 64 of 512 to 8192 104 us with 8192 and 123 with 131072.
#include <algorithm>
#include <type_traits>

#include "kv8_attention.cuh"

namespace gptrs {

void prefill_tc_fault(int* starve, uint32_t* wait_limit);   // the test switch of paged_prefill_tc.cu

namespace {

constexpr int kWarps = 4;
constexpr int kCols = 8;    // query heads of a CTA
constexpr int kDepth = 4;   // blocks of a warp's ring
constexpr int kCtas = 3;    // of an SM
constexpr int kMostRanks = 8;   // parts that a cluster merges
constexpr float kHeadroom = 15.f;   // log2 of the largest weight

// Weight of a part (warp, CTA, split) with reference m and sum l beside the largest reference; one without a reference has seen nothing (0) or nothing but NaN.
__device__ __forceinline__ float part_factor(float m, float l, float top) { return m == -INFINITY ? (l == 0.f ? 0.f : l) : kv8_exp2(m - top); }
__device__ __forceinline__ uint4 lds_16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// A row's blocks in parts of equal size, at most chunk_blocks each.
__device__ __forceinline__ void parts_of(const Kv8Attention& p, const Kv8Span& s, int* first, int* blocks, int* parts, int* per) {
    *first = s.begin / kKv8Tokens;
    *blocks = s.end > s.begin ? (s.end - 1) / kKv8Tokens + 1 - *first : 0;
    *parts = (*blocks + p.chunk_blocks - 1) / p.chunk_blocks;
    *per = *parts > 0 ? (*blocks + *parts - 1) / *parts : 1;
    *parts = (*blocks + *per - 1) / *per;
}

// Merges few parts (eight at most, see kv8_merge_kernel for more): dim / 4 threads have a row's head to themselves.
template <int kDim>
__global__ void __launch_bounds__(256) kv8_merge_few_kernel(const Kv8Attention p) {
    pdl_launch_dependents();
    pdl_wait();
    const long long item = (long long)blockIdx.x * (256 / (kDim / 4)) + threadIdx.x / (kDim / 4);
    const int row = kv8_row(p, (int)(item / p.q_heads)), d = threadIdx.x % (kDim / 4) * 4;
    if (row < 0) return;
    const long long at = (long long)row * p.q_heads + item % p.q_heads;
    const Kv8Span span = kv8_span(p, row);
    if (span.slot < 0) return;
    int first, blocks, parts = p.splits, per;
    if (p.n_tiles == 0) parts_of(p, span, &first, &blocks, &parts, &per);
    if (parts <= 1) return;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + at * p.splits;
    float2 x[kMostRanks];
    float4 v[kMostRanks];
    float top = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < kMostRanks; ++i)
        if (i < parts) { x[i] = ml[i]; top = fmaxf(top, x[i].x); }
#pragma unroll
    for (int i = 0; i < kMostRanks; ++i)   // a part that has seen nothing has no output
        v[i] = i < parts && !(x[i].x == -INFINITY && x[i].y == 0.f) ? *reinterpret_cast<const float4*>(p.part_o + (at * p.splits + i) * kDim + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kMostRanks; ++i)
        if (i < parts) {
            const float f = part_factor(x[i].x, x[i].y, top);
            l += x[i].y * f;
            o.x += v[i].x * f; o.y += v[i].y * f; o.z += v[i].z * f; o.w += v[i].w * f;
        }
    const float r = l == 0.f ? 0.f : __fdividef(1.f, l);
    *reinterpret_cast<uint2*>(p.out + at * kDim + d) = make_uint2(pack_bf16x2(o.x * r, o.y * r), pack_bf16x2(o.z * r, o.w * r));
}

struct AttentionLaunch {
    Kv8Attention a;
    uint32_t spins;               // polls of a bounded wait
    int starve;                   // test switch: the first block of a warp is never asked for
};

// kCluster: the splits of a row and kv head are a cluster (grid.y) that merges through distributed shared memory; else they are grid.x and write parts.
template <int kDim, bool kCluster>
__global__ void __launch_bounds__(kWarps * 32, kCtas) kv8_attention_kernel(const AttentionLaunch launch) {
    constexpr int kC = kDim / 32;      // chunks of 32 channels
    constexpr int kBlockBytes = (int)kv8_block_bytes(kDim);
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ __align__(8) uint64_t full[kWarps][kDepth];
    __shared__ float ml_part[kWarps][kCols][2];
    __shared__ __align__(16) float own_part[kCluster ? kCols * (kDim + 4) : 4];   // kCluster: output, reference and sum of this CTA's part

    const Kv8Attention& p = launch.a;
    const int split = kCluster ? blockIdx.y : blockIdx.x, pair = kCluster ? blockIdx.x : blockIdx.y, eights = (p.group + kCols - 1) / kCols;
    const int kv_head = pair / eights, head0 = kv_head * p.group + (pair % eights) * kCols;
    const int cols = min(kCols, p.group - (pair % eights) * kCols);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (lane == 0) {
        for (int i = 0; i < kDepth; ++i) mbar_init(&full[warp][i], 1);
        mbar_fence_init();
    }
    __syncwarp();
    pdl_launch_dependents();
    pdl_wait();
    const int row = kv8_row(p, blockIdx.z);
    if (row < 0) return;                          // (the whole cluster)
    // the query, on its way while the lengths are
    const __nv_bfloat16* const q_src = p.q + row * p.ldq + (long long)(head0 + min(g, cols - 1)) * kDim + 8 * t;
    uint4 raw[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) raw[c] = __ldg(reinterpret_cast<const uint4*>(q_src + 32 * c));
    const Kv8Span span = kv8_span(p, row);
    if (span.slot < 0) return;                    // (the whole cluster)
    int first, blocks, parts, per;
    parts_of(p, span, &first, &blocks, &parts, &per);
    if (!kCluster && split >= parts && !(split == 0 && parts == 0)) return;
    const int b0 = first + min(split * per, blocks) + warp, b_end = first + min((split + 1) * per, blocks);
    const int n_my = b_end > b0 ? (b_end - b0 + kWarps - 1) / kWarps : 0;                        // blocks b0, b0 + kWarps, ..
    const bool last_open = n_my > 0 && (b0 + (n_my - 1) * kWarps + 1) * kKv8Tokens > span.length;   // only a sequence's last block is not complete
    const int n_closed = n_my - (last_open ? 1 : 0);

    // ---- the warp's ring: blocks by bulk copies, their pages' numbers 32 at a time --------------------------------------------------------------
    unsigned char* const my_ring = ring + warp * (kDepth * kBlockBytes);
    const int* const numbers = p.table + span.slot * p.max_pages + b0;
    int my_page = 0;
    uint32_t bad[2] = {0, 0};                     // numbers that are none, of the 32 blocks asked for last and of those before them
    auto ask = [&](int j) {                       // whole warp, j one after the other
        if ((j & 31) == 0) {
            my_page = j + lane < n_closed ? numbers[(j + lane) * kWarps] : 0;
            const bool none = my_page < 0 || my_page >= p.n_pages;
            if (none) { atomicExch(p.status, 2); my_page = 0; }
            bad[(j >> 5) & 1] = __ballot_sync(0xffffffffu, none);
        }
        const int page = __shfl_sync(0xffffffffu, my_page, j & 31);
        if (lane == 0) {
            uint64_t* const bar = &full[warp][j % kDepth];
            mbar_expect_tx(bar, kBlockBytes);
            if (!(launch.starve && j == 0)) bulk_g2s(my_ring + j % kDepth * kBlockBytes, p.pool + ((long long)page * p.kv_heads + kv_head) * kBlockBytes, kBlockBytes, bar);
        }
    };
    for (int j = 0; j < kDepth && j < n_closed; ++j) ask(j);

    // ---- queries: column g of B, channels 32 c + 8 t + 4 s .. + 3; f16 with a power of two in front --------------------------------------------------
    uint32_t qf[kC][2][2];
    float q_scale;
    {
        uint32_t big = 0;
#pragma unroll
        for (int c = 0; c < kC; ++c) big = __vmaxu2(big, __vmaxu2(abs_bits_max2(raw[c].x, raw[c].y), abs_bits_max2(raw[c].z, raw[c].w)));
        uint32_t top = widest_half(big);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = pow2_exponent(top);
        const float factor = e == 128 ? 0.f : pow2(-e);
        q_scale = e == 128 ? __uint_as_float(0x7fc00000u) : pow2(e) * p.scale_log2;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            qf[c][0][0] = bf16x2_to_f16x2(raw[c].x, factor); qf[c][0][1] = bf16x2_to_f16x2(raw[c].y, factor);
            qf[c][1][0] = bf16x2_to_f16x2(raw[c].z, factor); qf[c][1][1] = bf16x2_to_f16x2(raw[c].w, factor);
        }
    }
    // the lane's two columns of S^T: heads 2 t, 2 t + 1
    const float qs0 = __shfl_sync(0xffffffffu, q_scale, 8 * t), qs1 = __shfl_sync(0xffffffffu, q_scale, 8 * t + 4);

    float o[2 * kC][4];
#pragma unroll
    for (int i = 0; i < 2 * kC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    bool failed = false;

    // Scores of kCount blocks (the first one's number and the distance to the next) -> weights, packed as the second operand of O^T = V^T P^T; o scaled to the
    // new references. count: tokens of a block with bit i of `none` do not count
    auto weigh = [&](auto count, const float (*s)[4], int b, const float2* scale, uint32_t none, uint32_t (*packed)[2]) {
        constexpr int kCount = decltype(count)::value;
        // tokens g, g + 8 of a block x heads 2 t, 2 t + 1. A scale that is not a number makes the weights of the tokens that are seen none, and
        // nothing else: 1 / scale stays 1.
        float w[kCount][4], x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
        for (int u = 0; u < kCount; ++u) {
            const float lv = __log2f(scale[u].y), c0 = scale[u].x * qs0, c1 = scale[u].x * qs1;
            const int tok = (b + u * kWarps) * kKv8Tokens + g;
            const bool counts = !((none >> u) & 1), see_lo = tok >= span.begin && tok < span.end && counts, see_hi = tok + 8 >= span.begin && tok + 8 < span.end && counts;
            w[u][0] = see_lo ? fmaf(s[u][0], c0, lv) : -INFINITY;
            w[u][1] = see_lo ? fmaf(s[u][1], c1, lv) : -INFINITY;
            w[u][2] = see_hi ? fmaf(s[u][2], c0, lv) : -INFINITY;
            w[u][3] = see_hi ? fmaf(s[u][3], c1, lv) : -INFINITY;
            x0 = fmaxf(x0, fmaxf(w[u][0], w[u][2]));
            x1 = fmaxf(x1, fmaxf(w[u][1], w[u][3]));
        }
#pragma unroll
        for (int d = 4; d < 32; d *= 2) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
        }
        // (rounded up: where a step of a score is more than 1, a reference further down would make the largest weight infinite)
        const float n0 = fmaxf(m0, __fadd_ru(x0, -kHeadroom)), n1 = fmaxf(m1, __fadd_ru(x1, -kHeadroom));
        const float u0 = n0 == -INFINITY ? 0.f : n0, u1 = n1 == -INFINITY ? 0.f : n1;   // nothing seen yet (or nothing but NaN)
        const float a0 = kv8_exp2(m0 - u0), a1 = kv8_exp2(m1 - u1);
        m0 = n0; m1 = n1;
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int u = 0; u < kCount; ++u) {
            const float inv = scale[u].y == scale[u].y ? __fdividef(1.f, scale[u].y) : 1.f;
            w[u][0] = kv8_exp2(w[u][0] - u0); w[u][2] = kv8_exp2(w[u][2] - u0);
            w[u][1] = kv8_exp2(w[u][1] - u1); w[u][3] = kv8_exp2(w[u][3] - u1);
            l0 = fmaf(w[u][0] + w[u][2], inv, l0);
            l1 = fmaf(w[u][1] + w[u][3], inv, l1);
            packed[u][0] = movmatrix_trans(pack_f16x2(w[u][0], w[u][1]));
            packed[u][1] = movmatrix_trans(pack_f16x2(w[u][2], w[u][3]));
        }
        if (__any_sync(0xffffffffu, a0 != 1.f || a1 != 1.f)) {
#pragma unroll
            for (int i = 0; i < 2 * kC; ++i) { o[i][0] *= a0; o[i][1] *= a1; o[i][2] *= a0; o[i][3] *= a1; }
        }
    };
    // kCount blocks of the ring from the j-th on: two at a time share the maxima's exchange between lanes and hide each other's latencies
    auto visit = [&](auto count, int j) {
        constexpr int kCount = decltype(count)::value;
        float s[kCount][4];
        float2 scale[kCount];
        uint4 vb[kCount][kC];
        uint32_t none = 0;
#pragma unroll
        for (int u = 0; u < kCount; ++u) {
            const int st = (j + u) % kDepth;
            bool got = false;
            for (uint32_t i = 0; i < launch.spins && !got; ++i) got = mbar_try_wait(&full[warp][st], (uint32_t)((j + u) / kDepth) & 1u);
            if (__any_sync(0xffffffffu, !got)) {
                // copies on their way write this CTA's shared memory: wait for them too
                for (int k = j + u; k < min(j + kDepth, n_closed); ++k)
                    for (uint32_t i = 0; i < launch.spins && !mbar_try_wait(&full[warp][k % kDepth], (uint32_t)(k / kDepth) & 1u); ++i) {}
                if (lane == 0) atomicExch(p.status, 3);
                failed = true;
                return;
            }
            const uint32_t at = smem_u32(my_ring + st * kBlockBytes) + lane * 16;
            scale[u] = *reinterpret_cast<const float2*>(my_ring + st * kBlockBytes + 32 * kDim);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] = 0.f;
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                const uint4 kb = lds_16(at + c * 512);
                uint32_t k[8];
                kv8_widen(kb.x, &k[0], &k[1]); kv8_widen(kb.z, &k[2], &k[3]);
                kv8_widen(kb.y, &k[4], &k[5]); kv8_widen(kb.w, &k[6], &k[7]);
                mma_f16_16816(s[u], k[0], k[2], k[1], k[3], qf[c][0][0], qf[c][0][1]);
                mma_f16_16816(s[u], k[4], k[6], k[5], k[7], qf[c][1][0], qf[c][1][1]);
            }
#pragma unroll
            for (int c = 0; c < kC; ++c) vb[u][c] = lds_16(at + 16 * kDim + c * 512);
            none |= ((bad[((j + u) >> 5) & 1] >> ((j + u) & 31)) & 1) << u;
        }
        __syncwarp();
        if (j + kDepth < n_closed) {              // every lane has read the stages
            fence_proxy_async();
            ask(j + kDepth);
            if (kCount == 2 && j + 1 + kDepth < n_closed) ask(j + 1 + kDepth);
        }
        uint32_t packed[kCount][2];
        weigh(count, s, b0 + j * kWarps, scale, none, packed);
#pragma unroll
        for (int u = 0; u < kCount; ++u)
#pragma unroll
            for (int c = 0; c < kC; ++c) {
                uint32_t v[8];
                kv8_widen(vb[u][c].x, &v[0], &v[2]); kv8_widen(vb[u][c].y, &v[1], &v[3]);
                kv8_widen(vb[u][c].z, &v[4], &v[6]); kv8_widen(vb[u][c].w, &v[5], &v[7]);
                mma_f16_16816(o[2 * c], v[0], v[1], v[2], v[3], packed[u][0], packed[u][1]);
                mma_f16_16816(o[2 * c + 1], v[4], v[5], v[6], v[7], packed[u][0], packed[u][1]);
            }
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    int j = 0;
    for (; j + 1 < n_closed && !failed; j += 2) visit(Two{}, j);
    if (j < n_closed && !failed) visit(One{}, j);
    if (last_open && !failed) {
        // the block that is not complete: bf16 rows; what lies behind the last token may be anything and counts as zero
        const int b = b0 + (n_my - 1) * kWarps, have = span.length - b * kKv8Tokens;
        const __nv_bfloat16* ks = p.open + (long long)span.slot * kv8_open_elems(p.kv_heads, kDim) + kv8_open_at(b, p.kv_heads, kv_head, 0, kDim);
        uint4 kr[kC][2];
        uint32_t v[2 * kC][4];
#pragma unroll
        for (int c = 0; c < kC; ++c)
#pragma unroll
            for (int r = 0; r < 2; ++r) kr[c][r] = g + 8 * r < have ? *reinterpret_cast<const uint4*>(ks + (g + 8 * r) * kDim + 32 * c + 8 * t) : make_uint4(0, 0, 0, 0);
        const unsigned short* vs = reinterpret_cast<const unsigned short*>(ks + kKv8Tokens * kDim);
#pragma unroll
        for (int i = 0; i < 2 * kC; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = 16 * i + 8 * (j & 1) + g, tok = 2 * t + 8 * (j >> 1);
                const uint32_t lo = tok < have ? vs[tok * kDim + d] : 0u, hi = tok + 1 < have ? vs[(tok + 1) * kDim + d] : 0u;
                v[i][j] = lo | hi << 16;
            }
        int e, ev;
        auto exponents = [&] {
            uint32_t big = 0, big_v = 0;
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int r = 0; r < 2; ++r) big = __vmaxu2(big, __vmaxu2(abs_bits_max2(kr[c][r].x, kr[c][r].y), abs_bits_max2(kr[c][r].z, kr[c][r].w)));
#pragma unroll
            for (int i = 0; i < 2 * kC; ++i) big_v = __vmaxu2(big_v, __vmaxu2(abs_bits_max2(v[i][0], v[i][1]), abs_bits_max2(v[i][2], v[i][3])));
            e = pow2_exponent(__reduce_max_sync(0xffffffffu, widest_half(big)));
            ev = pow2_exponent(__reduce_max_sync(0xffffffffu, widest_half(big_v)));
        };
        exponents();
        // What is not finite makes its token's weights none for the rows that see it. It counts as zero itself, or 0 x infinity would reach the others.
        uint32_t none = 0;   // tokens
        if (e == 128 || ev == 128) {   // (the whole warp)
#pragma unroll
            for (int c = 0; c < kC; ++c)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    if (drop_not_finite(kr[c][r].x) | drop_not_finite(kr[c][r].y) | drop_not_finite(kr[c][r].z) | drop_not_finite(kr[c][r].w)) none |= 1u << (g + 8 * r);
#pragma unroll
            for (int i = 0; i < 2 * kC; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t halves = drop_not_finite(v[i][j]);
                    none |= ((halves & 1u) | (halves >> 31) << 1) << (2 * t + 8 * (j >> 1));
                }
            none = __reduce_or_sync(0xffffffffu, none);
            exponents();
        }
        const float factor = pow2(-e), factor_v = pow2(-ev);
        float s[1][4] = {};
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            mma_f16_16816(s[0], bf16x2_to_f16x2(kr[c][0].x, factor), bf16x2_to_f16x2(kr[c][1].x, factor), bf16x2_to_f16x2(kr[c][0].y, factor), bf16x2_to_f16x2(kr[c][1].y, factor),
                          qf[c][0][0], qf[c][0][1]);
            mma_f16_16816(s[0], bf16x2_to_f16x2(kr[c][0].z, factor), bf16x2_to_f16x2(kr[c][1].z, factor), bf16x2_to_f16x2(kr[c][0].w, factor), bf16x2_to_f16x2(kr[c][1].w, factor),
                          qf[c][1][0], qf[c][1][1]);
        }
        if ((none >> g) & 1) s[0][0] = s[0][1] = __uint_as_float(0x7fc00000u);
        if ((none >> (g + 8)) & 1) s[0][2] = s[0][3] = __uint_as_float(0x7fc00000u);
        uint32_t packed[1][2];
        const float2 scale = make_float2(pow2(e), pow2(ev));
        weigh(One{}, s, b, &scale, 0, packed);
#pragma unroll
        for (int i = 0; i < 2 * kC; ++i)
            mma_f16_16816(o[i], bf16x2_to_f16x2(v[i][0], factor_v), bf16x2_to_f16x2(v[i][1], factor_v), bf16x2_to_f16x2(v[i][2], factor_v), bf16x2_to_f16x2(v[i][3], factor_v), packed[0][0],
                          packed[0][1]);
    }
#pragma unroll
    for (int d = 4; d < 32; d *= 2) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    // ---- the warps' parts (their rings are done with) -------------------------------------------------------------------------------------------------
    __syncthreads();
    float (*const o_part)[kCols][kDim + 1] = reinterpret_cast<float(*)[kCols][kDim + 1]>(ring);
#pragma unroll
    for (int i = 0; i < 2 * kC; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o_part[warp][2 * t + (j & 1)][16 * i + 8 * (j >> 1) + g] = o[i][j];
    if (g == 0) {
        ml_part[warp][2 * t][0] = m0; ml_part[warp][2 * t][1] = l0;
        ml_part[warp][2 * t + 1][0] = m1; ml_part[warp][2 * t + 1][1] = l1;
    }
    __syncthreads();
    const bool cluster = kCluster && gridDim.y > 1;
    for (int i = threadIdx.x; i < cols * (kDim / 4); i += kWarps * 32) {
        const int h = i / (kDim / 4), d = i % (kDim / 4) * 4;
        float top = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < kWarps; ++v) top = fmaxf(top, ml_part[v][h][0]);
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
            const float f = part_factor(ml_part[v][h][0], ml_part[v][h][1], top);
            l += ml_part[v][h][1] * f;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] += o_part[v][h][d + k] * f;
        }
        const long long at = (long long)row * p.q_heads + head0 + h;
        if (cluster) {
            float* const mine = own_part + h * (kDim + 4);
            *reinterpret_cast<float4*>(mine + d) = make_float4(x[0], x[1], x[2], x[3]);
            if (d == 0) { mine[kDim] = top; mine[kDim + 1] = l; }
        } else if (kCluster || parts <= 1) {
            const float r = l == 0.f ? 0.f : __fdividef(1.f, l);
            *reinterpret_cast<uint2*>(p.out + at * kDim + d) = make_uint2(pack_bf16x2(x[0] * r, x[1] * r), pack_bf16x2(x[2] * r, x[3] * r));
        } else {
            const long long part = at * p.splits + split;
            *reinterpret_cast<float4*>(p.part_o + part * kDim + d) = make_float4(x[0], x[1], x[2], x[3]);
            if (d == 0) { p.part_ml[2 * part] = top; p.part_ml[2 * part + 1] = l; }
        }
    }
    if (cluster) {   // the parts in the order of the ranks, four channels of a head per thread, the work dealt over the ranks
        const int ranks = gridDim.y, rank = (int)cluster_ctarank();
        cluster_sync_all();
        const uint32_t base = smem_u32(own_part);
        for (int i = threadIdx.x * ranks + rank; i < cols * (kDim / 4); i += kWarps * 32 * ranks) {
            const int h = i / (kDim / 4), d = i % (kDim / 4) * 4;
            float4 o4[kMostRanks];
            float2 ml[kMostRanks];
            float top = -INFINITY, l = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < kMostRanks; ++r)
                if (r < ranks) {
                    const uint32_t at = map_to_cta(base + (uint32_t)(h * (kDim + 4)) * 4, (uint32_t)r);
                    o4[r] = ld_dsmem_f4(at + d * 4);
                    const float4 y = ld_dsmem_f4(at + kDim * 4);
                    ml[r] = make_float2(y.x, y.y);
                    top = fmaxf(top, ml[r].x);
                }
#pragma unroll
            for (int r = 0; r < kMostRanks; ++r)
                if (r < ranks) {
                    const float f = part_factor(ml[r].x, ml[r].y, top);
                    l += ml[r].y * f;
                    x[0] += o4[r].x * f; x[1] += o4[r].y * f; x[2] += o4[r].z * f; x[3] += o4[r].w * f;
                }
            const float r = l == 0.f ? 0.f : __fdividef(1.f, l);
            *reinterpret_cast<uint2*>(p.out + ((long long)row * p.q_heads + head0 + h) * kDim + d) = make_uint2(pack_bf16x2(x[0] * r, x[1] * r), pack_bf16x2(x[2] * r, x[3] * r));
        }
        cluster_sync_all();   // the parts stay until every rank has read them
    }
}

// The parts of a row's head: dim / 4 threads take every kMergers-th part, four channels each, and their sums are added up in order.
constexpr int kMergers = 8;
template <int kDim>
__global__ void __launch_bounds__(kMergers * kDim / 4) kv8_merge_kernel(const Kv8Attention p) {
    __shared__ __align__(16) float sum[kMergers][kDim], total[kMergers];
    pdl_launch_dependents();
    pdl_wait();
    const int row = kv8_row(p, blockIdx.x), d = threadIdx.x % (kDim / 4) * 4, m = threadIdx.x / (kDim / 4);
    if (row < 0) return;
    const Kv8Span span = kv8_span(p, row);
    if (span.slot < 0) return;
    int first, blocks, parts = p.splits, per;
    if (p.n_tiles == 0) parts_of(p, span, &first, &blocks, &parts, &per);   // of a tile every part has its sum
    if (parts <= 1) return;
    const long long at = (long long)row * p.q_heads + blockIdx.y;
    const float* ml = p.part_ml + 2 * at * p.splits;
    float top = -INFINITY;
    for (int i = 0; i < parts; ++i) top = fmaxf(top, ml[2 * i]);
    float l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = m; i < parts; i += kMergers) {
        const float f = part_factor(ml[2 * i], ml[2 * i + 1], top);
        if (ml[2 * i] == -INFINITY && f == 0.f) continue;                     // and its part of the output is not there
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + (at * p.splits + i) * kDim + d);
        l += ml[2 * i + 1] * f;
        x.x += v.x * f; x.y += v.y * f; x.z += v.z * f; x.w += v.w * f;
    }
    *reinterpret_cast<float4*>(&sum[m][d]) = x;
    if (d == 0) total[m] = l;
    __syncthreads();
    if (m > 0) return;
    for (int i = 1; i < kMergers; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(&sum[i][d]);
        x.x += v.x; x.y += v.y; x.z += v.z; x.w += v.w;
        l += total[i];
    }
    const float r = l == 0.f ? 0.f : __fdividef(1.f, l);
    *reinterpret_cast<uint2*>(p.out + at * kDim + d) = make_uint2(pack_bf16x2(x.x * r, x.y * r), pack_bf16x2(x.z * r, x.w * r));
}

// Parts of a row and kv head (of eight of its query heads) that all fit into one wave of CTAs are merged by their cluster; others go one by one, as places
// come free, and meet in scratch.
int64_t pairs_of(const gptrs_kv8_cache& c) { return (int64_t)c.kv_heads * ((c.q_heads / c.kv_heads + kCols - 1) / kCols); }
int64_t places() { return (int64_t)kCtas * sm_count(); }
bool in_cluster(const gptrs_kv8_cache& c, int64_t rows, int splits) { return splits == 1 || (splits <= kMostRanks && rows * pairs_of(c) * splits <= places()); }
// One wave of clusters, down to a block per warp.
int cluster_parts(const gptrs_kv8_cache& c, int64_t rows, int64_t blocks) {
    return (int)std::max<int64_t>(1, std::min<int64_t>({places() / (rows * pairs_of(c)), kMostRanks, (blocks + kWarps - 1) / kWarps}));
}

// Whether the rows of tiles are faster one by one than a tile at a time, from estimates in us. One by one: a wave of CTAs (row x kv head) takes 3 us and what its
// longest row does; a tile takes about 12 us, and 2.3 for every 128 keys. (One prompt, 32 / 8 heads of 128: 16 tokens 4.0 against 12.2 us, 128 12.7 against
// 16.9, 256 26 against 19; 8 / 1 heads: 512 tokens 13.6 against 24, 2048 86 against 46.)
bool rows_one_by_one(const gptrs_kv8_cache& c, int64_t rows, int64_t n_tiles, int64_t max_len) {
    const int64_t seen = c.window > 0 ? std::min<int64_t>(max_len, c.window) : max_len, pairs = pairs_of(c);
    if (n_tiles * c.tile_tokens > 65535) return false;
    const double by_row = (double)((rows * pairs + kCtas * sm_count() - 1) / (kCtas * sm_count())) * (3. + seen / 2 / 64. * .9);
    const double by_tile = 12. + (double)((n_tiles * c.kv_heads + sm_count() - 1) / sm_count()) * (seen / 128.) * 2.3;
    return by_row < by_tile;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int kDim>
int launch_attention(const Kv8Attention& p, cudaStream_t st) {
    const unsigned pairs = (unsigned)(p.kv_heads * ((p.group + kCols - 1) / kCols));
    constexpr size_t smem = (size_t)kWarps * kDepth * kv8_block_bytes(kDim);
    static_assert(smem >= sizeof(float) * kWarps * kCols * (kDim + 1), "the warps' parts go where the rings were");
    static PerDeviceOnce attr_once;
    if (attr_once.first_time()) {
        GPTRS_CUDA_OK(cudaFuncSetAttribute(kv8_attention_kernel<kDim, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        GPTRS_CUDA_OK(cudaFuncSetAttribute(kv8_attention_kernel<kDim, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    }
    AttentionLaunch launch = {p, kSpinLimit, 0};
    uint32_t limit;
    prefill_tc_fault(&launch.starve, &limit);
    if (launch.starve) launch.spins = limit;
    int rc;
    const int64_t rows = p.n_tiles ? (int64_t)p.n_tiles * p.tile_tokens : p.rows;   // that kv8_row goes through
    if (p.n_tiles && !p.one_by_one) rc = kv8_prompt_attention(p, kDim, st);
    else if (p.clustered)
        return launch_kernel(kv8_attention_kernel<kDim, true>, dim3(pairs, (unsigned)p.splits, (unsigned)rows), dim3(kWarps * 32), smem, st,
                             p.splits, launch);
    else rc = launch_kernel(kv8_attention_kernel<kDim, false>, dim3((unsigned)p.splits, pairs, (unsigned)p.rows), dim3(kWarps * 32), smem, st, 1, launch);
    if (rc || p.splits == 1) return rc;
    // the merge waits for the parts itself (griddepcontrol.wait), so it may be launched ahead of their end
    const int pdl = g_use_pdl;
    g_use_pdl = 1;
    constexpr int kAtOnce = 256 / (kDim / 4);
    if (p.splits <= kMostRanks)
        rc = launch_kernel(kv8_merge_few_kernel<kDim>, dim3((unsigned)ceil_div(rows * p.q_heads, kAtOnce)), dim3(256), 0, st, 1, p);
    else
        rc = launch_kernel(kv8_merge_kernel<kDim>, dim3((unsigned)rows, (unsigned)p.q_heads), dim3(kMergers * kDim / 4), 0, st, 1, p);
    g_use_pdl = pdl;
    return rc;
}

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" {

int gptrs_cuda_kv8_splits(const gptrs_kv8_cache* c, int64_t rows, int64_t n_tiles, int64_t max_ctx_len) {
    if (!c || rows < 1 || c->kv_heads < 1 || c->q_heads < c->kv_heads) return 1;
    if (n_tiles > 0) {
        // a CTA per tile and kv head has an SM to itself: parts only where SMs would have nothing, at most one wave of them, of 1024 keys at least (us with 1 / 2 /
        // 4 / 8 parts: 500 tokens behind 32768, 32 / 8 heads of 128, 64 CTAs: 515 / 288 / 303 / -; 128 behind 8192: 136 / 84 / 55 / 42; 512 behind 16384, 8 / 1
        // heads: 343 / 143 / 84 / 56; 2048 behind nothing: 46 / 46 / 58 / -; 1024 behind nothing: 31 / 33 / 30 / -)
        const int64_t ctas = n_tiles * c->kv_heads, keys = c->window > 0 ? std::min<int64_t>(max_ctx_len, c->window + c->tile_tokens) : max_ctx_len;
        return rows > 65535 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(sm_count() / ctas, keys / 1024));
    }
    const int64_t seen = c->window > 0 ? std::min<int64_t>(max_ctx_len, c->window + kKv8Tokens) : max_ctx_len;
    const int64_t blocks = (seen + kKv8Tokens - 1) / kKv8Tokens, ctas = rows * pairs_of(*c), wave = places() / ctas;
    // Few rows: one wave of CTAs. Up to eight parts are merged by their cluster in the same launch; more, with a second kernel, pay where a warp keeps about a dozen
    // blocks (one sequence, 32 / 8 heads of 128, us with 8 / 16 / 32 / 55 parts: 4000 tokens 9.4 / 8.5 / 9.4 / -, 10000 15.7 / 11.7 / 11.7 / 14.0, 30000
    // 37.4 / 24.0 / 20.7 / 24.0).
    const int64_t many = std::min(wave, blocks / (12 * kWarps));
    if (many > kMostRanks) return (int)std::min<int64_t>(many, 65535);
    // Many rows: parts of about 1600 tokens, eight waves at most, since places that short sequences leave are taken by parts of long ones (32 / 8 heads of 128, us in
    // one wave / like this: 64 sequences of 512 - 8192 tokens 119 / 104, 32 of them 84 / 60, 16 38 / 36, 128 of them 209 / 189; 64 of 4000 - 32768 459 / 378, 8 of
    // them 75 / 66; 64 of 500 - 4000 68 / 64). Below 2600 tokens, and for few rows of moderate length, one wave is better (32 of 1000 - 2000 26.8 / 33.5; 8 of 512 -
    // 8192 24.1 / 29.3).
    const int64_t pieces = std::min((blocks + 40) / 100, std::max<int64_t>(1, 8 * places() / ctas));
    if (pieces > 1 && (wave <= 4 || pieces > kMostRanks)) return (int)std::min<int64_t>(pieces, 65535);
    return cluster_parts(*c, rows, blocks);
}

size_t gptrs_cuda_kv8_scratch_bytes(const gptrs_kv8_cache* c, int64_t rows, int64_t n_tiles, int splits) {
    if (!c || splits <= 1 || rows < 1 || c->kv_heads < 1 || c->q_heads < c->kv_heads || (n_tiles == 0 && in_cluster(*c, rows, splits))) return 0;
    return (size_t)rows * c->q_heads * splits * (c->dim + 2) * sizeof(float);
}

int gptrs_cuda_kv8_attention(const gptrs_kv8_cache* c, const gptrs_kv8_attention_step* s, void* stream) {
    const int rc = kv8_check(c);
    if (rc) return rc;
    GPTRS_REQUIRE(s && s->d_pool && s->d_open && s->d_page_table && s->d_length && s->d_status, "null pointer");
    GPTRS_REQUIRE(s->rows == 0 || (s->d_q && s->d_slot && s->d_ctx_len && s->d_out), "null pointer");   // (tensors without rows have none)
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
    const size_t scratch = gptrs_cuda_kv8_scratch_bytes(c, s->rows, s->n_tiles, s->splits);
    GPTRS_REQUIRE(scratch == 0 || (s->d_scratch && s->scratch_bytes >= scratch), "scratch is too small");
    if (s->rows == 0) return GPTRS_OK;
    // (a CTA has read its rows' queries of its heads before it or the merge writes there, and nobody else reads those)
    const char *q = static_cast<const char*>(s->d_q), *out = static_cast<const char*>(s->d_out);
    GPTRS_REQUIRE((q == out && p.ldq == width) || out >= q + 2 * ((s->rows - 1) * p.ldq + width) || q >= out + 2 * s->rows * width, "the output lies in rows of other queries");
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
    p.clustered = in_cluster(*c, s->rows, s->splits);
    p.tile_row = s->d_tile_row; p.tile_rows = s->d_tile_rows; p.n_tiles = (int)s->n_tiles; p.tile_tokens = c->tile_tokens;
    if (p.n_tiles > 0 && p.splits == 1 && rows_one_by_one(*c, s->rows, s->n_tiles, p.max_len)) {
        p.one_by_one = 1;
        p.clustered = 1;
        p.splits = cluster_parts(*c, s->rows, seen);
        p.chunk_blocks = std::max(1, ceil_div(seen, p.splits));
        return c->dim == 64 ? launch_attention<64>(p, as_stream(stream)) : launch_attention<128>(p, as_stream(stream));
    }
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
