// Append to the 8-bit cache (norm and rotation of queries and keys on the way), and reading tokens back.
//
// gptrs_cuda_kv8_append: a CTA takes the rows of a run that fall into one block (16 tokens) x one kv head with its query heads; it finds them from the last
// of these rows, which lies in the 16 rows (of short lists, the one row) that it looks at. Queries go by eight pairs a lane, with the products of gains and
// angles made once per row; keys and values by four. A block is written once, by the CTA with its last token: the largest magnitude over the CTA, then the
// bytes in order in shared memory; for runs of one row (decode steps) with the rows in front of it in its block, from the open rows.
// What bounds it is latency: of loads that depend on each other (slot and position; angles; open rows), so keys, values, the first queries and the angles
// (kept in shared memory) are asked for before anything is computed, and of the arithmetic behind them. 64 single tokens, 32 / 8 heads of 128: 4.4 us; six
// prompts of 925 to 2777 tokens (11104 rows), 16 / 4 heads, three axes: 58.6 us (125 MB, 33 % of the copy bandwidth; 38.6 us without the queries and the blocks;
// a warp instruction per scheduler in 44 % of the cycles, four CTAs an SM). Measured and left: CTAs that stay and fetch ahead into L2 (62.9), CTAs for queries
// and for keys apart (65.1).
#include <algorithm>

#include "kv8_cache.cuh"
#include "qk_rotate.cuh"

namespace gptrs {
namespace {

constexpr int kThreads = 128;

struct AppendParams {
    QkRotation r;
    int rotates;
    const __nv_bfloat16* qkv;
    long long ld;
    const int *positions, *slot, *run_first, *run_last, *table;
    long long max_pages, n_pages, n_slots;
    unsigned char* pool;
    __nv_bfloat16* open;
    __nv_bfloat16* q;
    int* status;
    int rows, q_heads, kv_heads, group;
    int tokens;   // of a sequence: positions that the table has pages for
};

// A lane's eight channels of a key or value in bf16: four of its first run, four of its second.
struct Packed {
    uint2 a, b;
    __device__ __forceinline__ void load(const __nv_bfloat16* src, int ca, int cb) { a = *reinterpret_cast<const uint2*>(src + ca); b = *reinterpret_cast<const uint2*>(src + cb); }
    __device__ __forceinline__ void store(__nv_bfloat16* dst, int ca, int cb) const { *reinterpret_cast<uint2*>(dst + ca) = a; *reinterpret_cast<uint2*>(dst + cb) = b; }
    __device__ __forceinline__ void get(float (&x)[4], float (&y)[4]) const {
        x[0] = bf16_lo(a.x); x[1] = bf16_hi(a.x); x[2] = bf16_lo(a.y); x[3] = bf16_hi(a.y);
        y[0] = bf16_lo(b.x); y[1] = bf16_hi(b.x); y[2] = bf16_lo(b.y); y[3] = bf16_hi(b.y);
    }
    __device__ __forceinline__ void set(const float (&x)[4], const float (&y)[4]) {
        a = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
        b = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    }
    // |x| of pairs as ordered whole numbers, with infinities and NaN above all finite values
    __device__ __forceinline__ uint32_t magnitude(uint32_t m) const { return __vmaxu2(__vmaxu2(abs_bits_max2(a.x, a.y), abs_bits_max2(b.x, b.y)), m); }
};

// x / scale rounded to the nearest whole number, plus 128, in the lowest byte. The quotient is what a division gives: the product with the correctly rounded
// inverse, and one correction by its exact remainder (Markstein). Adding 1.5 * 2^23 rounds it (ties to even).
__device__ __forceinline__ uint32_t biased_byte(float x, float scale, float inverse) {
    const float q = x * inverse;
    return __float_as_uint(fmaf(fmaf(-scale, q, x), inverse, q) + (12582912.f + 128.f));
}

// kTile: consecutive rows that a CTA looks at, 1 or 16. It works on the segments (rows of one run and block) whose last row is among them.
template <int kDim, int kTile>
__global__ void __launch_bounds__(kThreads, 4) kv8_append_kernel(const AppendParams p) {
    constexpr int kLanes = kDim / 8, kGroups = kThreads / kLanes, kPer = kKv8Tokens / kGroups;   // lanes of a head's row, rows at a time, tokens of a block per lane group
    constexpr int kPairs = kDim / 2;
    using Raw = RawVec<__nv_bfloat16, 4>;
    __shared__ __align__(16) unsigned char bytes[32 * kDim + 16];
    __shared__ __align__(16) float angles[2][kKv8Tokens][kPairs];   // cos, sin of the rows that are worked on
    __shared__ uint32_t largest[2][kThreads / 32];

    pdl_launch_dependents();
    pdl_wait();
    const int kv_head = blockIdx.y, tid = threadIdx.x, lane = tid / kLanes, in_group = tid % kLanes;   // lane group, lane in it
    const int row0 = blockIdx.x * kTile;
    int ca, cb;   // first channels of a lane's two runs
    pair_channels<4>(p.r, 4 * in_group, &ca, &cb);
    const bool turned = 4 * in_group < p.r.rot_half;

    auto source = [&](int row, int head) { return p.qkv + row * p.ld + (long long)head * kDim; };
    auto open_row = [&](int slot, int position, int which) {
        return p.open + (long long)slot * kv8_open_elems(p.kv_heads, kDim) + kv8_open_at(position / kKv8Tokens, p.kv_heads, kv_head, which, kDim) + position % kKv8Tokens * kDim;
    };
    // Angles of rows [from, from + n), n <= 16, to shared memory: a chain of loads (axis and position, table), all rows' at a time.
    const int my_pair = tid % kPairs, my_axis = p.rotates && p.r.pair_axis && my_pair < p.r.rot_half ? p.r.pair_axis[my_pair] : 0;
    auto fetch_angles = [&](int from, int n) {   // a thread has one pair
        if (!p.rotates || my_pair >= p.r.rot_half) return;
        constexpr int kRows = kThreads / kPairs, kSteps = kTile == 1 ? 2 : kKv8Tokens / kRows;
        const int* const at = p.r.axis_positions ? p.r.axis_positions + my_axis * p.r.axis_stride + from : p.positions + from;
        for (int k0 = tid / kPairs; k0 < n; k0 += kSteps * kRows) {
            int pos[kSteps];
#pragma unroll
            for (int i = 0; i < kSteps; ++i) pos[i] = k0 + i * kRows < n && my_axis < p.r.axes ? at[k0 + i * kRows] : -1;
            // (all loads in front of the first store or atomic, which would keep the ones behind them waiting)
            float c[kSteps], s[kSteps];
            bool bad = false;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                if (k0 + i * kRows < n && (pos[i] < 0 || pos[i] >= p.r.positions)) bad = true;
                const long long place = (pos[i] < 0 || pos[i] >= p.r.positions ? 0ll : (long long)pos[i] * p.r.rot_half) + my_pair;
                c[i] = p.r.cos[place];
                s[i] = p.r.sin[place];
            }
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int k = k0 + i * kRows;
                if (k < n) { angles[0][k][my_pair] = c[i]; angles[1][k][my_pair] = s[i]; }
            }
            if (bad) atomicExch(p.status, 2);
        }
    };
    // Norm and rotation of a query's or key's row in registers; all lanes of a warp take part. k: its place in `angles`.
    auto turn = [&](const float* gain, int k, float (&a)[4], float (&b)[4]) {
        if (!p.rotates) return;
        if (gain) {
            const float rms = rsqrtf(lane_group_sum(square_sum(a, b), kLanes) * (1.f / kDim) + p.r.eps);
            times_gain(gain, ca, cb, rms, a, b);
        }
        if (turned) {
            float c[4], s[4];
            load_vec(&angles[0][k][4 * in_group], c);
            load_vec(&angles[1][k][4 * in_group], s);
            rotate_pairs(!p.r.neighbours, a, b, c, s);
        }
    };
    auto put = [&](__nv_bfloat16* dst, const float (&a)[4], const float (&b)[4]) { store_vec(dst + ca, a); store_vec(dst + cb, b); };
    // The 16 tokens of a block, token lane + j kGroups of either kind in this thread's registers -> the page. All threads.
    auto write_block = [&](const Packed (&x)[2][kPer], int page) {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < kPer; ++j) m = x[which][j].magnitude(m);
            m = __reduce_max_sync(0xffffffffu, widest_half(m));
            if ((tid & 31) == 0) largest[which][tid >> 5] = m;
        }
        __syncthreads();
        const bool even = (lane & 1) == 0;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            uint32_t all = 0;
#pragma unroll
            for (int i = 0; i < kThreads / 32; ++i) all = max(all, largest[which][i]);
            const bool finite = all < 0x7f80u;
            const float scale = finite ? fmaxf(__fdiv_rn(__uint_as_float(all << 16), 127.f), kKv8MinScale) : __uint_as_float(0x7fc00000u);
            const float inverse = __frcp_rn(scale);
            uint32_t w[kPer][2];   // four bytes of either run
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                float v[2][4];
                x[which][j].get(v[0], v[1]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t u[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) u[k] = biased_byte(v[half][k], scale, inverse);
                    w[j][half] = finite ? __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410) : 0x80808080u;
                }
            }
            if (which == 0) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    *reinterpret_cast<uint32_t*>(bytes + kv8_key_at(lane + j * kGroups, ca)) = w[j][0];
                    *reinterpret_cast<uint32_t*>(bytes + kv8_key_at(lane + j * kGroups, cb)) = w[j][1];
                }
            } else {
                // an even and an odd token next to each other: their lane groups exchange a run, so that either has four channels of both
                uint32_t e[kPer], o[kPer];
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    const uint32_t got = __shfl_xor_sync(0xffffffffu, even ? w[j][1] : w[j][0], kLanes);
                    e[j] = even ? w[j][0] : got;
                    o[j] = even ? got : w[j][1];
                }
                const int ch = even ? ca : cb, token = lane & ~1;
                const uint32_t t0 = __byte_perm(e[0], o[0], 0x5140), t1 = __byte_perm(e[0], o[0], 0x7362);   // (channel 0, 1), (2, 3) of both tokens
                if constexpr (kPer == 2) {
                    const uint32_t u0 = __byte_perm(e[1], o[1], 0x5140), u1 = __byte_perm(e[1], o[1], 0x7362);
                    *reinterpret_cast<uint32_t*>(bytes + kv8_value_at(token, ch, kDim)) = __byte_perm(t0, u0, 0x5410);
                    *reinterpret_cast<uint32_t*>(bytes + kv8_value_at(token, ch + 1, kDim)) = __byte_perm(t0, u0, 0x7632);
                    *reinterpret_cast<uint32_t*>(bytes + kv8_value_at(token, ch + 2, kDim)) = __byte_perm(t1, u1, 0x5410);
                    *reinterpret_cast<uint32_t*>(bytes + kv8_value_at(token, ch + 3, kDim)) = __byte_perm(t1, u1, 0x7632);
                } else {
                    *reinterpret_cast<uint16_t*>(bytes + kv8_value_at(token, ch, kDim)) = (uint16_t)t0;
                    *reinterpret_cast<uint16_t*>(bytes + kv8_value_at(token, ch + 1, kDim)) = (uint16_t)(t0 >> 16);
                    *reinterpret_cast<uint16_t*>(bytes + kv8_value_at(token, ch + 2, kDim)) = (uint16_t)t1;
                    *reinterpret_cast<uint16_t*>(bytes + kv8_value_at(token, ch + 3, kDim)) = (uint16_t)(t1 >> 16);
                }
            }
            if (tid == 0) reinterpret_cast<float*>(bytes + 32 * kDim)[which] = scale;
        }
        if (tid < 2) reinterpret_cast<float*>(bytes + 32 * kDim)[2 + tid] = 0.f;
        __syncthreads();
        if (page >= 0) {
            uint4* dst = reinterpret_cast<uint4*>(p.pool + ((long long)page * p.kv_heads + kv_head) * kv8_block_bytes(kDim));
            for (int i = tid; i < 2 * kDim + 1; i += kThreads) dst[i] = reinterpret_cast<const uint4*>(bytes)[i];
        }
    };
    // a key as it comes -> normed, rotated, rounded. k: its place in `angles`.
    auto finish_key = [&](Packed x, int k) {
        float a[4], b[4];
        x.get(a, b);
        turn(p.r.k_gain, k, a, b);
        if (p.rotates) x.set(a, b);
        return x;
    };
    auto page_of = [&](int slot, int block) { return kv8_page(p.table, slot, p.max_pages, block, p.n_pages, p.status); };

    if (kTile == 1) {
        // ---- a run of one row: everything is asked for at once ---------------------------------------------------------------------------------
        Raw qa, qb;
        Packed own = {};
        if (lane < p.group) { const __nv_bfloat16* src = source(row0, kv_head * p.group + lane); qa.load(src + ca); qb.load(src + cb); }
        if (lane < 2) own.load(source(row0, p.q_heads + lane * p.kv_heads + kv_head), ca, cb);   // lane group 0 has the key, 1 the value
        const int slot = p.slot[row0], position = p.positions[row0], first = p.run_first[row0], last = p.run_last[row0];
        if (slot < 0) return;
        if (first == row0 && last == row0 && slot < p.n_slots && position >= 0 && position < p.tokens) {
            fetch_angles(row0, 1);
            const bool completes = position % kKv8Tokens == kKv8Tokens - 1;
            Packed x[2][kPer];
            int page = -1;
            if (completes) {
#pragma unroll
                for (int which = 0; which < 2; ++which)
#pragma unroll
                    for (int j = 0; j < kPer; ++j) x[which][j].load(open_row(slot, position - (kKv8Tokens - 1) + lane + j * kGroups, which), ca, cb);
                page = page_of(slot, position / kKv8Tokens);
            }
            __syncthreads();
            for (int h0 = 0; h0 < p.group; h0 += kGroups) {
                const int h = h0 + lane;
                float a[4] = {}, b[4] = {};
                if (h0 > 0 && h < p.group) { const __nv_bfloat16* src = source(row0, kv_head * p.group + h); qa.load(src + ca); qb.load(src + cb); }
                if (h < p.group) { qa.get(a); qb.get(b); }
                turn(p.r.q_gain, 0, a, b);
                if (h < p.group) put(p.q + ((long long)row0 * p.q_heads + kv_head * p.group + h) * kDim, a, b);
            }
            const Packed key = finish_key(own, 0);
            if (lane == 0) own = key;
            if (completes) {   // by way of shared memory to the threads that have the block's last token
                __nv_bfloat16* const last_token = reinterpret_cast<__nv_bfloat16*>(bytes);
                if (lane < 2) own.store(last_token + lane * kDim, ca, cb);
                __syncthreads();
                if (lane + (kPer - 1) * kGroups == kKv8Tokens - 1) {
                    x[0][kPer - 1].load(last_token, ca, cb);
                    x[1][kPer - 1].load(last_token + kDim, ca, cb);
                }
                write_block(x, page);   // (its first barrier stands between this and its writing over last_token)
            }
            if (lane < 2) own.store(open_row(slot, position, lane), ca, cb);
            return;
        }
    }

    // ---- segments --------------------------------------------------------------------------------------------------------------------------------
    // lane i of every warp: row row0 + i
    int slot_i = -1, position_i = 0, first_i = 0, last_i = 0;
    const int row_i = row0 + (tid & 31);
    if ((tid & 31) < kTile && row_i < p.rows) { slot_i = p.slot[row_i]; position_i = p.positions[row_i]; first_i = p.run_first[row_i]; last_i = p.run_last[row_i]; }
    bool ends = false;
    if (slot_i >= 0) {
        if (slot_i >= p.n_slots || first_i < 0 || first_i > row_i || last_i < row_i || last_i >= p.rows || position_i < row_i - first_i ||
            position_i >= p.tokens)   // (rows in front of the table's end, which is a block's, go on)
            atomicExch(p.status, 2);
        else
            ends = position_i % kKv8Tokens == kKv8Tokens - 1 || row_i == last_i;
    }
    const uint32_t segments = __ballot_sync(0xffffffffu, ends);
    for (uint32_t todo = segments; todo; todo &= todo - 1) {
        const int from = __ffs(todo) - 1, row_b = row0 + from;
        if (kTile > 1 && __popc(segments & ((1u << from) - 1u)) % gridDim.z != blockIdx.z) continue;   // another CTA's
        const int slot = __shfl_sync(0xffffffffu, slot_i, from), position = __shfl_sync(0xffffffffu, position_i, from), first = __shfl_sync(0xffffffffu, first_i, from),
                  last = __shfl_sync(0xffffffffu, last_i, from);
        const int block = position / kKv8Tokens, token_b = position % kKv8Tokens, row_a = max(first, row_b - token_b), token_a = token_b - (row_b - row_a), n = row_b - row_a + 1;
        const int start = position - (row_b - first), end = (int)min((long long)position + (last - row_b), p.tokens - 1ll);   // of the run
        const bool continued = start % kKv8Tokens != 0, completes = token_b == kKv8Tokens - 1;
        // keys and values of tokens lane + j kGroups: new rows, or open ones of the run's first block
        Packed x[2][kPer] = {};
#pragma unroll
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const int token = lane + j * kGroups;
                if (token >= token_a && token <= token_b) x[which][j].load(source(row_a + token - token_a, p.q_heads + which * p.kv_heads + kv_head), ca, cb);
                else if (completes) x[which][j].load(open_row(slot, block * kKv8Tokens + token, which), ca, cb);
            }
        // queries: eight pairs a lane, so that dim / 16 lanes have a row (one of 16) and take its heads, kBatch on their way
        constexpr int kQLanes = kDim / 16, kAtOnce = kThreads / kQLanes / kKv8Tokens, kBatch = 4;
        const int q_lane = tid % kQLanes, q_row = tid / kQLanes % kKv8Tokens, q_first = tid / kQLanes / kKv8Tokens;
        const bool q_live = q_row < n, q_turned = 8 * q_lane < p.r.rot_half;
        int qca, qcb;
        pair_channels<8>(p.r, 8 * q_lane, &qca, &qcb);
        const __nv_bfloat16* const q_src = source(row_a + min(q_row, n - 1), kv_head * p.group);
        __nv_bfloat16* const q_dst = p.q + ((long long)(row_a + min(q_row, n - 1)) * p.q_heads + kv_head * p.group) * kDim;
        RawVec<__nv_bfloat16, 8> qa[kBatch], qb[kBatch];
        auto load_queries = [&](int h0) {
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int h = h0 + j * kAtOnce + q_first;
                if (q_live && h < p.group) { qa[j].load(q_src + h * kDim + qca); qb[j].load(q_src + h * kDim + qcb); }
            }
        };
        load_queries(0);
        fetch_angles(row_a, n);
        const int page = completes ? page_of(slot, block) : -1;
        __syncthreads();
        {
            const bool apart = !p.r.neighbours;
            Turn<8> t;
            if (p.rotates && apart) t.set(p.r.q_gain, qca, qcb, q_turned, &angles[0][min(q_row, n - 1)][8 * q_lane], &angles[1][min(q_row, n - 1)][8 * q_lane]);
            for (int h0 = 0; h0 < p.group; h0 += kBatch * kAtOnce) {
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    if (h0 + j * kAtOnce >= p.group) break;
                    const int h = h0 + j * kAtOnce + q_first;
                    const bool live = q_live && h < p.group;
                    float a[8] = {}, b[8] = {};
                    if (live) { qa[j].get(a); qb[j].get(b); }
                    if (p.rotates) {
                        const float rms = p.r.q_gain ? rsqrtf(lane_group_sum(square_sum2(a, b), kQLanes) * (1.f / kDim) + p.r.eps) : 1.f;
                        if (apart) {
                            t.apply(a, b, rms, q_turned);
                        } else {
                            if (p.r.q_gain) times_gain(p.r.q_gain, qca, qcb, rms, a, b);
                            if (q_turned) {
                                float c[8], s[8];
                                load_vec(&angles[0][min(q_row, n - 1)][8 * q_lane], c);
                                load_vec(&angles[1][min(q_row, n - 1)][8 * q_lane], s);
                                rotate_pairs(false, a, b, c, s);
                            }
                        }
                    }
                    if (live) { store_vec(q_dst + h * kDim + qca, a); store_vec(q_dst + h * kDim + qcb, b); }
                }
                if (h0 + kBatch * kAtOnce < p.group) load_queries(h0 + kBatch * kAtOnce);
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {   // rows of earlier calls are as they are to be
            const int token = lane + j * kGroups;
            const bool fresh = token >= token_a && token <= token_b;
            const Packed key = finish_key(x[0][j], fresh ? token - token_a : 0);
            if (fresh) x[0][j] = key;
        }
        if (completes) write_block(x, page);
        // The rows of the run's last two blocks stay as they are, in the open rows. A run that goes on from the middle of a block and ends two blocks or more
        // further on would have them written over rows of that block that another CTA may not have read yet: there the CTA with the run's first segment, which
        // has read them (all its threads have, in front of write_block's barriers), does it for all.
        const bool by_first = continued && end / kKv8Tokens >= start / kKv8Tokens + 2;
        if (!by_first && block >= end / kKv8Tokens - 1) {
#pragma unroll
            for (int which = 0; which < 2; ++which)
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    const int token = lane + j * kGroups;
                    if (token >= token_a && token <= token_b) x[which][j].store(open_row(slot, block * kKv8Tokens + token, which), ca, cb);
                }
        }
        __syncthreads();   // `bytes`, `largest` and `angles` may be written again
        if (by_first && row_a == first) {
            for (int b0 = (end / kKv8Tokens - 1) * kKv8Tokens; b0 <= end; b0 += kKv8Tokens) {
                const int count = min(kKv8Tokens, end - b0 + 1), from_row = first + (b0 - start);
                fetch_angles(from_row, count);
                __syncthreads();
#pragma unroll
                for (int which = 0; which < 2; ++which)
#pragma unroll
                    for (int j = 0; j < kPer; ++j) {
                        const int token = lane + j * kGroups;
                        Packed row = {};
                        if (token < count) row.load(source(from_row + token, p.q_heads + which * p.kv_heads + kv_head), ca, cb);
                        if (which == 0) row = finish_key(row, min(token, count - 1));
                        if (token < count) row.store(open_row(slot, b0 + token, which), ca, cb);
                    }
                __syncthreads();
            }
        }
    }
}

struct GatherParams {
    const unsigned char* pool;
    const __nv_bfloat16* open;
    const int *table, *slot, *positions, *length;
    long long max_pages, n_pages, n_slots;
    void *k, *v;
    int* status;
    int rows, kv_heads;
};
// eight channels of a token per thread; the CTAs of neighbouring tokens read the same lines
template <int kDim, typename T>
__global__ void __launch_bounds__(kThreads) kv8_gather_kernel(const GatherParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const long long item = (long long)blockIdx.x * kThreads + threadIdx.x;
    const int per_row = p.kv_heads * (kDim / 8);
    const long long row = item / per_row;
    if (row >= p.rows) return;
    const int head = (int)(item % per_row) / (kDim / 8), d0 = (int)(item % (kDim / 8)) * 8;
    const int slot = p.slot[row], position = p.positions[row];
    float k[8] = {}, v[8] = {};
    bool found = slot >= 0 && slot < p.n_slots && position >= 0 && position / kKv8Tokens < p.max_pages && position < p.length[slot >= 0 && slot < p.n_slots ? slot : 0];
    if (found) {
        const int block = position / kKv8Tokens, token = position % kKv8Tokens;
        if (block < p.length[slot] / kKv8Tokens) {
            const int page = kv8_page(p.table, slot, p.max_pages, block, p.n_pages, p.status);
            found = page >= 0;
            if (found) {
                const unsigned char* b = p.pool + ((long long)page * p.kv_heads + head) * kv8_block_bytes(kDim);
                const float2 scale = *reinterpret_cast<const float2*>(b + 32 * kDim);
                const uint2 kb = *reinterpret_cast<const uint2*>(b + kv8_key_at(token, d0));
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    k[i] = (float)((int)(((i < 4 ? kb.x : kb.y) >> (8 * (i & 3))) & 255) - 128) * scale.x;
                    v[i] = (float)((int)b[kv8_value_at(token, d0 + i, kDim)] - 128) * scale.y;
                }
            }
        } else {
            const __nv_bfloat16* src = p.open + (long long)slot * kv8_open_elems(p.kv_heads, kDim) + kv8_open_at(block, p.kv_heads, head, 0, kDim) + token * kDim + d0;
#pragma unroll
            for (int i = 0; i < 8; ++i) { k[i] = __bfloat162float(src[i]); v[i] = __bfloat162float(src[kKv8Tokens * kDim + i]); }
        }
    }
    if (!found) atomicExch(p.status, 2);
    const long long at = (row * p.kv_heads + head) * kDim + d0;
    float (*const kk)[4] = reinterpret_cast<float(*)[4]>(k), (*const vv)[4] = reinterpret_cast<float(*)[4]>(v);
    store_vec(static_cast<T*>(p.k) + at, kk[0]);
    store_vec(static_cast<T*>(p.k) + at + 4, kk[1]);
    store_vec(static_cast<T*>(p.v) + at, vv[0]);
    store_vec(static_cast<T*>(p.v) + at + 4, vv[1]);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int kv8_check(const gptrs_kv8_cache* c) {
    GPTRS_REQUIRE(c, "null pointer");
    gptrs_kv8_cache want = *c;
    const int rc = gptrs_cuda_kv8_layout(&want);
    if (rc) return rc;
    GPTRS_REQUIRE(c->block_bytes == want.block_bytes && c->page_bytes == want.page_bytes && c->tile_tokens == want.tile_tokens, "call gptrs_cuda_kv8_layout first");
    return GPTRS_OK;
}

}  // namespace gptrs

using namespace gptrs;

extern "C" {

int gptrs_cuda_kv8_layout(gptrs_kv8_cache* c) {
    GPTRS_REQUIRE(c, "null pointer");
    GPTRS_REQUIRE(c->q_heads > 0 && c->kv_heads > 0 && c->q_heads % c->kv_heads == 0 && c->kv_heads <= 65535, "bad head counts");
    GPTRS_REQUIRE(c->window >= 0, "bad window");
    if (c->dim != 64 && c->dim != 128) return fail(GPTRS_UNIMPLEMENTED, "the 8-bit cache takes heads of 64 and 128 channels");
    const int group = c->q_heads / c->kv_heads;
    if (group > 64) return fail(GPTRS_UNIMPLEMENTED, "the 8-bit cache takes up to 64 query heads per kv head");
    if (!(c->scale > 0.f)) {
        GPTRS_REQUIRE(c->scale == 0.f, "the scale of the scores is positive, or 0 for 1 / sqrt(dim)");
        c->scale = 1.f / sqrtf((float)c->dim);
    }
    c->tile_tokens = 2 * (128 / group);
    c->block_bytes = kv8_block_bytes(c->dim);
    c->page_bytes = c->block_bytes * c->kv_heads;
    c->open_bytes = 2 * kv8_open_elems(c->kv_heads, c->dim);
    return GPTRS_OK;
}

int gptrs_cuda_kv8_append(const gptrs_kv8_cache* c, const gptrs_kv8_append_step* s, void* stream) {
    const int rc = kv8_check(c);
    if (rc) return rc;
    GPTRS_REQUIRE(s && s->d_page_table && s->d_pool && s->d_open && s->d_status, "null pointer");
    GPTRS_REQUIRE(s->rows == 0 || (s->d_qkv && s->d_positions && s->d_slot && s->d_run_first && s->d_run_last && s->d_q), "null pointer");   // (tensors without rows have none)
    GPTRS_REQUIRE(s->rows >= 0 && s->rows <= 0x3fffffff, "bad row count");
    GPTRS_REQUIRE(s->max_pages >= 1 && s->n_pages >= 1 && s->n_slots >= 1, "empty cache");
    AppendParams p = {};
    const int64_t width = (int64_t)(c->q_heads + 2 * c->kv_heads) * c->dim;
    p.ld = s->ld ? s->ld : width;
    GPTRS_REQUIRE(p.ld >= width && p.ld % 8 == 0, "rows overlap, or do not start at multiples of 16 bytes");
    GPTRS_REQUIRE(aligned16(s->d_qkv) && aligned16(s->d_pool) && aligned16(s->d_open) && aligned16(s->d_q), "pointers must be 16-byte aligned");
    if (s->rotation) {
        const int rr = qk_rotation_of(*s->rotation, s->rows, &p.r);
        if (rr) return rr;
        GPTRS_REQUIRE(p.r.q_heads == c->q_heads && p.r.kv_heads == c->kv_heads && p.r.dim == c->dim, "the rotation is of other heads");
        if (p.r.rot_half % 8) return fail(GPTRS_UNIMPLEMENTED, "the append takes rotations of a multiple of 8 pairs");
        GPTRS_REQUIRE(aligned16(p.r.cos) && aligned16(p.r.sin) && aligned16(p.r.q_gain) && aligned16(p.r.k_gain), "tables and gains must be 16-byte aligned");
        p.rotates = 1;
    } else {
        p.r.dim = c->dim;
    }
    if (s->rows == 0) return GPTRS_OK;
    const char *in = static_cast<const char*>(s->d_qkv), *q = static_cast<const char*>(s->d_q);
    GPTRS_REQUIRE(q >= in + 2 * ((s->rows - 1) * p.ld + width) || in >= q + 2 * s->rows * c->q_heads * c->dim, "queries go into rows that other heads are still read from");
    p.qkv = static_cast<const __nv_bfloat16*>(s->d_qkv);
    p.positions = s->d_positions; p.slot = s->d_slot; p.run_first = s->d_run_first; p.run_last = s->d_run_last; p.table = s->d_page_table;
    p.max_pages = s->max_pages; p.n_pages = s->n_pages; p.n_slots = s->n_slots;
    p.pool = static_cast<unsigned char*>(s->d_pool);
    p.open = static_cast<__nv_bfloat16*>(s->d_open);
    p.q = static_cast<__nv_bfloat16*>(s->d_q);
    p.status = s->d_status;
    p.rows = (int)s->rows; p.q_heads = c->q_heads; p.kv_heads = c->kv_heads; p.group = c->q_heads / c->kv_heads;
    p.tokens = (int)std::min<int64_t>(std::min<int64_t>(s->max_pages, 0x7fffffff) * kKv8Tokens, 0x7fffffff - kKv8Tokens + 1);   // a whole number of blocks
    // A CTA per row and kv head for lists that are short or may be single tokens, else per 16 rows: a prompt has one segment in them. Where they are single tokens
    // after all, four CTAs deal the segments among them, as long as the three that find nothing cost little. us, 32 / 8 heads of 128, per row / per 16 / four
    // for 16: 64 single tokens 4.2 / 64 / 20, 512 14 / 66 / 44; a prompt of 256 10.9 / 7.8 / 8.4, of 1000 23 / 10.5 / 11.2, of 4 x 1000 62 / 41 / 42, six of
    // 925 to 2777 - / 104 / 119, 6 x 2777 - / 146 / 176.
    const bool few = s->rows <= 256 || s->rows <= s->n_slots;
    const dim3 grid((unsigned)ceil_div(s->rows, few ? 1 : kKv8Tokens), (unsigned)c->kv_heads, few || s->rows > 4096 ? 1u : 4u);
    auto kernel = c->dim == 64 ? (few ? kv8_append_kernel<64, 1> : kv8_append_kernel<64, 16>) : (few ? kv8_append_kernel<128, 1> : kv8_append_kernel<128, 16>);
    return launch_kernel(kernel, grid, dim3(kThreads), 0, as_stream(stream), 1, p);
}

int gptrs_cuda_kv8_gather(const gptrs_kv8_cache* c, const void* d_pool, int64_t n_pages, const void* d_open, int64_t n_slots, const int32_t* d_page_table,
                          int64_t max_pages, const int32_t* d_slot, const int32_t* d_positions, const int32_t* d_length, int dtype, void* d_k,
                          void* d_v, int32_t* d_status, int64_t rows, void* stream) {
    const int rc = kv8_check(c);
    if (rc) return rc;
    GPTRS_REQUIRE(d_pool && d_open && d_page_table && d_length && d_status, "null pointer");
    GPTRS_REQUIRE(rows == 0 || (d_slot && d_positions && d_k && d_v), "null pointer");
    GPTRS_REQUIRE(dtype == GPTRS_BF16 || dtype == GPTRS_F32, "keys and values come back in bf16 or f32");
    GPTRS_REQUIRE(rows >= 0 && rows <= 0x3fffffff, "bad row count");
    GPTRS_REQUIRE(max_pages >= 1 && n_pages >= 1 && n_slots >= 1, "empty cache");
    GPTRS_REQUIRE(aligned16(d_pool) && aligned16(d_open) && aligned16(d_k) && aligned16(d_v), "pointers must be 16-byte aligned");
    if (rows == 0) return GPTRS_OK;
    GatherParams p = {static_cast<const unsigned char*>(d_pool), static_cast<const __nv_bfloat16*>(d_open), d_page_table, d_slot, d_positions, d_length,
                      (long long)max_pages, (long long)n_pages, (long long)n_slots, d_k, d_v, d_status, (int)rows, c->kv_heads};
    const int64_t ctas = (rows * c->kv_heads * (c->dim / 8) + kThreads - 1) / kThreads;
    GPTRS_REQUIRE(ctas <= 0x7fffffff, "grid too large");
    const dim3 grid((unsigned)ctas), block(kThreads);
    if (c->dim == 64)
        return dtype == GPTRS_F32 ? launch_kernel(kv8_gather_kernel<64, float>, grid, block, 0, as_stream(stream), 1, p)
                                  : launch_kernel(kv8_gather_kernel<64, __nv_bfloat16>, grid, block, 0, as_stream(stream), 1, p);
    return dtype == GPTRS_F32 ? launch_kernel(kv8_gather_kernel<128, float>, grid, block, 0, as_stream(stream), 1, p)
                              : launch_kernel(kv8_gather_kernel<128, __nv_bfloat16>, grid, block, 0, as_stream(stream), 1, p);
}

}  // extern "C"
