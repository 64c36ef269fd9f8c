// Norms of queries and keys per head and their rotation in one pass, positions on several axes (see qk_rotate.cuh).
//
// With gains g and angles (c, s), out_a = x_a r g_a c - x_b r g_b s and out_b = x_b r g_b c + x_a r g_a s, r = 1 / rms of the head. Every value is read and
// written once; sums of squares are f32, the result is rounded once. 9001 rows of 32 + 8 + 8 heads of 128 in bf16 on three axes: 43.4 us (28.2 at the copy
// bandwidth for the queries and keys alone; a plain copy of the same bytes takes 35). In place only queries and keys are written; the ring reads the
// values beside them all the same, since a row is one piece.
//
// Three kernels. qk_norm_rope_ring_kernel streams rows through shared memory. qk_norm_rope_wide_kernel holds them in registers: a warp takes some heads of one
// kind (queries, keys, values) of a row, a group of its lanes a head at a time, kVec pairs a lane, so that loads and stores are 16 bytes a lane; the four
// products of gains and angles are made once for the warp's heads, and the next head is on its way while one is worked on. What holds it up is that little is
// on its way beside the instructions. us, 32 / 8 heads of 128, ring / wide: bf16, three axes, 1 row 3.3 / 3.4, 148 3.4 / 4.2, 2000 13.4 / 20.6, 9001 43.4 /
// 69.2; f32, one axis, 1 row 3.3 / 2.5, 64 3.6 / 3.0, 148 3.8 / 4.2, 2000 22.3 / 25.1: so the ring is taken but for few rows of f32. Sizes that do not come
// in pieces of four go pair by pair (up to 512 channels).
#include <algorithm>

#include "qk_rotate.cuh"

namespace gptrs {

int qk_rotation_of(const gptrs_qk_rotation& r, int64_t rows, QkRotation* out) {
    GPTRS_REQUIRE(r.q_heads > 0 && r.kv_heads > 0, "bad head counts");
    GPTRS_REQUIRE(r.dim >= 2 && r.dim % 2 == 0 && r.dim <= 512, "dim is even and at most 512");
    GPTRS_REQUIRE(r.rot_half >= 0 && 2 * r.rot_half <= r.dim, "at most dim / 2 pairs");
    GPTRS_REQUIRE(r.pairs == GPTRS_PAIRS_HALVES || r.pairs == GPTRS_PAIRS_NEIGHBOURS, "unknown pairing");
    GPTRS_REQUIRE((r.d_q_gain == nullptr) == (r.d_k_gain == nullptr), "gains of queries and keys come together");
    GPTRS_REQUIRE(r.rot_half == 0 || (r.d_cos && r.d_sin && r.positions > 0), "tables are missing");
    GPTRS_REQUIRE(r.axes >= 0 && r.axes <= 255, "bad number of axes");
    GPTRS_REQUIRE(r.axes <= 1 || ((r.d_axis_positions || rows == 0) && r.d_pair_axis), "several axes need their positions and the axis of every pair");
    GPTRS_REQUIRE(r.axis_stride == 0 || r.axis_stride >= rows, "axis_stride is shorter than the rows");
    *out = QkRotation{r.q_heads, r.kv_heads, r.dim, r.rot_half, r.pairs == GPTRS_PAIRS_NEIGHBOURS, r.axes > 1 ? r.axes : 1, r.eps, r.d_q_gain, r.d_k_gain, r.d_cos,
                      r.d_sin, (long long)r.positions, (long long)(r.axis_stride ? r.axis_stride : rows), r.d_axis_positions, r.d_pair_axis};
    return GPTRS_OK;
}

namespace {

struct NormRopeParams {
    QkRotation r;
    const void* in;
    void* out;
    long long ld_in, ld_out;
    const int* positions;
    int* status;
    int heads;    // of the rows that are worked on: without the values where they stay in place
    int copies;   // values are copied
    int lanes;    // of a head
    // warps' work: rows x parts (of queries, of keys, of values) of part_heads heads
    long long items;
    int parts, q_parts, k_parts, part_heads;
};
constexpr int kThreads = 256;
// cos and sin of the kVec pairs from `first` on at a row; axes: the pairs' axes, a byte each
template <int kVec>
__device__ __forceinline__ void lane_angles(const NormRopeParams& p, int row, int first, const uint32_t (&axes)[kVec / 4], float (&c)[kVec], float (&s)[kVec]) {
    const QkRotation& r = p.r;
    bool bad = false;   // (reported behind the loads: an atomic in between would keep the next ones waiting)
    auto place = [&](int axis) {
        long long pos = -1;
        if (axis < r.axes) pos = r.axis_positions ? r.axis_positions[axis * r.axis_stride + row] : p.positions[row];
        if (pos < 0 || pos >= r.positions) { bad = true; pos = 0; }
        return pos * r.rot_half + first;
    };
#pragma unroll
    for (int i = 0; i < kVec / 4; ++i) {
        const int axis = axes[i] & 255;
        if (axes[i] == axis * 0x01010101u) {
            const long long at = place(axis) + 4 * i;
            const float4 x = *reinterpret_cast<const float4*>(r.cos + at), y = *reinterpret_cast<const float4*>(r.sin + at);
            c[4 * i] = x.x; c[4 * i + 1] = x.y; c[4 * i + 2] = x.z; c[4 * i + 3] = x.w;
            s[4 * i] = y.x; s[4 * i + 1] = y.y; s[4 * i + 2] = y.z; s[4 * i + 3] = y.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const long long at = place((axes[i] >> (8 * k)) & 255) + 4 * i + k;
                c[4 * i + k] = r.cos[at];
                s[4 * i + k] = r.sin[at];
            }
        }
    }
    if (bad) atomicExch(p.status, 2);
}

constexpr int kAhead = 2;   // heads of a lane group on their way

// Pairs apart: first channels in a, second ones in b. Neighbours: a and b hold pairs each; a lane's channels of a and of b are worked on in the same way,
// with (a0, a2, ..), (a1, a3, ..) in the place of a, b.
template <typename T, int kVec, bool kNeighbours>
__global__ void __launch_bounds__(kThreads, 2) qk_norm_rope_wide_kernel(const NormRopeParams p) {
    constexpr int kHalf = kVec / 2;
    pdl_launch_dependents();
    pdl_wait();
    const QkRotation& r = p.r;
    const int lanes = p.lanes, lane = threadIdx.x & (lanes - 1), group = (threadIdx.x & 31) / lanes, n_groups = 32 / lanes;
    const int first = lane * kVec;             // pair
    const bool some = 2 * first < r.dim, turned = first < r.rot_half;
    int ca, cb;
    pair_channels<kVec>(r, first, &ca, &cb);
    uint32_t axes[kVec / 4] = {};
    if (turned && r.pair_axis) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) axes[k / 4] |= (uint32_t)r.pair_axis[first + k] << (8 * (k & 3));
    }
    const float width = 1.f / r.dim;
    const long long warps = (long long)gridDim.x * (kThreads / 32);
    for (long long item = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); item < p.items; item += warps) {
        const int row = (int)(item / p.parts), part = (int)(item % p.parts);
        const int kind = part < p.q_parts ? 0 : part < p.q_parts + p.k_parts ? 1 : 2;
        const int begin = kind == 0 ? part * p.part_heads : r.q_heads + (kind == 1 ? part - p.q_parts : part - p.q_parts - p.k_parts) * p.part_heads + (kind == 2 ? r.kv_heads : 0);
        const int end = min(begin + p.part_heads, kind == 0 ? r.q_heads : r.q_heads + kind * r.kv_heads);
        const T* in = static_cast<const T*>(p.in) + row * p.ld_in + ca;
        T* out = static_cast<T*>(p.out) + row * p.ld_out + ca;
        const int b_off = cb - ca;
        RawVec<T, kVec> ra[kAhead], rb[kAhead];
        auto load = [&](int j, int h) {
            if (h < end && some) { ra[j].load(in + h * r.dim); rb[j].load(in + h * r.dim + b_off); }
        };
#pragma unroll
        for (int j = 0; j < kAhead; ++j) load(j, begin + group + j * n_groups);
        if (kind == 2) {   // values are copied
            for (int h0 = begin + group; h0 < end; h0 += kAhead * n_groups) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    const int h = h0 + j * n_groups;
                    if (h < end && some) { ra[j].store(out + h * r.dim); rb[j].store(out + h * r.dim + b_off); }
                    load(j, h + kAhead * n_groups);
                }
            }
            continue;
        }
        // gains times angles, two pairs at a time
        uint64_t ac[kHalf], bs[kHalf], bc[kHalf], as[kHalf];
        {
            float c[kVec], s[kVec], ga[kVec], gb[kVec];
#pragma unroll
            for (int k = 0; k < kVec; ++k) { c[k] = 1.f; s[k] = 0.f; ga[k] = gb[k] = 1.f; }
            if (turned) lane_angles<kVec>(p, row, first, axes, c, s);
            const float* gain = kind ? r.k_gain : r.q_gain;
            if (gain && some) { load_vec(gain + ca, ga); load_vec(gain + cb, gb); }
            if (kNeighbours) {
                float x[kVec], y[kVec];
#pragma unroll
                for (int k = 0; k < kHalf; ++k) { x[k] = ga[2 * k]; y[k] = ga[2 * k + 1]; x[kHalf + k] = gb[2 * k]; y[kHalf + k] = gb[2 * k + 1]; }
#pragma unroll
                for (int k = 0; k < kVec; ++k) { ga[k] = x[k]; gb[k] = y[k]; }
            }
#pragma unroll
            for (int k = 0; k < kHalf; ++k) {
                const uint64_t c2 = pair_of(c[2 * k], c[2 * k + 1]), s2 = pair_of(s[2 * k], s[2 * k + 1]);
                const uint64_t a2 = pair_of(ga[2 * k], ga[2 * k + 1]), b2 = pair_of(gb[2 * k], gb[2 * k + 1]);
                ac[k] = mul2(a2, c2); as[k] = mul2(a2, s2); bc[k] = mul2(b2, c2); bs[k] = mul2(b2, s2) ^ 0x8000000080000000ull;
            }
        }
        for (int h0 = begin; h0 < end; h0 += kAhead * n_groups) {
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            if (h0 + j * n_groups >= end) break;
            const int h = h0 + j * n_groups + group, at = h * r.dim;
            const bool live = h < end && some;
            float xa[kVec], xb[kVec];
            ra[j].get(xa);
            rb[j].get(xb);
            load(j, h + kAhead * n_groups);
            uint64_t a[kHalf], b[kHalf], sum = 0;
#pragma unroll
            for (int k = 0; k < kHalf; ++k) {
                a[k] = kNeighbours ? (k < kHalf / 2 ? pair_of(xa[4 * k], xa[4 * k + 2]) : pair_of(xb[4 * k - kVec], xb[4 * k - kVec + 2])) : pair_of(xa[2 * k], xa[2 * k + 1]);
                b[k] = kNeighbours ? (k < kHalf / 2 ? pair_of(xa[4 * k + 1], xa[4 * k + 3]) : pair_of(xb[4 * k - kVec + 1], xb[4 * k - kVec + 3])) : pair_of(xb[2 * k], xb[2 * k + 1]);
                sum = fma2(a[k], a[k], fma2(b[k], b[k], sum));
            }
            float rms = 1.f;
            if (r.q_gain) {   // every lane takes part in the sums, groups past the last head included
                const float2 both = split(sum);
                rms = rsqrtf(lane_group_sum(live ? both.x + both.y : 0.f, lanes) * width + r.eps);
            }
            const uint64_t rms2 = pair_of(rms, rms);
#pragma unroll
            for (int k = 0; k < kHalf; ++k) {
                const uint64_t ar = mul2(a[k], rms2), br = mul2(b[k], rms2);
                const float2 x = split(turned ? fma2(ar, ac[k], mul2(br, bs[k])) : mul2(ar, ac[k])), y = split(turned ? fma2(br, bc[k], mul2(ar, as[k])) : mul2(br, bc[k]));
                if (!kNeighbours) {
                    xa[2 * k] = x.x; xa[2 * k + 1] = x.y; xb[2 * k] = y.x; xb[2 * k + 1] = y.y;
                } else if (k < kHalf / 2) {
                    xa[4 * k] = x.x; xa[4 * k + 1] = y.x; xa[4 * k + 2] = x.y; xa[4 * k + 3] = y.y;
                } else {
                    xb[4 * k - kVec] = x.x; xb[4 * k - kVec + 1] = y.x; xb[4 * k - kVec + 2] = x.y; xb[4 * k - kVec + 3] = y.y;
                }
            }
            if (live) { store_vec(out + at, xa); store_vec(out + at + b_off, xb); }
          }
        }
    }
}

// Rows come into a ring in shared memory by bulk copies, are worked on in place and leave by bulk copies, so that what is on its way
// needs no registers; angles (a chain of loads: axis, position, table) are put beside them by warps of their own, which also ask for the rows. A thread keeps its
// channels' gains over all rows where every lane group has one head. A row is at most a stage of 24 KB: four of them and three CTAs fill an SM
// for rows of up to 18 KB.
constexpr int kRing = 4, kRingThreads = 384, kMostAngleThreads = 128, kRingCtas = 3;   // CTAs: of an SM
struct RingParams {
    NormRopeParams n;
    long long rows;
    int row_bytes, store_bytes, stage_bytes, angle_threads, groups;
};
template <typename T, int kVec, bool kNeighbours>
__global__ void __launch_bounds__(kRingThreads, kRingCtas) qk_norm_rope_ring_kernel(const RingParams q) {
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ __align__(16) float s_cos[kRing][kMostAngleThreads], s_sin[kRing][kMostAngleThreads];
    __shared__ __align__(8) uint64_t full[kRing], empty[kRing];
    const NormRopeParams& p = q.n;
    const QkRotation& r = p.r;
    const int tid = threadIdx.x;
    if (tid == 0) {
        for (int i = 0; i < kRing; ++i) { mbar_init(&full[i], 1 + q.angle_threads); mbar_init(&empty[i], 1); }
        mbar_fence_init();
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();
    bool failed = false;
    if (tid < q.angle_threads) {
        // ---- rows and angles ---------------------------------------------------------------------------------------------------------------------
        const bool turns = tid < r.rot_half;
        const int axis = turns && r.pair_axis ? r.pair_axis[tid] : 0;
        auto position = [&](long long row) -> long long {
            if (!turns || row >= q.rows || axis >= r.axes) return -1;
            return r.axis_positions ? r.axis_positions[axis * r.axis_stride + row] : p.positions[row];
        };
        long long row = blockIdx.x, pos = position(row);
        int i = 0;
        for (; row < q.rows; row += gridDim.x, ++i) {
            const int st = i % kRing;
            if (i >= kRing && !mbar_wait_bounded(&empty[st], (uint32_t)(i / kRing - 1) & 1u)) { failed = true; break; }
            if (tid == 0) {
                mbar_expect_tx(&full[st], q.row_bytes);
                bulk_g2s(ring + st * q.stage_bytes, static_cast<const T*>(p.in) + row * p.ld_in, q.row_bytes, &full[st]);
            }
            const long long next = position(row + gridDim.x);
            if (turns) {
                if (pos < 0 || pos >= r.positions) { atomicExch(p.status, 2); pos = 0; }
                s_cos[st][tid] = r.cos[pos * r.rot_half + tid];
                s_sin[st][tid] = r.sin[pos * r.rot_half + tid];
            }
            pos = next;
            mbar_arrive(&full[st]);
        }
        // rows on their way that nobody waits for any more
        if (failed && tid == 0)
            for (int k = max(0, i - kRing); k < i; ++k) mbar_wait_bounded(&full[k % kRing], (uint32_t)(k / kRing) & 1u);
    } else {
        // ---- a head per lane group ------------------------------------------------------------------------------------------------------------------
        const int worker = tid - q.angle_threads, lanes = p.lanes, lane = worker & (lanes - 1), group = worker / lanes, workers = blockDim.x - q.angle_threads;
        const int first = lane * kVec, normed = r.q_heads + r.kv_heads;
        const bool some = 2 * first < r.dim, turned = first < r.rot_half;
        int ca, cb;
        pair_channels<kVec>(r, first, &ca, &cb);
        const bool one_pass = q.groups >= normed;
        float ga[kVec], gb[kVec];
        auto gains = [&](int h) {
#pragma unroll
            for (int k = 0; k < kVec; ++k) ga[k] = gb[k] = 1.f;
            if (r.q_gain && some && h < normed) {
                const float* gain = h < r.q_heads ? r.q_gain : r.k_gain;
                load_vec(gain + ca, ga);
                load_vec(gain + cb, gb);
            }
        };
        gains(group);
        const float width = 1.f / r.dim;
        int i = 0;
        for (long long row = blockIdx.x; row < q.rows; row += gridDim.x, ++i) {
            const int st = i % kRing;
            if (!failed && !mbar_wait_bounded(&full[st], (uint32_t)(i / kRing) & 1u)) failed = true;
            failed = __any_sync(0xffffffffu, failed);
            T* const at = reinterpret_cast<T*>(ring + st * q.stage_bytes);
            for (int h0 = 0; h0 < normed && !failed; h0 += q.groups) {
                const int h = h0 + group;
                const bool live = h < normed && some;
                if (!one_pass) gains(h);
                T* const head = at + h * r.dim;
                float a[kVec] = {}, b[kVec] = {};
                if (live) {
                    RawVec<T, kVec> ra, rb;
                    ra.load(head + ca);
                    rb.load(head + cb);
                    ra.get(a);
                    rb.get(b);
                }
                float rms = 1.f;
                if (r.q_gain) rms = rsqrtf(lane_group_sum(square_sum(a, b), lanes) * width + r.eps);
                if (live) {
#pragma unroll
                    for (int k = 0; k < kVec; ++k) { a[k] *= rms * ga[k]; b[k] *= rms * gb[k]; }
                    if (turned) {
                        float c[kVec], s[kVec];
                        load_vec(s_cos[st] + first, c);
                        load_vec(s_sin[st] + first, s);
                        rotate_pairs(!kNeighbours, a, b, c, s);
                    }
                    store_vec(head + ca, a);
                    store_vec(head + cb, b);
                }
            }
            fence_proxy_async();
            asm volatile("bar.sync 1, %0;\n" ::"r"(workers) : "memory");
            if (worker == 0 && !failed) {
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n" ::"l"(static_cast<T*>(p.out) + row * p.ld_out), "r"(smem_u32(at)), "r"(q.store_bytes)
                             : "memory");
                asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
                // the row before this one has been read out of its stage
                asm volatile("cp.async.bulk.wait_group.read 1;\n" ::: "memory");
                if (i > 0) mbar_arrive(&empty[(i - 1) % kRing]);
            }
        }
        if (worker == 0) asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory");
    }
    if (failed) atomicExch(p.status, 3);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const NormRopeParams p) {
    constexpr int kVec = 1, kRuns = 8;   // pairs of a lane at a time; 32 lanes x 8 x 2 channels
    pdl_launch_dependents();
    pdl_wait();
    const QkRotation& r = p.r;
    const long long row = blockIdx.x;
    const int lanes = p.lanes, lane = threadIdx.x & (lanes - 1), n_groups = kThreads / lanes;
    const int normed = r.q_heads + r.kv_heads, position = p.positions ? p.positions[row] : 0;
    int ca[kRuns], cb[kRuns], first[kRuns];
    float c[kRuns][kVec], s[kRuns][kVec];
#pragma unroll
    for (int j = 0; j < kRuns; ++j) {
        first[j] = (lane + j * lanes) * kVec;
        if (2 * first[j] >= r.dim) { first[j] = -1; continue; }
        pair_channels<kVec>(r, first[j], &ca[j], &cb[j]);
        pair_angles<kVec>(r, (int)row, position, first[j], p.status, c[j], s[j]);
    }
    const T* in = static_cast<const T*>(p.in) + row * p.ld_in;
    T* out = static_cast<T*>(p.out) + row * p.ld_out;
    // every lane of a warp takes part in the sums, groups past the last head included
    for (int h0 = 0; h0 < p.heads; h0 += n_groups) {
        const int h = h0 + threadIdx.x / lanes;
        const bool live = h < p.heads;
        float a[kRuns][kVec], b[kRuns][kVec], sum = 0.f;
#pragma unroll
        for (int j = 0; j < kRuns; ++j)
            if (live && first[j] >= 0) {
                load_vec(in + h * r.dim + ca[j], a[j]);
                load_vec(in + h * r.dim + cb[j], b[j]);
                sum += square_sum(a[j], b[j]);
            }
        const float* gain = h < r.q_heads ? r.q_gain : r.k_gain;
        float rms = 1.f;
        if (gain) rms = rsqrtf(lane_group_sum(sum, lanes) / r.dim + r.eps);
#pragma unroll
        for (int j = 0; j < kRuns; ++j)
            if (live && first[j] >= 0) {
                if (h < normed) {
                    if (gain) times_gain(gain, ca[j], cb[j], rms, a[j], b[j]);
                    if (first[j] < r.rot_half) rotate_pairs(!r.neighbours, a[j], b[j], c[j], s[j]);
                }
                store_vec(out + h * r.dim + ca[j], a[j]);
                store_vec(out + h * r.dim + cb[j], b[j]);
            }
    }
}

int lanes_of(int vectors) {
    int n = 1;
    while (n < vectors && n < 32) n *= 2;
    return n;
}
template <typename T, int kVec>
int launch_wide(NormRopeParams& p, int64_t rows, cudaStream_t st) {
    const QkRotation& r = p.r;
    p.lanes = lanes_of(r.dim / 2 / kVec);
    const int at_once = 32 / p.lanes;
    auto cut = [&](int heads) {
        p.part_heads = heads;
        p.q_parts = ceil_div(r.q_heads, heads);
        p.k_parts = ceil_div(r.kv_heads, heads);
        p.parts = p.q_parts + p.k_parts * (p.copies ? 2 : 1);
        p.items = rows * p.parts;
    };
    // a warp has four heads per lane group where that leaves work for every warp, else one
    cut(4 * at_once);
    if (p.items < 16 * (int64_t)sm_count()) cut(at_once);
    const dim3 grid((unsigned)std::min<int64_t>((p.items + kThreads / 32 - 1) / (kThreads / 32), 2 * (int64_t)sm_count())), block(kThreads);
    if (r.neighbours) return launch_kernel(qk_norm_rope_wide_kernel<T, kVec, true>, grid, block, 0, st, 1, p);
    return launch_kernel(qk_norm_rope_wide_kernel<T, kVec, false>, grid, block, 0, st, 1, p);
}
template <typename T, int kVec>
int launch_ring(NormRopeParams& p, int64_t rows, int row_bytes, cudaStream_t st) {
    const QkRotation& r = p.r;
    RingParams q = {};
    p.lanes = lanes_of(r.dim / 2 / kVec);
    q.n = p;
    q.rows = rows;
    q.row_bytes = row_bytes;
    q.store_bytes = p.copies ? row_bytes : (int)((r.q_heads + r.kv_heads) * r.dim * sizeof(T));
    q.stage_bytes = (row_bytes + 127) / 128 * 128;
    q.angle_threads = std::max(32, (r.rot_half + 31) / 32 * 32);
    const int threads = std::min((kRingThreads - q.angle_threads) / 32 * 32, ceil_div((int64_t)(r.q_heads + r.kv_heads) * p.lanes, 32) * 32);
    q.groups = threads / p.lanes;
    const size_t smem = (size_t)kRing * q.stage_bytes;
    auto kernel = r.neighbours ? qk_norm_rope_ring_kernel<T, kVec, true> : qk_norm_rope_ring_kernel<T, kVec, false>;
    static PerDeviceOnce attr_once[2];
    if (attr_once[r.neighbours].first_time()) GPTRS_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing * 24576));
    const dim3 grid((unsigned)std::min<int64_t>(rows, kRingCtas * (int64_t)sm_count()));
    return launch_kernel(kernel, grid, dim3(threads + q.angle_threads), smem, st, 1, q);
}
template <typename T>
int launch_norm_rope(NormRopeParams& p, int64_t rows, cudaStream_t st) {
    const QkRotation& r = p.r;
    auto aligned = [](const void* q, size_t b) { return (reinterpret_cast<uintptr_t>(q) & (b - 1)) == 0; };
    auto in_pieces = [&](int n) {   // rows go by 2 n channels a lane
        return r.dim % (2 * n) == 0 && r.dim <= 64 * n && r.rot_half % n == 0 && p.ld_in % n == 0 && p.ld_out % n == 0 && aligned(p.in, n * sizeof(T)) && aligned(p.out, n * sizeof(T)) &&
               aligned(r.q_gain, 16) && aligned(r.k_gain, 16) && aligned(r.cos, 16) && aligned(r.sin, 16);
    };
    constexpr int kPiece = 16 / sizeof(T);
    const int64_t row_bytes = (int64_t)(r.q_heads + 2 * r.kv_heads) * r.dim * sizeof(T);
    const bool many = sizeof(T) == 2 || rows >= sm_count();
    if (many && in_pieces(kPiece) && row_bytes <= 24576 && r.rot_half <= kMostAngleThreads) return launch_ring<T, kPiece>(p, rows, (int)row_bytes, st);
    if (sizeof(T) == 2 && in_pieces(8)) return launch_wide<T, sizeof(T) == 2 ? 8 : 4>(p, rows, st);
    if (in_pieces(4)) return launch_wide<T, 4>(p, rows, st);
    p.lanes = lanes_of(r.dim / 2);
    return launch_kernel(qk_norm_rope_kernel<T>, dim3((unsigned)rows), dim3(kThreads), 0, st, 1, p);
}

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" int gptrs_cuda_qk_norm_rope(const gptrs_qk_rotation* r, const void* d_qkv, int dtype, int64_t ld_in, const int32_t* d_positions, void* d_out,
                                       int64_t ld_out, int32_t* d_status, int64_t rows, void* stream) {
    GPTRS_REQUIRE(r && d_status, "null pointer");
    GPTRS_REQUIRE(rows == 0 || (d_qkv && d_out), "null pointer");   // (tensors without rows have none)
    GPTRS_REQUIRE(dtype == GPTRS_F32 || dtype == GPTRS_BF16, "rows are f32 or bf16");
    GPTRS_REQUIRE(rows >= 0 && rows <= 0x7fffffff, "bad row count");
    NormRopeParams p = {};
    const int rc = qk_rotation_of(*r, rows, &p.r);
    if (rc) return rc;
    GPTRS_REQUIRE(rows == 0 || p.r.rot_half == 0 || p.r.axis_positions || d_positions, "positions are missing");
    const int64_t width = (int64_t)(r->q_heads + 2 * r->kv_heads) * r->dim;
    p.ld_in = ld_in ? ld_in : width;
    p.ld_out = ld_out ? ld_out : width;
    GPTRS_REQUIRE(p.ld_in >= width && p.ld_out >= width, "rows overlap");
    const bool in_place = d_qkv == d_out;
    GPTRS_REQUIRE(!in_place || p.ld_in == p.ld_out, "in place the strides are the same");
    if (rows == 0) return GPTRS_OK;
    if (!in_place) {   // rows are worked on in no order: the target may lie between the source's rows, not in them
        const int64_t size = dtype == GPTRS_F32 ? 4 : 2, apart = ((intptr_t)d_out - (intptr_t)d_qkv) / size, in_end = (rows - 1) * p.ld_in + width, out_end = (rows - 1) * p.ld_out + width;
        const int64_t shift = p.ld_in == p.ld_out ? (apart % p.ld_in + p.ld_in) % p.ld_in : 0;
        GPTRS_REQUIRE(apart >= in_end || -apart >= out_end || (shift >= width && shift <= p.ld_in - width), "the target's rows lie in the source's");
    }
    p.in = d_qkv; p.out = d_out; p.positions = d_positions; p.status = d_status;
    p.copies = !in_place;
    p.heads = r->q_heads + (in_place ? 1 : 2) * r->kv_heads;
    return dtype == GPTRS_F32 ? launch_norm_rope<float>(p, rows, as_stream(stream)) : launch_norm_rope<__nv_bfloat16>(p, rows, as_stream(stream));
}
