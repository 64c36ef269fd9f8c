// Scores of rows against a vocabulary without logits in memory: log sum exp, log-probabilities of given tokens, greedy or sampled picks.
//
// z = x . w^T on the tcgen05 tensor cores, x rows as the M side. A unit is a tile of rows x a stretch of the vocabulary, which a CTA (one per SM) walks over in tiles of
// up to 256 tokens. What a row needs to know of its logits is a running state in registers (maximum and sum, best token, the target's logit), so a logit lives
// from the accumulator to the exponential and nowhere else.
//   warps 0 - 7   a thread per row and half of the tile's tokens. The accumulator in tensor memory is read out every 128 to 512 of dim (up to 1024 where draws keep its readers busy) and added up in f32 registers: the
//                 tensor cores cut what does not fit into the sum that they add to, 16 products at a time, which over all of dim would cost log-probabilities digits.
//                 Up to 16 rows the logits then go through shared memory, and a warp takes a row with a token per lane
//   warp 8        requests stages of 64 of dim
//   warp 9        one thread issues the products into one of two accumulators
// Up to 128 rows a tile is 128 rows and one CTA's. Above, a cluster of two CTAs works on 256 rows (cta_group::2): each brings its 128 rows of x and half of the tokens, 32 KB
// for 64 of dim where a CTA by itself brings 48, and an SM takes about 64 bytes a cycle out of L2.
// Units go row tile first, so that the CTAs that run at one time share stretches of w through L2. A second kernel joins the parts of a row; it compares tokens where
// values are equal, so results do not depend on an order.
//
// What bounds it (times of the kernels in a graph; calls from Python by themselves take 2 to 60 us more): up to 128 rows w's bytes (one row of 50257 x 2048 42 us, 31.5 at the rate of a copy;
// of 131072 x 4096 16 rows 164 us, 64 rows 184, drawn 234, 128 rows 192, drawn 250; 164). Above, the products: 4001 rows of 131072 x 2048 1.37 to 1.58 ms as the power cap allows, the tensor pipe
// busy in 96 to 98 % of the cycles (1.26 at the rate of short products). 416 drawn rows of 131072 x 4096 415 to 440 us: they are two tiles of 256 (262 us for 416 rows, 322 for 512), and a
// draw costs a hash a logit. Below a dim of some hundred, and with a cap, the epilogue: 2048 rows of 50257 x 320 96 us (39), 64 rows of 131072 x 2048 108 us, with a bias 121, with a
// cap, which is a call and a tanhf a logit, 218 (82); 2048 rows 0.81, 0.97 and 1.50 ms (0.65). One row of 4000 x 4096 26 us (5): dim is walked over in order, by 125 CTAs of 32 tokens.
// Every wait is bounded: on a timeout code 3 goes to the status word, the roles leave their loops, tensor memory is freed.
#include <algorithm>

#include "umma_common.cuh"

namespace gptrs {

void prefill_tc_fault(int* starve, uint32_t* wait_limit);   // the test switch of paged_prefill_tc.cu

namespace {

constexpr int kRows = 128;                      // of a CTA
constexpr int kStageDim = 64;                   // bf16 of a 128-byte swizzle span
// How a call's rows are worked on: up to 16 of them, up to 128, more (by pairs of CTAs).
enum { kFew, kOne, kPairs };
constexpr int kCols = 256;                      // most tokens of a tile
constexpr int kMostStages = 16;                 // (as many as fit: narrow tiles have small stages, and need more of them under way)
constexpr int x_bytes(int mode) { return 128 * (mode == kFew ? 64 : 128); }        // of a stage; products of 64 rows where there are 16 at most
// Stages that an accumulator adds up: 128 of dim where w's bytes bound the call, 512 where the products do and each handing over takes time from them. The cuts go one way: sums of products
// of one sign come out low by 2.8, 6.4 and 15 times 2^-24 of themselves with 128, 256 and 512 of dim (f32 sums in an order of their own are off by 0.7 either way). Of logits that are not, relative
// errors of lse at a dim of 4096 are 1.0e-7 and 4.0e-7 with 128 and 512 (f32 sums one by one 5.8e-7); 4001 rows in 131072 tokens take 1.72 ms with 256, 1.54 with 512. One row of
// 50257 x 2048 whose lse is about 15 takes 41.7 us and is 1.3e-6 off, with 256 40.6 and 2.5e-6, with 64 43.7 and 0.9e-6 (f32 sums 0.6e-6; a step of f32 is 0.95e-6); one of 4000 x 4096 27, 23 and 33 us.
constexpr int drain_of(int mode) { return mode == kPairs ? 8 : 2; }
constexpr int kEpilogue = 256, kThreads = kEpilogue + 128;   // two warps of the last four only make their group whole
// Registers of a thread at launch, and what the groups of four warps make of them: the shares add up to less than the block has, so every request ends.
constexpr int kLaunchRegs = 168, kEpilogueRegs = 208, kOtherRegs = 80;
static_assert(2 * kEpilogueRegs + kOtherRegs <= 3 * kLaunchRegs, "more registers than the block is launched with");
constexpr int kZRow = kCols + 4;                // floats of a row of logits in shared memory (kFew)
constexpr int stage_bytes(int mode, int cols) { return x_bytes(mode) + 128 * (mode == kPairs ? cols / 2 : cols); }
constexpr size_t kSmem = 200 * 1024 + 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kJoinThreads = 256;

// Of a row and a stretch: sum exp z = (1 + rest) exp m, the best token (-1: none) and its z, the target's z (NaN: not here). The largest term is apart from the others, so that what
// is small beside it keeps its digits: a token that is nearly certain has a log-probability of about -rest.
struct __align__(32) Part { float m, rest, best, z; int token; float given; float pad[2]; };
__device__ __forceinline__ Part no_part() { return {-INFINITY, -1.f, -INFINITY, -INFINITY, -1, NAN}; }

struct ScoreParams {
    CUtensorMap x_map, w_map;
    const float* bias;
    const uint32_t* seed_at;
    const int* target;
    Part* parts;                  // [rows][row_parts]: of stretches (kFew), or halves of them
    int *pick, *status;
    float *pick_logprob, *logprob, *lse;
    int rows, dim, vocab;
    int row_tiles, stretches, tiles, cols;   // a stretch is `tiles` tiles of `cols` tokens
    int x_rows;                   // of a copy of x
    int row_parts, stages;
    float cap, inv_t;             // cap 0: none, negative: see capped(); inv_t 0: greedy
    uint32_t seed, wait_limit;
    int starve;
};

__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16; x *= 0x7feb352du; x ^= x >> 15; x *= 0x846ca68bu; x ^= x >> 16;
    return x;
}
__device__ __forceinline__ uint32_t draw(uint32_t seed, int row, int token) { return mix(seed ^ mix((uint32_t)token + 0x9e3779b9u * (uint32_t)(row + 1))); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// (h + 1/2 rounds to 2^32 for the last 128 of h: below 1, so that no token's value is -inf for its noise)
__device__ __forceinline__ float gumbel(uint32_t h) { return -logf(-log1pf(-fminf(((float)h + 0.5f) * (1.f / 4294967296.f), 1.f - 0x1p-24f))); }
// cap tanh(z / cap), the same for -cap, which says that there is a bias: a token that it leaves out stays out, where the cap would make -cap of it. (A call's place is a call and no more:
// asked for at the loop of logits, 416 draws took 438 us instead of 423 without a cap.)
__device__ __noinline__ float capped(float z, float cap) { return cap < 0.f && z == -INFINITY ? z : cap * tanhf(z / cap); }
__device__ __forceinline__ void join(Part& a, const Part& b) {
    const float m = fmaxf(a.m, b.m);
    const float ref = m == -INFINITY ? 0.f : m;   // (a sum that is NaN stays one)
    const bool mine = a.m == m;
    a.rest = (mine ? a.rest : b.rest) + (1.f + (mine ? b.rest : a.rest)) * ex2(((mine ? b.m : a.m) - ref) * kLog2e);
    a.m = m;
    if (b.token >= 0 && (a.token < 0 || b.best > a.best || (b.best == a.best && b.token < a.token))) { a.best = b.best; a.z = b.z; a.token = b.token; }
    if (b.given == b.given) a.given = b.given;
}

template <bool kPair>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    if constexpr (kPair)   // the barrier may be the other CTA's
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n" ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <bool kPair>
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kPair)
        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                     : "memory");
    else
        umma_bf16(d, a, b, idesc, accumulate);
}
template <bool kPair>
__device__ __forceinline__ void commit(uint64_t* bar) {   // to the barrier of both CTAs
    if constexpr (kPair)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
    else
        umma_commit(bar);
}

// The best token among the lanes' and the sum of all.
__device__ __forceinline__ Part join_lanes(Part a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Part b = {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.rest, o), __shfl_xor_sync(0xffffffffu, a.best, o),
                        __shfl_xor_sync(0xffffffffu, a.z, o), __shfl_xor_sync(0xffffffffu, a.token, o), __shfl_xor_sync(0xffffffffu, a.given, o)};
        join(a, b);
    }
    return a;
}

template <int kMode, bool kSample>
__global__ void __launch_bounds__(kThreads, 1) vocab_scores_kernel(const __grid_constant__ ScoreParams p) {
    constexpr bool kPair = kMode == kPairs;
    constexpr int kDrain = drain_of(kMode), kABytes = x_bytes(kMode), kCtas = kPair ? 2 : 1;
    constexpr uint32_t kTmemCols = 2 * kCols;
    constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)((kMode == kFew ? 64 : kCtas * kRows) >> 4) << 24);   // f32 accumulator, bf16 operands
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[kMostStages], empty[kMostStages], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_holder;
    __shared__ __align__(16) float s_z[kMode == kFew ? 16 : 1][kZRow];
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = kPair ? (int)cluster_ctarank() : 0;   // the first CTA's thread issues the products of both
    if (tid == 0) {
        for (int i = 0; i < kMostStages; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], kCtas * kEpilogue / 32); }
        mbar_fence_init();
    }
    if (warp == 9) {
        if constexpr (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_holder)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_holder)), "r"(kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        }
    }
    tc_fence_before();
    if constexpr (kPair) cluster_sync_all();   // the other CTA's barriers are there
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_holder;
    pdl_launch_dependents();
    pdl_wait();
    const int steps = (p.dim + kStageDim - 1) / kStageDim, units = p.row_tiles * p.stretches, my_cols = p.cols / kCtas, stages = p.stages, stage_size = stage_bytes(kMode, p.cols);
    // Draws take the epilogue longer than two accumulators of kDrain last. With the first two of a tile up to twice as long (a quarter of dim) the products go on meanwhile: 416 rows of
    // 131072 x 4096 430 -> 405 us, and lse is off by 6.2e-7 instead of 4.0e-7 (f32 sums one by one 5.8e-7).
    const int lead = kPair && kSample ? min(2 * kDrain, max(kDrain, steps / 4)) : kDrain;
    auto behind = [&](int k0) { return k0 + (k0 < 2 * lead ? lead : kDrain); };   // the first stage of the next accumulator
    struct Unit { int row0, begin, end; };
    auto unit_of = [&](int u) {
        const int begin = u / p.row_tiles * (p.tiles * p.cols);
        return Unit{(u % p.row_tiles) * (kCtas * kRows) + rank * kRows, begin, min(p.vocab, begin + p.tiles * p.cols)};
    };
    bool failed = false;

    if (warp >= 10) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
    } else if (warp == 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
        if (elect_one()) {
            int it = 0, s = 0;
            uint32_t phase = 1;
            const uint32_t bytes = (uint32_t)(kCtas * (p.x_rows + my_cols) * 128);
            for (int u = blockIdx.x / kCtas; u < units && !failed; u += gridDim.x / kCtas) {
                const Unit unit = unit_of(u);
                for (int n0 = unit.begin; n0 < unit.end && !failed; n0 += p.cols) {
                    for (int k = 0; k < steps; ++k, ++it) {
                        if (it >= stages && !mbar_wait_polled(&empty[s], phase, p.wait_limit, 256)) { failed = true; break; }
                        const uint32_t at = smem + s * stage_size, bar = kPair ? map_to_cta(smem_u32(&full[s]), 0) : smem_u32(&full[s]);
                        if (rank == 0) mbar_expect_tx(&full[s], bytes);
                        if (!(p.starve && it == 0)) load_2d<kPair>(at, &p.x_map, k * kStageDim, unit.row0, bar);
                        load_2d<kPair>(at + kABytes, &p.w_map, k * kStageDim, n0 + rank * my_cols, bar);
                        if (++s == stages) { s = 0; phase ^= 1u; }
                    }
                }
            }
            // Stages in flight write the CTAs' shared memory (only after a timeout are there any left unread). Of a pair the first CTA waits for both: the other one stays until the end.
            if (rank == 0)
                for (int i = max(it - stages, 0); i < it; ++i) mbar_wait_parked(smem_u32(&full[i % stages]), (uint32_t)(i / stages) & 1u, p.wait_limit);
            if (failed) atomicExch(p.status, 3);
        }
        __syncwarp();
    } else if (warp == 9) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
        if (rank == 0 && elect_one()) {
            int s = 0, n = 0;
            uint32_t phase = 0;
            const uint32_t idesc = kIdesc | ((uint32_t)(p.cols >> 3) << 17);
            for (int u = blockIdx.x / kCtas; u < units && !failed; u += gridDim.x / kCtas) {
                const Unit unit = unit_of(u);
                for (int n0 = unit.begin; n0 < unit.end && !failed; n0 += p.cols) {
                    for (int k0 = 0; k0 < steps && !failed; k0 = behind(k0), ++n) {
                        const int buf = n & 1, k1 = min(behind(k0), steps);
                        if (n >= 2 && !mbar_wait_polled(&acc_empty[buf], (uint32_t)((n >> 1) - 1) & 1u, p.wait_limit, 256)) { failed = true; break; }
                        tc_fence_after();
                        for (int k = k0; k < k1; ++k) {
                            if (!mbar_wait_polled(&full[s], phase, p.wait_limit, 256)) { failed = true; break; }
                            tc_fence_after();
                            const uint64_t a = make_smem_desc(smem + s * stage_size), b = make_smem_desc(smem + s * stage_size + kABytes);
#pragma unroll
                            for (int i = 0; i < 4; ++i) multiply<kPair>(tmem + (uint32_t)(buf * kCols), a + 2 * i, b + 2 * i, idesc, (k > k0 || i > 0) ? 1u : 0u);
                            commit<kPair>(&empty[s]);
                            if (++s == stages) { s = 0; phase ^= 1u; }
                        }
                        if (!failed) commit<kPair>(&acc_full[buf]);
                    }
                }
            }
            if (failed) atomicExch(p.status, 3);
        }
        __syncwarp();
    } else if constexpr (kMode == kFew) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kEpilogueRegs));
        // Warps 0 and 4 hold the rows in their first 16 lanes, 128 tokens each, and hand the logits to all eight: warp w has the rows w and w + 8, a lane every 32nd token. After a
        // timeout every warp still goes through all tiles, without waiting, so that the barriers are met.
        const int half = warp >> 2;
        const bool holds = (warp & 3) == 0;
        const uint32_t seed = p.seed_at ? *p.seed_at : p.seed;
        int n = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x) {
            const Unit unit = unit_of(u);
            Part a[2];
            int target[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                a[r] = no_part();
                target[r] = p.target && warp + 8 * r < p.rows ? p.target[warp + 8 * r] : -1;
            }
            for (int n0 = unit.begin; n0 < unit.end; n0 += p.cols) {
                uint64_t acc[kCols / 4];
#pragma unroll
                for (int i = 0; i < kCols / 4; ++i) acc[i] = 0;
                for (int k0 = 0; k0 < steps; k0 += kDrain, ++n) {
                    const int buf = n & 1;
                    if (!failed && !mbar_wait_polled(&acc_full[buf], (uint32_t)(n >> 1) & 1u, p.wait_limit, 64)) failed = true;
                    failed = __any_sync(0xffffffffu, failed);
                    if (failed) break;
                    tc_fence_after();
                    if (holds && 128 * half < p.cols) {
                        uint32_t v[2][32];   // a quarter on its way while the one in front is added
                        const uint32_t at = tmem + (uint32_t)(buf * kCols + 128 * half);
                        tmem_ld_32_begin(at, v[0]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            if (128 * half + 32 * c >= p.cols) break;
                            tmem_ld_32_end(v[c & 1]);
                            if (c < 3 && 128 * half + 32 * (c + 1) < p.cols) tmem_ld_32_begin(at + 32u * (c + 1), v[(c + 1) & 1]);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                acc[16 * c + i] = add2(acc[16 * c + i], pair_of(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])));
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&acc_empty[buf]);
                }
                if (holds && lane < 16) {
#pragma unroll
                    for (int i = 0; i < kCols / 8; ++i) {
                        const float2 x = split(acc[2 * i]), y = split(acc[2 * i + 1]);
                        *reinterpret_cast<float4*>(&s_z[lane][128 * half + 4 * i]) = make_float4(x.x, x.y, y.x, y.y);
                    }
                }
                asm volatile("bar.sync 1, %0;\n" ::"n"(kEpilogue) : "memory");
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int row = warp + 8 * r;
                    if (row >= p.rows) break;
#pragma unroll
                    for (int i = 0; i < kCols / 32; ++i) {
                        const int at = 32 * i + lane, token = n0 + at;
                        if (at >= p.cols || token >= unit.end) continue;
                        float z = s_z[row][at];
                        if (p.bias) z += __ldg(p.bias + token);
                        if (p.cap != 0.f) z = capped(z, p.cap);
                        if (token == target[r]) a[r].given = z;
                        float value = z;
                        if constexpr (kSample) value = fmaf(z, p.inv_t, gumbel(draw(seed, row, token)));
                        if (value > a[r].best) { a[r].best = value; a[r].z = z; a[r].token = token; }
                        const bool up = z > a[r].m;
                        const float e = ex2((up ? a[r].m - z : z - (a[r].m == -INFINITY ? 0.f : a[r].m)) * kLog2e);
                        a[r].rest = up ? (1.f + a[r].rest) * e : a[r].rest + e;
                        a[r].m = up ? z : a[r].m;
                    }
                }
                asm volatile("bar.sync 1, %0;\n" ::"n"(kEpilogue) : "memory");
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = warp + 8 * r;
                if (row >= p.rows) break;
                const Part all = join_lanes(a[r]);
                if (lane == 0 && !failed) p.parts[(size_t)row * p.stretches + u] = all;
            }
        }
        if (failed && lane == 0) atomicExch(p.status, 3);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kEpilogueRegs));
        // Quarters of 32 tokens that a warp has none of are left out; a warp without rows only hands accumulators back.
        const int half = warp >> 2, in_tile = (warp & 3) * 32 + lane, width = (p.cols / 2 + 15) / 16 * 16;   // of the first half
        const uint32_t acc0 = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * width);
        const uint32_t seed = p.seed_at ? *p.seed_at : p.seed;
        uint32_t handed[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) handed[i] = kPair ? map_to_cta(smem_u32(&acc_empty[i]), 0) : smem_u32(&acc_empty[i]);
        int n = 0;
        for (int u = blockIdx.x / kCtas; u < units && !failed; u += gridDim.x / kCtas) {
            const Unit unit = unit_of(u);
            const int row = unit.row0 + in_tile;
            const bool rows = unit.row0 + (warp & 3) * 32 < p.rows;
            const int target = p.target && row < p.rows ? p.target[row] : -1;
            Part a = no_part();
            for (int n0 = unit.begin; n0 < unit.end && !failed; n0 += p.cols) {
                const int first = n0 + half * width, some = rows ? min(half ? p.cols - width : width, unit.end - first) : 0;   // this half's tokens
                uint64_t acc[kCols / 4];
#pragma unroll
                for (int i = 0; i < kCols / 4; ++i) acc[i] = 0;
                for (int k0 = 0; k0 < steps; k0 = behind(k0), ++n) {
                    const int buf = n & 1;
                    if (!failed && !mbar_wait_polled(&acc_full[buf], (uint32_t)(n >> 1) & 1u, p.wait_limit, 64)) failed = true;
                    failed = __any_sync(0xffffffffu, failed);
                    if (failed) break;
                    tc_fence_after();
                    if (some > 0) {
                        uint32_t v[2][32];   // a quarter on its way while the one in front is added
                        tmem_ld_32_begin(acc0 + (uint32_t)(buf * kCols), v[0]);
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            if (32 * c >= some) break;
                            tmem_ld_32_end(v[c & 1]);
                            if (c < 3 && 32 * (c + 1) < some) tmem_ld_32_begin(acc0 + (uint32_t)(buf * kCols + 32 * (c + 1)), v[(c + 1) & 1]);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                acc[16 * c + i] = add2(acc[16 * c + i], pair_of(__uint_as_float(v[c & 1][2 * i]), __uint_as_float(v[c & 1][2 * i + 1])));
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (kPair)   // (the reads of tensor memory are complete, and nothing else is handed over: no fence over the cluster, which takes as long as they do)
                            asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(handed[buf]) : "memory");
                        else mbar_arrive_addr(handed[buf]);
                    }
                }
                if (failed || some <= 0) continue;
                const int wanted = (unsigned)(target - first) < (unsigned)some ? target - first : -1;
                const bool given = __any_sync(0xffffffffu, wanted >= 0);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (32 * c >= some) break;
                    float z[32];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 two = split(acc[16 * c + i]);
                        z[2 * i] = two.x;
                        z[2 * i + 1] = two.y;
                    }
                    const int n_c = first + 32 * c, some_c = some - 32 * c;
                    if (p.bias) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < some_c) z[i] += __ldg(p.bias + n_c + i);
                    }
                    if (p.cap != 0.f) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) z[i] = capped(z[i], p.cap);
                    }
                    if (some_c < 32) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i >= some_c) z[i] = -INFINITY;
                    }
                    if (given) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (wanted == 32 * c + i) a.given = z[i];
                    }
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; ++i) mx[i & 1] = fmaxf(mx[i & 1], z[i]);
                    const float top = fmaxf(mx[0], mx[1]);
                    if constexpr (kSample) {
                        // g <= -log v: a bound of one logarithm on the special function unit keeps all but a few tokens (as many as a running maximum has steps, about) from the
                        // noise in full. Sixteen at a time, so that the best of the ones in front counts. Room for the bound's errors: the logarithm's, and five roundings of
                        // numbers as large as z / T, which the value and the best are too wherever a token comes near the best, so that theirs is the size that counts.
#pragma unroll
                        for (int d = 0; d < 32; d += 16) {
                            uint32_t may = 0;
                            const float near = a.best - fmaf(fabsf(a.best), 0x1p-21f, 1e-3f);
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float low = __uint_as_float((draw(seed, row, n_c + d + i) >> 9) | 0x3f800000u) - 1.f;   // v from below
                                if (fmaf(lg2(low), -kLn2, z[d + i] * p.inv_t) > near) may |= 1u << i;
                            }
                            if (some_c - d < 16) may &= (1u << max(some_c - d, 0)) - 1u;
                            while (may) {
                                const int i = __ffs(may) - 1;
                                may &= may - 1;
                                float zi = z[d];
#pragma unroll
                                for (int j = 1; j < 16; ++j) zi = i == j ? z[d + j] : zi;
                                const float value = fmaf(zi, p.inv_t, gumbel(draw(seed, row, n_c + d + i)));
                                if (value > a.best || a.token < 0) { a.best = value; a.z = zi; a.token = n_c + d + i; }
                            }
                        }
                    }
                    const bool up = top > a.m;
                    if (__any_sync(0xffffffffu, up)) {   // the first of the largest: what a greedy pick takes, and what the sum of the others leaves out
                        int at = 0;
#pragma unroll
                        for (int i = 31; i >= 0; --i)
                            if (z[i] == top) at = i;
                        if constexpr (!kSample)
                            if (up) { a.best = a.z = top; a.token = n_c + at; }
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (up && i == at) z[i] = -INFINITY;
                    }
                    // sum exp z: differences first, so that what is rounded is small where it counts
                    const float to = up ? top : a.m, ref = to == -INFINITY ? 0.f : to;
                    const uint64_t ref2 = pair_of(-ref, -ref), log2 = pair_of(kLog2e, kLog2e);
                    uint64_t sums[2] = {0, 0};
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 e = split(mul2(add2(pair_of(z[2 * i], z[2 * i + 1]), ref2), log2));
                        sums[i & 1] = add2(sums[i & 1], pair_of(ex2(e.x), ex2(e.y)));
                    }
                    const float2 s = split(add2(sums[0], sums[1]));
                    a.rest = (up ? (1.f + a.rest) * ex2((a.m - ref) * kLog2e) : a.rest) + (s.x + s.y);
                    a.m = to;
                }
            }
            if (row < p.rows && !failed) p.parts[(size_t)row * p.row_parts + 2 * (u / p.row_tiles) + half] = a;
        }
        if (failed && lane == 0) atomicExch(p.status, 3);
    }
    tc_fence_before();
    if constexpr (kPair) cluster_sync_all();   // what the other CTA signals and reads is here until both are done
    else __syncthreads();
    if (warp == 9) {
        if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// A warp per row.
__global__ void __launch_bounds__(kJoinThreads) vocab_join_kernel(const __grid_constant__ ScoreParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31, n = p.row_parts;
    if (row >= p.rows) return;
    const Part* parts = p.parts + (size_t)row * n;
    Part a = no_part();
    for (int i = lane; i < n; i += 32) join(a, parts[i]);
    a = join_lanes(a);
    if (lane) return;
    // Log-probabilities from the difference to the largest logit, not to lse: rounded to f32 that is off by more than a token that is nearly certain has.
    const float others = log1pf(a.rest);
    if (p.lse) p.lse[row] = a.m + others;
    if (p.pick) p.pick[row] = max(a.token, 0);   // (nothing compares with NaN: the first token)
    if (p.pick_logprob) p.pick_logprob[row] = a.z - a.m - others;
    if (p.logprob) {
        const int target = p.target[row];
        if (target >= p.vocab) atomicExch(p.status, 2);
        p.logprob[row] = target < 0 ? 0.f : a.given - a.m - others;
    }
}

// How a call is cut: stretches of equal numbers of equal tiles, so many that units (row tiles x stretches) fill the SMs (or pairs of them) once, twice, up to eight times: whichever
// leaves the fewest tokens to the one that has most, a tile's own cost counted as 8 tokens and a unit's as 32.
struct Cut { int mode, row_tiles, stretches, tiles, cols; };
Cut cut(int64_t rows, int64_t vocab) {
    const int mode = rows <= 16 ? kFew : rows <= kRows ? kOne : kPairs;
    const bool pair = mode == kPairs;
    const int places = pair ? sm_count() / 2 : sm_count(), grain = pair ? 32 : 16, row_tiles = ceil_div(rows, pair ? 2 * kRows : kRows), grains = ceil_div(vocab, grain);
    Cut c = {mode, row_tiles, 1, 1, grain};
    int64_t best = -1;
    for (int waves = 1; waves <= 8; ++waves) {
        const int n = std::max(1, std::min(grains, places * waves / row_tiles));
        const int tiles = ceil_div(vocab, (int64_t)n * kCols), cols = (ceil_div(vocab, (int64_t)n * tiles) + grain - 1) / grain * grain;
        const int stretches = ceil_div(vocab, (int64_t)tiles * cols);
        const int64_t cost = (int64_t)ceil_div((int64_t)row_tiles * stretches, places) * (tiles * (cols + 8) + 32);
        if (best < 0 || cost < best) { best = cost; c = {mode, row_tiles, stretches, tiles, cols}; }
    }
    return c;
}

int encode(CUtensorMap* map, const void* base, int64_t cols, int64_t rows, int64_t ld, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(GPTRS_EXECUTION, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {kStageDim, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GPTRS_EXECUTION, "cuTensorMapEncodeTiled failed for scores (" + std::to_string((int)r) + ")");
    return GPTRS_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

using Kernel = void (*)(ScoreParams);
constexpr Kernel kKernels[3][2] = {{vocab_scores_kernel<kFew, false>, vocab_scores_kernel<kFew, true>},
                                   {vocab_scores_kernel<kOne, false>, vocab_scores_kernel<kOne, true>},
                                   {vocab_scores_kernel<kPairs, false>, vocab_scores_kernel<kPairs, true>}};

// A kernel compiled for fewer registers than its groups ask for would wait for them without end: none is launched then.
int registers_to_share() {
    static const int regs = [] {   // a thread's; of a kernel that has others, or none that are known
        for (int i = 0; i < 6; ++i) {
            cudaFuncAttributes attr;
            const int found = cudaFuncGetAttributes(&attr, kKernels[i / 2][i & 1]) == cudaSuccess ? attr.numRegs : 0;
            if (found != kLaunchRegs) return found;
        }
        return kLaunchRegs;
    }();
    if (regs != kLaunchRegs) return fail(GPTRS_EXECUTION, "vocab_scores_kernel has " + std::to_string(regs) + " registers a thread, not those that its warps share out");
    return GPTRS_OK;
}

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" {

size_t gptrs_cuda_vocab_scores_scratch_bytes(const gptrs_vocab_scores* s) {
    if (!s || s->rows < 1 || s->vocab < 1) return 0;
    if (s->rows > 0x3fffffff || s->vocab > 0x3fffffff) return 0;
    const Cut c = cut(s->rows, s->vocab);
    return (size_t)s->rows * (c.mode == kFew ? 1 : 2) * c.stretches * sizeof(Part);
}

int gptrs_cuda_vocab_scores(const gptrs_vocab_scores* s, void* stream) {
    GPTRS_REQUIRE(s && s->d_weight && s->d_status && (s->rows == 0 || s->d_hidden), "null pointer");
    GPTRS_REQUIRE(s->rows >= 0 && s->rows <= 0x3fffffff && s->vocab >= 1 && s->vocab <= 0x3fffffff && s->dim >= 8 && s->dim <= 0x3fffffff, "bad sizes");
    ScoreParams p = {};
    const int64_t ldx = s->ldh ? s->ldh : s->dim, ldw = s->ldw ? s->ldw : s->dim;
    GPTRS_REQUIRE(s->dim % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && ldx >= s->dim && ldw >= s->dim && ldx < ((int64_t)1 << 31) && ldw < ((int64_t)1 << 31),
                  "dim and the strides must be multiples of 8, and rows must not overlap");
    GPTRS_REQUIRE(aligned16(s->d_hidden) && aligned16(s->d_weight) && (reinterpret_cast<uintptr_t>(s->d_scratch) & 31) == 0, "pointers must be 16-byte aligned, scratch 32");
    // (its reciprocal is a factor: far from 1 it, or logits times it, would leave f32)
    GPTRS_REQUIRE(s->temperature <= 0.f || (s->temperature >= 1e-20f && s->temperature <= 1e20f), "a temperature above 0 must be 1e-20 .. 1e20");
    GPTRS_REQUIRE(s->soft_cap >= 0.f && s->soft_cap < 3e38f, "bad soft cap");
    GPTRS_REQUIRE(!s->d_logprob || s->d_target, "log-probabilities of targets need targets");
    GPTRS_REQUIRE(s->rows == 0 || (s->d_scratch && s->scratch_bytes >= gptrs_cuda_vocab_scores_scratch_bytes(s)), "scratch is too small");
    if (s->rows == 0) return GPTRS_OK;
    int rc = registers_to_share();
    if (rc) return rc;
    const Cut c = cut(s->rows, s->vocab);
    const bool pair = c.mode == kPairs;
    p.row_parts = c.mode == kFew ? c.stretches : 2 * c.stretches;
    p.stages = (int)std::min<int64_t>(kMostStages, (int64_t)(kSmem - 1024) / stage_bytes(c.mode, c.cols));
    p.row_tiles = c.row_tiles; p.stretches = c.stretches; p.tiles = c.tiles; p.cols = c.cols;
    p.x_rows = s->rows < kRows ? (int)(s->rows + 7) / 8 * 8 : kRows;   // (rows that nobody has are not read out: whatever lies there)
    rc = encode(&p.x_map, s->d_hidden, s->dim, s->rows, ldx, p.x_rows);
    if (!rc) rc = encode(&p.w_map, s->d_weight, s->dim, s->vocab, ldw, pair ? c.cols / 2 : c.cols);
    if (rc) return rc;
    p.bias = s->d_bias; p.seed_at = s->d_seed; p.target = s->d_target;
    p.parts = static_cast<Part*>(s->d_scratch);
    p.pick = s->d_pick; p.pick_logprob = s->d_pick_logprob; p.logprob = s->d_logprob; p.lse = s->d_lse; p.status = s->d_status;
    p.rows = (int)s->rows; p.dim = (int)s->dim; p.vocab = (int)s->vocab;
    p.cap = s->d_bias ? -s->soft_cap : s->soft_cap; p.inv_t = s->temperature > 0.f ? 1.f / s->temperature : 0.f; p.seed = s->seed;
    prefill_tc_fault(&p.starve, &p.wait_limit);
    static PerDeviceOnce attr_once;
    if (attr_once.first_time())
        for (int i = 0; i < 6; ++i) GPTRS_CUDA_OK(cudaFuncSetAttribute(kKernels[i / 2][i & 1], cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    const int64_t units = (int64_t)p.row_tiles * p.stretches, places = pair ? sm_count() / 2 : sm_count();
    // (a CTA counts its stages in 32 bits)
    GPTRS_REQUIRE(units < ((int64_t)1 << 30) && (units / places + 1) * p.tiles * ceil_div(p.dim, kStageDim) < ((int64_t)1 << 31), "too many rows for one call");
    rc = launch_kernel(kKernels[c.mode][p.inv_t > 0.f], dim3((unsigned)((units < places ? units : places) * (pair ? 2 : 1))), dim3(kThreads), kSmem, as_stream(stream), 1, p,
                       pair ? 2 : 1);
    if (rc) return rc;
    // the second kernel waits for the first one itself (griddepcontrol.wait), so it may be launched ahead of its end
    const int pdl = g_use_pdl;
    g_use_pdl = 1;
    rc = launch_kernel(vocab_join_kernel, dim3((unsigned)ceil_div(p.rows, kJoinThreads / 32)), dim3(kJoinThreads), 0, as_stream(stream), 1, p);
    g_use_pdl = pdl;
    return rc;
}

}  // extern "C"
