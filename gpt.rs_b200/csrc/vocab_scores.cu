// Scores of rows against a vocabulary without logits in memory: log sum exp, log-probabilities of given tokens, greedy or sampled picks.
//
// A row's result is put together from parts of the vocabulary: (m, l) with sum exp z = l exp m, the best token with its z, the target's z. Parts are
// joined in their order by a second kernel, so results do not depend on which CTA is done first.
#include "common.cuh"

namespace gptrs {
namespace {

constexpr int kTile = 64, kStep = 32, kThreads = 256;

struct Part { float m, l, best, z; int token; float given; };   // of a row and a part of the vocabulary; token -1, given NaN: none in it

struct ScoreParams {
    const __nv_bfloat16 *x, *w;
    long long ldx, ldw;
    const float* bias;
    const uint32_t* seed_at;
    const int* target;
    Part* parts;                  // [rows][n_parts]
    int *pick, *status;
    float *pick_logprob, *logprob, *lse;
    int rows, dim, vocab, n_parts;
    float cap, inv_t;             // inv_t 0: greedy
    uint32_t seed;
};

__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16; x *= 0x7feb352du; x ^= x >> 15; x *= 0x846ca68bu; x ^= x >> 16;
    return x;
}
__device__ __forceinline__ float gumbel(uint32_t seed, int row, int token) {
    const uint32_t h = mix(seed ^ mix((uint32_t)token + 0x9e3779b9u * (uint32_t)(row + 1)));
    return -logf(-log1pf(-(((float)h + 0.5f) * (1.f / 4294967296.f))));
}
__device__ __forceinline__ void join(Part& a, const Part& b) {   // b behind a in the vocabulary
    const float m = fmaxf(a.m, b.m);
    if (m != -INFINITY) a.l = a.l * (a.m == m ? 1.f : expf(a.m - m)) + b.l * (b.m == m ? 1.f : expf(b.m - m));
    else a.l += b.l;   // (a sum that is NaN stays one)
    a.m = m;
    if (b.token >= 0 && (a.token < 0 || b.best > a.best)) { a.best = b.best; a.z = b.z; a.token = b.token; }
    if (b.given == b.given) a.given = b.given;
}

__global__ void __launch_bounds__(kThreads) vocab_scores_kernel(const ScoreParams p) {
    __shared__ float sx[kStep][kTile + 1], sw[kStep][kTile + 1];
    pdl_launch_dependents();
    pdl_wait();
    const int row0 = blockIdx.x * kTile, n0 = blockIdx.y * kTile, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < p.dim; k0 += kStep) {
        for (int i = threadIdx.x; i < kTile * kStep; i += kThreads) {
            const int r = i / kStep, k = i % kStep;
            sx[k][r] = row0 + r < p.rows && k0 + k < p.dim ? __bfloat162float(p.x[(row0 + r) * p.ldx + k0 + k]) : 0.f;
            sw[k][r] = n0 + r < p.vocab && k0 + k < p.dim ? __bfloat162float(p.w[(n0 + r) * p.ldw + k0 + k]) : 0.f;
        }
        __syncthreads();
        for (int k = 0; k < kStep; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sx[k][ty * 4 + i], sw[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
    const uint32_t seed = p.seed_at ? *p.seed_at : p.seed;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        const int row = row0 + ty * 4 + i;
        const int target = p.target && row < p.rows ? p.target[row] : -1;
        Part a = {-INFINITY, 0.f, -INFINITY, 0.f, -1, NAN};
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tx * 4 + j;
            if (n >= p.vocab || row >= p.rows) break;
            float z = acc[i][j] + (p.bias ? p.bias[n] : 0.f);
            if (p.cap > 0.f) z = p.cap * tanhf(z / p.cap);
            const Part b = {z != z ? 0.f : z, z != z ? z : z == -INFINITY ? 0.f : 1.f, p.inv_t > 0.f ? z * p.inv_t + gumbel(seed, row, n) : z, z, n, n == target ? z : NAN};
            join(a, b);
        }
#pragma unroll
        for (int o = 1; o < 16; o *= 2) {   // the lane in front has the tokens in front
            Part b = {__shfl_down_sync(0xffffffffu, a.m, o), __shfl_down_sync(0xffffffffu, a.l, o), __shfl_down_sync(0xffffffffu, a.best, o),
                      __shfl_down_sync(0xffffffffu, a.z, o), __shfl_down_sync(0xffffffffu, a.token, o), __shfl_down_sync(0xffffffffu, a.given, o)};
            if (tx + o < 16) join(a, b);
        }
        if (tx == 0 && row < p.rows) p.parts[(size_t)row * p.n_parts + blockIdx.y] = a;
    }
}

__global__ void __launch_bounds__(kThreads) vocab_join_kernel(const ScoreParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= p.rows) return;
    const Part* parts = p.parts + (size_t)row * p.n_parts;
    const int per = (p.n_parts + 31) / 32;
    Part a = {-INFINITY, 0.f, -INFINITY, 0.f, -1, NAN};
    for (int i = lane * per; i < min((lane + 1) * per, p.n_parts); ++i) join(a, parts[i]);
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        Part b = {__shfl_down_sync(0xffffffffu, a.m, o), __shfl_down_sync(0xffffffffu, a.l, o), __shfl_down_sync(0xffffffffu, a.best, o),
                  __shfl_down_sync(0xffffffffu, a.z, o), __shfl_down_sync(0xffffffffu, a.token, o), __shfl_down_sync(0xffffffffu, a.given, o)};
        if (lane + o < 32) join(a, b);
    }
    if (lane) return;
    const float log_l = logf(a.l);
    if (p.lse) p.lse[row] = a.m + log_l;
    if (p.pick) p.pick[row] = a.token;
    if (p.pick_logprob) p.pick_logprob[row] = a.z - a.m - log_l;
    if (p.logprob) {
        const int target = p.target ? p.target[row] : -1;
        if (target >= p.vocab) atomicExch(p.status, 2);
        p.logprob[row] = target < 0 ? 0.f : a.given - a.m - log_l;
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" {

size_t gptrs_cuda_vocab_scores_scratch_bytes(const gptrs_vocab_scores* s) {
    if (!s || s->rows < 1 || s->vocab < 1) return 0;
    return (size_t)s->rows * ceil_div(s->vocab, kTile) * sizeof(Part);
}

int gptrs_cuda_vocab_scores(const gptrs_vocab_scores* s, void* stream) {
    GPTRS_REQUIRE(s && s->d_weight && s->d_status && (s->rows == 0 || s->d_hidden), "null pointer");
    GPTRS_REQUIRE(s->rows >= 0 && s->rows <= 0x3fffffff && s->vocab >= 1 && s->vocab <= 0x3fffffff && s->dim >= 8 && s->dim <= 0x3fffffff, "bad sizes");
    ScoreParams p = {};
    p.ldx = s->ldh ? s->ldh : s->dim;
    p.ldw = s->ldw ? s->ldw : s->dim;
    GPTRS_REQUIRE(s->dim % 8 == 0 && p.ldx % 8 == 0 && p.ldw % 8 == 0 && p.ldx >= s->dim && p.ldw >= s->dim && p.ldx < ((int64_t)1 << 31) && p.ldw < ((int64_t)1 << 31),
                  "dim and the strides must be multiples of 8, and rows must not overlap");
    GPTRS_REQUIRE(aligned16(s->d_hidden) && aligned16(s->d_weight) && aligned16(s->d_scratch), "pointers must be 16-byte aligned");
    GPTRS_REQUIRE(s->temperature == s->temperature && s->soft_cap >= 0.f && s->soft_cap < 3e38f, "bad temperature or soft cap");
    GPTRS_REQUIRE(!s->d_logprob || s->d_target, "log-probabilities of targets need targets");
    GPTRS_REQUIRE(s->rows == 0 || (s->d_scratch && s->scratch_bytes >= gptrs_cuda_vocab_scores_scratch_bytes(s)), "scratch is too small");
    if (s->rows == 0) return GPTRS_OK;
    p.x = static_cast<const __nv_bfloat16*>(s->d_hidden); p.w = static_cast<const __nv_bfloat16*>(s->d_weight);
    p.bias = s->d_bias; p.seed_at = s->d_seed; p.target = s->d_target;
    p.parts = static_cast<Part*>(s->d_scratch);
    p.pick = s->d_pick; p.pick_logprob = s->d_pick_logprob; p.logprob = s->d_logprob; p.lse = s->d_lse; p.status = s->d_status;
    p.rows = (int)s->rows; p.dim = (int)s->dim; p.vocab = (int)s->vocab; p.n_parts = ceil_div(s->vocab, kTile);
    p.cap = s->soft_cap; p.inv_t = s->temperature > 0.f ? 1.f / s->temperature : 0.f; p.seed = s->seed;
    const int rc = launch_kernel(vocab_scores_kernel, dim3((unsigned)ceil_div(p.rows, kTile), (unsigned)p.n_parts), dim3(kThreads), 0, as_stream(stream), 1, p);
    if (rc) return rc;
    return launch_kernel(vocab_join_kernel, dim3((unsigned)ceil_div(p.rows, kThreads / 32)), dim3(kThreads), 0, as_stream(stream), 1, p);
}

}  // extern "C"
