// Norms of queries and keys per head and their rotation in one pass, positions on several axes (see qk_rotate.cuh).
//
// A CTA takes one row; a group of lanes takes a head at a time, all heads of a group with the same angles, which it reads once. With rows of
// 16-byte pieces (kVec 4, up to 256 channels) a lane holds four pairs; other sizes go pair by pair (up to 512 channels). Every value is read
// once and written once; the norm is f32, the result is rounded once.
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
    GPTRS_REQUIRE(r.axes <= 1 || (r.d_axis_positions && r.d_pair_axis), "several axes need their positions and the axis of every pair");
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
    int lanes;    // of a head
};
constexpr int kThreads = 256;

// kRuns: vectors of pairs per lane
template <typename T, int kVec, int kRuns>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const NormRopeParams p) {
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

template <typename T>
int launch_norm_rope(NormRopeParams& p, int64_t rows, cudaStream_t st) {
    const QkRotation& r = p.r;
    auto aligned = [](const void* q, size_t n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; };
    const size_t piece = 4 * sizeof(T);
    const bool wide = r.dim % 8 == 0 && r.dim <= 256 && r.rot_half % 4 == 0 && p.ld_in % 4 == 0 && p.ld_out % 4 == 0 && aligned(p.in, piece) && aligned(p.out, piece) &&
                      aligned(r.cos, 16) && aligned(r.sin, 16) && aligned(r.q_gain, 16) && aligned(r.k_gain, 16);
    const int vectors = r.dim / 2 / (wide ? 4 : 1);
    p.lanes = 1;
    while (p.lanes < vectors && p.lanes < 32) p.lanes *= 2;
    const dim3 grid((unsigned)rows), block(kThreads);
    if (wide) return launch_kernel(qk_norm_rope_kernel<T, 4, 1>, grid, block, 0, st, 1, p);
    return launch_kernel(qk_norm_rope_kernel<T, 1, 8>, grid, block, 0, st, 1, p);
}

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" int gptrs_cuda_qk_norm_rope(const gptrs_qk_rotation* r, const void* d_qkv, int dtype, int64_t ld_in, const int32_t* d_positions, void* d_out,
                                       int64_t ld_out, int32_t* d_status, int64_t rows, void* stream) {
    GPTRS_REQUIRE(r && d_qkv && d_out && d_status, "null pointer");
    GPTRS_REQUIRE(dtype == GPTRS_F32 || dtype == GPTRS_BF16, "rows are f32 or bf16");
    GPTRS_REQUIRE(rows >= 0 && rows <= 0x7fffffff, "bad row count");
    NormRopeParams p = {};
    const int rc = qk_rotation_of(*r, rows, &p.r);
    if (rc) return rc;
    GPTRS_REQUIRE(p.r.rot_half == 0 || p.r.axis_positions || d_positions, "positions are missing");
    const int64_t width = (int64_t)(r->q_heads + 2 * r->kv_heads) * r->dim;
    p.ld_in = ld_in ? ld_in : width;
    p.ld_out = ld_out ? ld_out : width;
    GPTRS_REQUIRE(p.ld_in >= width && p.ld_out >= width, "rows overlap");
    const bool in_place = d_qkv == d_out;
    GPTRS_REQUIRE(!in_place || p.ld_in == p.ld_out, "in place the strides are the same");
    if (rows == 0) return GPTRS_OK;
    p.in = d_qkv; p.out = d_out; p.positions = d_positions; p.status = d_status;
    p.heads = r->q_heads + (in_place ? 1 : 2) * r->kv_heads;
    return dtype == GPTRS_F32 ? launch_norm_rope<float>(p, rows, as_stream(stream)) : launch_norm_rope<__nv_bfloat16>(p, rows, as_stream(stream));
}
