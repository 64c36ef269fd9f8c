// Norm and rotation of one head of a projection row, shared by gptrs_cuda_qk_norm_rope and the append to the 8-bit cache.
//
// A head is dim / 2 pairs of channels: pair i < rot_half is rotated and is (i, i + rot_half) or (2 i, 2 i + 1), a later one is (2 i, 2 i + 1) and
// stays. A lane takes kVec consecutive pairs, two runs of kVec consecutive channels each: [i ..], [i + rot_half ..] of rotated halves, [2 i ..],
// [2 i + kVec ..] else. So both loads are as wide as a row allows and no value crosses lanes but for the sum of squares.
#pragma once
#include "common.cuh"

namespace gptrs {

struct QkRotation {
    int q_heads, kv_heads, dim, rot_half, neighbours, axes;
    float eps;
    const float *q_gain, *k_gain, *cos, *sin;
    long long positions, axis_stride;
    const int* axis_positions;
    const unsigned char* pair_axis;
};
// Checks a rotation and fills in the form the kernels take (qk_rotate.cu). rows: of the call, for axis_stride 0.
int qk_rotation_of(const gptrs_qk_rotation& r, int64_t rows, QkRotation* out);

#ifdef __CUDACC__

__device__ __forceinline__ void load_vec(const float* p, float (&v)[4]) {
    const float4 x = *reinterpret_cast<const float4*>(p);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(x.x); v[1] = bf16_hi(x.x); v[2] = bf16_lo(x.y); v[3] = bf16_hi(x.y);
}
// kVec consecutive values as they come from memory, and as floats
template <typename T, int kVec> struct RawVec;
template <> struct RawVec<__nv_bfloat16, 8> {
    uint4 x;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { x = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = x; }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
    }
};
template <> struct RawVec<__nv_bfloat16, 4> {
    uint2 x;
    __device__ __forceinline__ void load(const __nv_bfloat16* p) { x = *reinterpret_cast<const uint2*>(p); }
    __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint2*>(p) = x; }
    __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = bf16_lo(x.x); v[1] = bf16_hi(x.x); v[2] = bf16_lo(x.y); v[3] = bf16_hi(x.y); }
};
template <> struct RawVec<float, 4> {
    float4 x;
    __device__ __forceinline__ void load(const float* p) { x = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<float4*>(p) = x; }
    __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
};
__device__ __forceinline__ void load_vec(const float* p, float (&v)[8]) {
    const float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + 4);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void load_vec(const float* p, float (&v)[1]) { v[0] = *p; }
__device__ __forceinline__ void load_vec(const __nv_bfloat16* p, float (&v)[1]) { v[0] = __bfloat162float(*p); }
__device__ __forceinline__ void store_vec(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[4]) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
__device__ __forceinline__ void store_vec(float* p, const float (&v)[1]) { *p = v[0]; }
__device__ __forceinline__ void store_vec(__nv_bfloat16* p, const float (&v)[1]) { *p = __float2bfloat16_rn(v[0]); }

// first channels of a lane's two runs, for its first pair i
template <int kVec>
__device__ __forceinline__ void pair_channels(const QkRotation& r, int i, int* ca, int* cb) {
    const bool apart = !r.neighbours && i < r.rot_half;
    *ca = apart ? i : 2 * i;
    *cb = apart ? i + r.rot_half : 2 * i + kVec;
}

// cos and sin of the pairs i .. i + kVec - 1 at a row; (1, 0) for pairs that stay
template <int kVec>
__device__ __forceinline__ void pair_angles(const QkRotation& r, int row, int position, int i, int* status, float (&c)[kVec], float (&s)[kVec]) {
    if (i >= r.rot_half) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) { c[k] = 1.f; s[k] = 0.f; }
        return;
    }
    const float *cos = r.cos + i, *sin = r.sin + i;
    bool bad = false;   // (reported behind the loads: an atomic in between would keep the next ones waiting)
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
        const int axis = r.pair_axis ? r.pair_axis[i + k] : 0;
        long long pos = -1;
        if (axis < r.axes) pos = r.axis_positions ? r.axis_positions[axis * r.axis_stride + row] : position;
        if (pos < 0 || pos >= r.positions) { bad = true; pos = 0; }
        c[k] = cos[pos * r.rot_half + k];
        s[k] = sin[pos * r.rot_half + k];
    }
    if (bad) atomicExch(status, 2);
}

// the rotation of a lane's pairs, whose channels are `apart` (pair k = a[k], b[k]) or neighbours
template <int kVec>
__device__ __forceinline__ void rotate_pairs(bool apart, float (&a)[kVec], float (&b)[kVec], const float (&c)[kVec], const float (&s)[kVec]) {
    if (kVec == 1 || apart) {
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
            const float x = a[k], y = b[k];
            a[k] = x * c[k] - y * s[k];
            b[k] = y * c[k] + x * s[k];
        }
    } else {
#pragma unroll
        for (int k = 0; k < kVec; k += 2) {
            constexpr int h = kVec / 2;
            const float x = a[k], y = a[k + 1], u = b[k], v = b[k + 1];
            a[k] = x * c[k / 2] - y * s[k / 2];
            a[k + 1] = y * c[k / 2] + x * s[k / 2];
            b[k] = u * c[h + k / 2] - v * s[h + k / 2];
            b[k + 1] = v * c[h + k / 2] + u * s[h + k / 2];
        }
    }
}

template <int kVec>
__device__ __forceinline__ float square_sum(const float (&a)[kVec], const float (&b)[kVec]) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < kVec; ++k) t += a[k] * a[k] + b[k] * b[k];
    return t;
}
template <int kVec>
__device__ __forceinline__ void times_gain(const float* gain, int ca, int cb, float r, float (&a)[kVec], float (&b)[kVec]) {
    float ga[kVec], gb[kVec];
    load_vec(gain + ca, ga);
    load_vec(gain + cb, gb);
#pragma unroll
    for (int k = 0; k < kVec; ++k) { a[k] = a[k] * r * ga[k]; b[k] = b[k] * r * gb[k]; }
}
// With gains g and angles (c, s) of pairs apart, out_a = r (x_a g_a c - x_b g_b s) and out_b = r (x_b g_b c + x_a g_a s): the four products of gains and angles
// are made once for several heads, two pairs at a time.
template <int kVec>
struct Turn {
    uint64_t ac[kVec / 2], bs[kVec / 2], bc[kVec / 2], as[kVec / 2];
    // gain NULL: no norm; turned false: angles (1, 0)
    __device__ __forceinline__ void set(const float* gain, int ca, int cb, bool turned, const float* cos, const float* sin) {
        float ga[kVec], gb[kVec], c[kVec], s[kVec];
#pragma unroll
        for (int k = 0; k < kVec; ++k) { ga[k] = gb[k] = c[k] = 1.f; s[k] = 0.f; }
        if (gain) { load_vec(gain + ca, ga); load_vec(gain + cb, gb); }
        if (turned) { load_vec(cos, c); load_vec(sin, s); }
#pragma unroll
        for (int k = 0; k < kVec / 2; ++k) {
            const uint64_t c2 = pair_of(c[2 * k], c[2 * k + 1]), s2 = pair_of(s[2 * k], s[2 * k + 1]);
            const uint64_t a2 = pair_of(ga[2 * k], ga[2 * k + 1]), b2 = pair_of(gb[2 * k], gb[2 * k + 1]);
            ac[k] = mul2(a2, c2); as[k] = mul2(a2, s2); bc[k] = mul2(b2, c2); bs[k] = mul2(b2, s2) ^ 0x8000000080000000ull;
        }
    }
    __device__ __forceinline__ void apply(float (&a)[kVec], float (&b)[kVec], float rms, bool turned) const {
        const uint64_t rms2 = pair_of(rms, rms);
#pragma unroll
        for (int k = 0; k < kVec / 2; ++k) {
            const uint64_t ar = mul2(pair_of(a[2 * k], a[2 * k + 1]), rms2), br = mul2(pair_of(b[2 * k], b[2 * k + 1]), rms2);
            // (a channel that stays does not meet the other one, which may be infinite)
            const float2 x = split(turned ? fma2(ar, ac[k], mul2(br, bs[k])) : mul2(ar, ac[k])), y = split(turned ? fma2(br, bc[k], mul2(ar, as[k])) : mul2(br, bc[k]));
            a[2 * k] = x.x; a[2 * k + 1] = x.y; b[2 * k] = y.x; b[2 * k + 1] = y.y;
        }
    }
};
template <int kVec>
__device__ __forceinline__ float square_sum2(const float (&a)[kVec], const float (&b)[kVec]) {
    uint64_t t = 0;
#pragma unroll
    for (int k = 0; k < kVec / 2; ++k) {
        const uint64_t a2 = pair_of(a[2 * k], a[2 * k + 1]), b2 = pair_of(b[2 * k], b[2 * k + 1]);
        t = fma2(a2, a2, fma2(b2, b2, t));
    }
    const float2 v = split(t);
    return v.x + v.y;
}
// sum over the `lanes` (a power of two) neighbouring lanes of a head
__device__ __forceinline__ float lane_group_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

#endif  // __CUDACC__

}  // namespace gptrs
