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
    if (r.pair_axis == nullptr) {
        long long pos = r.axis_positions ? r.axis_positions[row] : position;
        if (pos < 0 || pos >= r.positions) { atomicExch(status, 2); pos = 0; }
        load_vec(cos + pos * r.rot_half, c);
        load_vec(sin + pos * r.rot_half, s);
    } else {
#pragma unroll
        for (int k = 0; k < kVec; ++k) {
            const int axis = r.pair_axis[i + k];
            long long pos = -1;
            if (axis < r.axes) pos = r.axis_positions ? r.axis_positions[axis * r.axis_stride + row] : position;
            if (pos < 0 || pos >= r.positions) { atomicExch(status, 2); pos = 0; }
            c[k] = cos[pos * r.rot_half + k];
            s[k] = sin[pos * r.rot_half + k];
        }
    }
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
// sum over the `lanes` (a power of two) neighbouring lanes of a head
__device__ __forceinline__ float lane_group_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

#endif  // __CUDACC__

}  // namespace gptrs
