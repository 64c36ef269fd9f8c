// The paged KV cache in 8 bits: layout of its blocks, and how a warp turns them into operands of mma.m16n8k16 (f16).
//
// A whole number of 8 bits is exact in f16 (11 bits), so products with keys and values lose nothing but the query's and the probability's
// rounding; the block's scale is applied to f32 results. A byte becomes f16 without a conversion instruction: 0x6400 | u is 1024 + u, and
// subtracting 1152 leaves u - 128 (a permute and a subtraction per two values).
#pragma once
#include "common.cuh"

namespace gptrs {

int kv8_check(const gptrs_kv8_cache* c);   // that gptrs_cuda_kv8_layout has filled it in (kv8_append.cu)

constexpr int kKv8Tokens = 16;             // of a block
constexpr float kKv8MinScale = 8.673617379884035e-19f;   // 2^-60: keeps 1 / scale and log2(scale) finite
constexpr float kKv8Log2e = 1.4426950408889634f;

__host__ __device__ constexpr long long kv8_block_bytes(int dim) { return 32ll * dim + 16; }
__host__ __device__ constexpr long long kv8_open_elems(int kv_heads, int dim) { return 2ll * kv_heads * 2 * kKv8Tokens * dim; }   // of a slot
// byte of a key / value of a block
__host__ __device__ constexpr int kv8_key_at(int token, int d) { return d / 32 * 512 + (token & 7) * 64 + d % 32 / 8 * 16 + (token >> 3) * 8 + (d & 7); }
__host__ __device__ constexpr int kv8_value_at(int token, int d, int dim) {
    return 16 * dim + d / 32 * 512 + (d & 7) * 64 + (token & 7) / 2 * 16 + d % 32 / 8 * 4 + (token >> 3) * 2 + (token & 1);
}
// open rows of a slot: first element of (block, kv head, keys or values)
__host__ __device__ constexpr long long kv8_open_at(int block, int kv_heads, int head, int is_value, int dim) {
    return (((long long)(block & 1) * kv_heads + head) * 2 + is_value) * kKv8Tokens * dim;
}

// The page of a block: its number, or -1 (with code 2 in the status word where the table holds a number that is none).
__device__ __forceinline__ int kv8_page(const int* table, int slot, long long max_pages, int block, long long n_pages, int* status) {
    const int page = table[slot * max_pages + block];
    if (page < n_pages) return page < 0 ? -1 : page;
    atomicExch(status, 2);
    return -1;
}

__device__ __forceinline__ uint32_t hsub2_bits(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// four bytes -> two pairs of f16
__device__ __forceinline__ void kv8_widen(uint32_t bytes, uint32_t* lo, uint32_t* hi) {
    *lo = hsub2_bits(__byte_perm(bytes, 0x64646464u, 0x4140), 0x64806480u);
    *hi = hsub2_bits(__byte_perm(bytes, 0x64646464u, 0x4342), 0x64806480u);
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
// D(16x8,f32) += A(16x16,f16,row) * B(16x8,f16,col)
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {   // 8 x 8 of 16 bits, a row of pairs per 4 lanes -> transposed
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float kv8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// Values of 16 bits (bf16) of one operand -> f16 with a power of two in front, chosen so that the largest lies in [1, 2): exact for everything
// down to 2^-14 of it, and off by at most 2^-25 of it below. The exponent field of the largest |x|, from the bits of its bf16:
__device__ __forceinline__ int pow2_exponent(uint32_t largest_abs_bits) {   // -60 .. 126; 128: not finite
    if (largest_abs_bits >= 0x7f80u) return 128;
    return max((int)(largest_abs_bits >> 7) - 127, -60);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }   // -126 .. 127
__device__ __forceinline__ uint32_t abs_bits_max2(uint32_t a, uint32_t b) { return __vmaxu2(a & 0x7fff7fffu, b & 0x7fff7fffu); }
// The halves of v that are not finite become zero; ones in their place.
__device__ __forceinline__ uint32_t drop_not_finite(uint32_t& v) {
    const uint32_t none = __vcmpgeu2(v & 0x7fff7fffu, 0x7f807f80u);
    v &= ~none;
    return none;
}
__device__ __forceinline__ uint32_t widest_half(uint32_t v) { return max(v & 0xffffu, v >> 16); }
__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t v, float factor) { return pack_f16x2(bf16_lo(v) * factor, bf16_hi(v) * factor); }

}  // namespace gptrs
