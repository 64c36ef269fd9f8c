// What the two attention kernels over the 8-bit cache share: the arguments of a launch and the tokens a row sees.
#pragma once
#include "kv8_cache.cuh"

namespace gptrs {

struct Kv8Attention {
    const __nv_bfloat16* q;
    long long ldq;
    const unsigned char* pool;
    const __nv_bfloat16* open;
    const int *table, *slot, *ctx_len, *length;
    __nv_bfloat16* out;
    float *part_o, *part_ml;      // [row][head][split][dim], [row][head][split][2]
    int* status;
    long long n_pages, max_pages;
    int n_slots, rows, q_heads, kv_heads, group, window, max_len, splits, chunk_blocks;
    float scale_log2;
    const int *tile_row, *tile_rows;
    int n_tiles;
};
int kv8_prompt_attention(const Kv8Attention& p, int dim, cudaStream_t stream);   // tiles of rows (kv8_prompt.cu)

struct Kv8Span { int slot, begin, end, length; };   // visible tokens [begin, end) of a row, and what its sequence has
__device__ __forceinline__ Kv8Span kv8_span(const Kv8Attention& p, int row) {
    Kv8Span s = {p.slot[row], 0, 0, 0};
    if (s.slot < 0) return s;
    if (s.slot >= p.n_slots) { atomicExch(p.status, 2); s.slot = 0; return s; }
    s.length = p.length[s.slot];
    s.end = p.ctx_len[row];
    if (s.end < 0 || s.end > p.max_len || s.end > s.length) { atomicExch(p.status, 2); s.end = max(0, min(min(s.end, p.max_len), s.length)); }
    s.begin = p.window > 0 ? max(0, s.end - p.window) : 0;
    return s;
}

}  // namespace gptrs
