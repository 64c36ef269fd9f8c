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
    int n_tiles, tile_tokens;     // most rows of a tile
    int one_by_one;               // the rows of the tiles go one by one
    int clustered;                // parts of a row are merged by their cluster
};
int kv8_prompt_attention(const Kv8Attention& p, int dim, cudaStream_t stream);   // tiles of rows (kv8_prompt.cu)

// The i-th of the rows that a launch goes through: without tiles row i, else row i % tile_tokens of tile i / tile_tokens; -1: there is none (code 2 for a tile
// that is not within the rows).
__device__ __forceinline__ int kv8_row(const Kv8Attention& p, int i) {
    if (p.n_tiles == 0) return i < p.rows ? i : -1;
    const int tile = i / p.tile_tokens, in_tile = i % p.tile_tokens;
    if (tile >= p.n_tiles) return -1;
    const int row0 = p.tile_row[tile], n_rows = p.tile_rows[tile];
    if (row0 < 0 || n_rows < 0 || n_rows > p.tile_tokens || row0 > p.rows - n_rows) {
        atomicExch(p.status, 2);
        return -1;
    }
    return in_tile < n_rows ? row0 + in_tile : -1;
}

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
