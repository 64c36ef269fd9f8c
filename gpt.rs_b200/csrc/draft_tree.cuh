// Trees of drafted tokens over the paged bf16 cache: the arguments that append, attention and acceptance share, and how a kernel reads them.
//
// pool[page][kv head][keys, values][16 tokens][128 channels] in bf16, the 16-byte chunk c of token t at c ^ (t & 7) (paged_attention.cu). Node i of a
// tree lies at position length + i of its slot.
#pragma once
#include "common.cuh"

namespace gptrs {

constexpr int kTreeDim = 128;
constexpr int kTreePage = 16;                            // tokens of a page
constexpr int kTreeBlock = kTreePage * kTreeDim * 2;     // bytes of the keys or values of a page and kv head
constexpr int kMostNodes = 256;

struct DraftTrees {
    const int *first, *slot, *length, *parent, *table;
    long long n_pages;
    int n_trees, rows, n_slots, max_pages, q_heads, kv_heads, group, max_nodes;
};
// Checks what a host can see and fills in the kernels' view.
int draft_trees(const gptrs_draft_trees* t, DraftTrees* out);   // tree_cache.cu

#ifdef __CUDACC__
struct TreeSpan { int slot, row0, nodes, length; };      // slot < 0: padding, nodes = 0
__device__ __forceinline__ TreeSpan tree_span(const DraftTrees& t, int s, int* status) {
    TreeSpan r = {t.slot[s], t.first[s], t.first[s + 1], t.length[s]};
    r.nodes -= r.row0;
    if (r.slot < 0) return {-1, 0, 0, 0};
    if (r.slot >= t.n_slots || r.row0 < 0 || r.nodes < 0 || r.row0 > t.rows - r.nodes || r.nodes > t.max_nodes || r.length < 0 ||
        r.length > t.max_pages * kTreePage - r.nodes) {
        atomicExch(status, 2);
        return {-1, 0, 0, 0};
    }
    return r;
}
__device__ __forceinline__ int tree_parent_of(int up, int i, int* status) {
    if (up >= -1 && up < i) return up;
    atomicExch(status, 2);
    return -1;
}
__device__ __forceinline__ int tree_parent(const DraftTrees& t, const TreeSpan& s, int i, int* status) { return tree_parent_of(t.parent[s.row0 + i], i, status); }
// First byte of the keys of (position, kv head 0) in a pool; -1: its page is out of range.
__device__ __forceinline__ long long tree_place(const DraftTrees& t, int slot, int position, int* status) {
    const int page = t.table[(long long)slot * t.max_pages + position / kTreePage];
    if (page >= 0 && page < t.n_pages) return (long long)page * t.kv_heads * (2 * kTreeBlock) + position % kTreePage * (2 * kTreeDim);
    atomicExch(status, 2);
    return -1;
}
#endif

}  // namespace gptrs
