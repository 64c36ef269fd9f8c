// Trees of drafted tokens: rotation and append to the paged bf16 cache, and what becomes of the cache when a path through the tree is accepted.
#include "draft_tree.cuh"

namespace gptrs {

int draft_trees(const gptrs_draft_trees* t, DraftTrees* out) {
    GPTRS_REQUIRE(t, "null pointer");
    GPTRS_REQUIRE(t->dim == kTreeDim, "trees over the paged bf16 cache need dim 128");
    GPTRS_REQUIRE(t->q_heads > 0 && t->kv_heads > 0 && t->q_heads % t->kv_heads == 0 && t->q_heads / t->kv_heads <= 32 && t->q_heads <= 4096, "bad head counts");
    GPTRS_REQUIRE(t->scale >= 0.f && t->scale < 3e38f, "the scale of the scores must be positive (0: 1 / sqrt(dim))");
    GPTRS_REQUIRE(t->max_nodes >= 1 && t->max_nodes <= kMostNodes, "max_nodes must be 1 .. 256");
    GPTRS_REQUIRE(t->n_trees >= 0 && t->n_trees <= 65535 && t->rows >= 0 && t->rows <= t->n_trees * kMostNodes, "bad number of trees or rows");
    GPTRS_REQUIRE(t->n_trees == 0 || (t->d_first && t->d_slot && t->d_length && t->d_page_table), "null pointer");
    GPTRS_REQUIRE(t->rows == 0 || t->d_parent, "null pointer");
    GPTRS_REQUIRE(t->max_pages >= 1 && t->max_pages * kTreePage < ((int64_t)1 << 31) && t->n_slots >= 1 && t->n_slots <= 0x7fffffff && t->n_pages >= 1 && t->n_pages <= 0x7fffffff,
                  "bad cache sizes");
    *out = {t->d_first, t->d_slot, t->d_length, t->d_parent, t->d_page_table, t->n_pages, (int)t->n_trees, (int)t->rows, (int)t->n_slots, (int)t->max_pages, t->q_heads,
            t->kv_heads, t->q_heads / t->kv_heads, t->max_nodes};
    return GPTRS_OK;
}

namespace {

constexpr int kThreads = 256;

struct AppendParams {
    DraftTrees t;
    const __nv_bfloat16* qkv;
    long long ld;
    const float *cos, *sin;
    int half, positions;          // rotated pairs (a multiple of 8), rows of the tables
    __nv_bfloat16* q;
    unsigned char* pool;
    int* status;
};

// A CTA per node. A thread takes two chunks of eight channels of a head: a pair that rotates together (c, c + half / 8), or two that stay. Rows, parents and the page are asked for
// together, in front of the walk up the tree (shared reads, where global ones would wait for each other): what bounds a small call is the two trips to memory, tree and row.
// 64 trees of 20 to 64 nodes, 32 / 8 heads: 14.3 us, 10 at the rate of a copy (256 threads, two tasks in front 16.2; with the rows behind
// the walk 17.5; 64 threads 14.3); one tree of 26 nodes 2.7, a launch (64 threads 3.7). 40 / 8, 64 / 8 and 12 / 12 heads 16.6, 21.5 and 12.4: tasks beyond three a thread, 48 heads, are
// loaded behind the walk. (Kernels in a graph; a call from Python by itself takes 2 us more.)
constexpr int kAppendThreads = 128, kAhead = 3;   // tasks of a thread that are asked for in front
__global__ void __launch_bounds__(kAppendThreads) tree_append_kernel(const AppendParams p) {
    __shared__ int up[kMostNodes];
    pdl_launch_dependents();
    pdl_wait();
    const int node = blockIdx.x, tid = threadIdx.x;
    const TreeSpan s = tree_span(p.t, blockIdx.y, p.status);
    if (node >= s.nodes) return;   // the whole CTA
    const int heads = p.t.q_heads + 2 * p.t.kv_heads, row = s.row0 + node, turning = p.half / 8, tasks = heads * 8;
    const uint4* src = reinterpret_cast<const uint4*>(p.qkv + row * p.ld);
    auto chunks = [&](int i, int* c0, int* c1) {
        const int k = i & 7;
        *c0 = k < turning ? k : 2 * k;
        *c1 = k < turning ? k + turning : 2 * k + 1;
    };
    uint4 a[kAhead], b[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const int i = tid + j * kAppendThreads;
        int c0, c1;
        chunks(i, &c0, &c1);
        if (i < tasks) { a[j] = src[(i >> 3) * 16 + c0]; b[j] = src[(i >> 3) * 16 + c1]; }
    }
    int parent[kMostNodes / kAppendThreads];
#pragma unroll
    for (int j = 0; j < kMostNodes / kAppendThreads; ++j) parent[j] = tid + j * kAppendThreads <= node ? p.t.parent[s.row0 + tid + j * kAppendThreads] : -1;
    const long long place = tree_place(p.t, s.slot, s.length + node, p.status);
#pragma unroll
    for (int j = 0; j < kMostNodes / kAppendThreads; ++j) up[tid + j * kAppendThreads] = tree_parent_of(parent[j], tid + j * kAppendThreads, p.status);
    __syncthreads();
    int at = s.length;
    for (int i = up[node]; i >= 0; i = up[i]) ++at;   // (a parent is below its child: this ends)
    if (at >= p.positions && p.half > 0) { atomicExch(p.status, 2); at = 0; }
    auto finish = [&](int i, uint4 a, uint4 b) {
        const int head = i >> 3, k = i & 7;
        const bool is_q = head < p.t.q_heads, is_v = head >= p.t.q_heads + p.t.kv_heads;
        int c0, c1;
        chunks(i, &c0, &c1);
        if (k < turning && !is_v) {
            const float *cos = p.cos + (long long)at * p.half + 8 * k, *sin = p.sin + (long long)at * p.half + 8 * k;
            uint32_t *aw = &a.x, *bw = &b.x;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float4 c = reinterpret_cast<const float4*>(cos)[j], n = reinterpret_cast<const float4*>(sin)[j];
                const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float a0 = bf16_lo(aw[2 * j + h]), a1 = bf16_hi(aw[2 * j + h]), b0 = bf16_lo(bw[2 * j + h]), b1 = bf16_hi(bw[2 * j + h]);
                    aw[2 * j + h] = pack_bf16x2(a0 * cs[2 * h] - b0 * sn[2 * h], a1 * cs[2 * h + 1] - b1 * sn[2 * h + 1]);
                    bw[2 * j + h] = pack_bf16x2(b0 * cs[2 * h] + a0 * sn[2 * h], b1 * cs[2 * h + 1] + a1 * sn[2 * h + 1]);
                }
            }
        }
        if (is_q) {
            uint4* dst = reinterpret_cast<uint4*>(p.q) + ((long long)row * p.t.q_heads + head) * 16;
            dst[c0] = a;
            dst[c1] = b;
        } else if (place >= 0) {
            const int kv = is_v ? head - p.t.q_heads - p.t.kv_heads : head - p.t.q_heads, turn = (s.length + node) & 7;
            unsigned char* dst = p.pool + place + (2 * kv + is_v) * kTreeBlock;
            *reinterpret_cast<uint4*>(dst + ((c0 ^ turn) << 4)) = a;
            *reinterpret_cast<uint4*>(dst + ((c1 ^ turn) << 4)) = b;
        }
    };
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        if (tid + j * kAppendThreads < tasks) finish(tid + j * kAppendThreads, a[j], b[j]);
    for (int i = tid + kAhead * kAppendThreads; i < tasks; i += kAppendThreads) {
        int c0, c1;
        chunks(i, &c0, &c1);
        finish(i, src[(i >> 3) * 16 + c0], src[(i >> 3) * 16 + c1]);
    }
}

struct AcceptParams {
    DraftTrees t;
    const int *token, *pick;
    void* const* pools;
    int n_layers;
    int *count, *path, *next, *new_length;
    int* status;
};

// A CTA per (layer, tree); each walks the tree by itself. The k-th node of the path comes from a place behind k (numbers grow along a path), so a thread that moves one column
// of chunks in the order of k never reads what it has written. What bounds it is latency: loads of the walk, table, pool. 64 trees with nine nodes accepted, 26 layers, 8 kv heads 14.7
// us (7.3 at the rate of a copy); one tree 3.9 (kernels in a graph; a call from Python by itself takes 2 us more). Several layers to a CTA, so that fewer walk, 21.3.
__global__ void __launch_bounds__(kThreads, 8) tree_accept_kernel(const AcceptParams p) {
    __shared__ int pick[kMostNodes], follow[kMostNodes], path[kMostNodes];
    __shared__ long long from[kMostNodes], to[kMostNodes];
    static_assert(kThreads >= kMostNodes, "a thread per node");
    pdl_launch_dependents();
    pdl_wait();
    const int s = blockIdx.y, tid = threadIdx.x;
    const TreeSpan span = tree_span(p.t, s, p.status);
    int up = -1, token = 0;
    if (tid < span.nodes) {
        up = tree_parent(p.t, span, tid, p.status);
        token = p.token[span.row0 + tid];
        pick[tid] = p.pick[span.row0 + tid];
    }
    follow[tid] = kMostNodes;
    __syncthreads();
    if (up >= 0 && token == pick[up]) atomicMin(&follow[up], tid);   // the lowest child that its parent's pick agrees with
    __syncthreads();
    int count = 0, last = 0;
    if (span.nodes > 0)
        for (int i = 0; i < kMostNodes; i = follow[i]) {
            if (tid == 0) path[count] = i;
            last = i;
            ++count;
        }
    __syncthreads();
    if (blockIdx.x == 0) {
        if (tid < p.t.max_nodes) p.path[(long long)s * p.t.max_nodes + tid] = tid < count ? path[tid] : -1;
        if (tid == 0) {
            p.count[s] = count;
            p.next[s] = count ? pick[last] : -1;
            p.new_length[s] = p.t.length[s] + count;
        }
    }
    if (p.n_layers == 0 || count < 2) return;
    if (tid < count) {
        const bool moves = path[tid] != tid;
        from[tid] = moves ? tree_place(p.t, span.slot, span.length + path[tid], p.status) : -1;
        to[tid] = moves ? tree_place(p.t, span.slot, span.length + tid, p.status) : -1;
    }
    __syncthreads();
    unsigned char* pool = static_cast<unsigned char*>(p.pools[blockIdx.x]);
    constexpr int kAtOnce = 4;   // with eight, and the registers for them, half as many CTAs are there at a time: 64 trees, 26 layers 18.4 us instead of 14.7
    for (int col = tid; col < p.t.kv_heads * 32; col += kThreads) {
        unsigned char* base = pool + (col >> 4) * kTreeBlock;
        const int chunk = col & 15;
        for (int k0 = 1; k0 < count; k0 += kAtOnce) {
            uint4 v[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int k = k0 + j;
                if (k < count && from[k] >= 0 && to[k] >= 0) v[j] = *reinterpret_cast<const uint4*>(base + from[k] + ((chunk ^ ((span.length + path[k]) & 7)) << 4));
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const int k = k0 + j;
                if (k < count && from[k] >= 0 && to[k] >= 0) *reinterpret_cast<uint4*>(base + to[k] + ((chunk ^ ((span.length + k) & 7)) << 4)) = v[j];
            }
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" {

int gptrs_cuda_tree_append(const gptrs_draft_trees* t, const gptrs_tree_append_step* s, void* stream) {
    AppendParams p = {};
    const int rc = draft_trees(t, &p.t);
    if (rc) return rc;
    GPTRS_REQUIRE(s && s->d_pool && s->d_status && (t->rows == 0 || (s->d_qkv && s->d_q)), "null pointer");
    GPTRS_REQUIRE(s->rotary_dim >= 0 && s->rotary_dim <= kTreeDim && s->rotary_dim % 16 == 0, "rotary_dim must be a multiple of 16, at most 128");
    GPTRS_REQUIRE(s->rotary_dim == 0 || (s->d_cos && s->d_sin && s->positions >= 1 && s->positions <= 0x7fffffff), "rotary tables missing");
    GPTRS_REQUIRE(aligned16(s->d_qkv) && aligned16(s->d_q) && aligned16(s->d_pool) && aligned16(s->d_cos) && aligned16(s->d_sin), "pointers must be 16-byte aligned");
    const int64_t width = (int64_t)(t->q_heads + 2 * t->kv_heads) * kTreeDim, out_width = (int64_t)t->q_heads * kTreeDim;
    p.ld = s->ld ? s->ld : width;
    GPTRS_REQUIRE(p.ld >= width && p.ld % 8 == 0 && p.ld < ((int64_t)1 << 31), "rows of qkv overlap, or do not start at multiples of 16 bytes");
    if (t->rows == 0) return GPTRS_OK;
    const char *in = static_cast<const char*>(s->d_qkv), *out = static_cast<const char*>(s->d_q);
    GPTRS_REQUIRE(out >= in + 2 * ((t->rows - 1) * p.ld + width) || in >= out + 2 * t->rows * out_width, "the queries lie in rows of qkv");
    p.qkv = static_cast<const __nv_bfloat16*>(s->d_qkv);
    p.cos = s->d_cos; p.sin = s->d_sin;
    p.half = (int)s->rotary_dim / 2; p.positions = (int)s->positions;
    p.q = static_cast<__nv_bfloat16*>(s->d_q);
    p.pool = static_cast<unsigned char*>(s->d_pool);
    p.status = s->d_status;
    return launch_kernel(tree_append_kernel, dim3((unsigned)t->max_nodes, (unsigned)t->n_trees), dim3(kAppendThreads), 0, as_stream(stream), 1, p);
}

int gptrs_cuda_tree_accept(const gptrs_draft_trees* t, const gptrs_tree_accept_step* s, void* stream) {
    AcceptParams p = {};
    const int rc = draft_trees(t, &p.t);
    if (rc) return rc;
    GPTRS_REQUIRE(s && s->d_status && (t->rows == 0 || (s->d_token && s->d_pick)), "null pointer");
    GPTRS_REQUIRE(t->n_trees == 0 || (s->d_count && s->d_path && s->d_next && s->d_new_length), "null pointer");
    GPTRS_REQUIRE(s->n_layers >= 0 && s->n_layers <= 65535 && (s->n_layers == 0 || s->d_pools), "bad number of layers");
    GPTRS_REQUIRE(t->n_trees == 0 || s->d_new_length >= t->d_length + t->n_trees || t->d_length >= s->d_new_length + t->n_trees, "the new lengths lie where the lengths are read");
    if (t->n_trees == 0) return GPTRS_OK;
    p.token = s->d_token; p.pick = s->d_pick;
    p.pools = s->d_pools; p.n_layers = (int)s->n_layers;
    p.count = s->d_count; p.path = s->d_path; p.next = s->d_next; p.new_length = s->d_new_length;
    p.status = s->d_status;
    return launch_kernel(tree_accept_kernel, dim3((unsigned)(s->n_layers ? s->n_layers : 1), (unsigned)t->n_trees), dim3(kThreads), 0, as_stream(stream), 1, p);
}

}  // extern "C"
