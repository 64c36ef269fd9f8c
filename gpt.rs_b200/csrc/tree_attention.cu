// Attention of trees of drafted tokens over the paged bf16 cache: node i of a tree sees the sequence's tokens, its ancestors and itself.
//
// The rows of a tree and kv head (row = node x group + query head) share the keys that they see, all but the last few dozen, so they are the M side of
// tcgen05 products: a CTA holds a tile of 128 rows and walks over keys in blocks of 64 (four pages), two CTAs to an SM:
//   S[128 x 64] = Q . K^T      both from shared memory (K-major, 128-byte swizzle, which is how the pool holds a page), two accumulators in tensor memory
//   softmax                    warps 0 - 3, a thread per row: running maximum that moves only when a block's maximum is 2^8 above it, weights as bf16 over S
//   O[128 x 128] += P . V      P from tensor memory, V as an MN-major operand
// Warp 4 issues the products, S two blocks ahead of P . V; warps 5 and 6 request the pages of K and V.
// Blocks that reach behind the sequence's tokens are masked by a bit per node: the ancestors of every node of the tile are collected once per tile. In them
// values of nodes that are not finite are taken out of the stage before the product (a weight of 0 does not help there) and added to the rows that
// see them at the end.
//
// Work. A unit is a block of 64 keys of a (tree, kv head, pair of row tiles). Every group of CTAs (two for trees of more than 128 rows, which then share the keys
// through L2; else one) takes the same number of consecutive units, whatever the trees' lengths: where a group begins or ends inside an item, its rows' sums go to
// scratch, and a second kernel joins the parts in the order of the keys. So the result depends on the call alone, not on what runs beside it.
// Every wait is bounded: on a timeout code 3 goes to the status word, the roles leave their loops, tensor memory is freed.
#include "draft_tree.cuh"
#include "umma_common.cuh"

namespace gptrs {

void prefill_tc_fault(int* starve, uint32_t* wait_limit);   // the test switch of paged_prefill_tc.cu

namespace {

constexpr int kRows = 128;
constexpr int kKeys = 64;                       // of a block
constexpr int kPages = kKeys / kTreePage;
constexpr int kSoftmaxWarps = kRows / 32, kMmaWarp = kSoftmaxWarps;
constexpr int kThreads = (kSoftmaxWarps + 3) * 32;
constexpr int kQHalf = kRows * 128;             // bytes of 64 channels of the queries
constexpr int kHalf = kKeys * 128;              // of a block's keys or values
constexpr int kStage = 2 * kHalf;
constexpr uint32_t kTmemCols = 256;             // two S, O
constexpr uint32_t kOCol = 128;
constexpr size_t kSmem = 2 * kQHalf + 4 * kStage + 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLag = 8.f;                     // log2 units that a row's maximum may be ahead of its reference
constexpr float kLargeScore = 1048576.f;        // above it a product and a sum rounded once (fma) are further apart than an exponent may be off
constexpr int kMinUnits = 2;                    // of a group
constexpr int kWords = kMostNodes / 32;

struct Part { long long first, end; int tree, head, round, pad; };   // units of the item that a group begins in
struct Head { long long units; int groups, pad[13]; };

struct AttentionParams {
    CUtensorMap map;
    DraftTrees t;
    const __nv_bfloat16* q;
    long long ldq;
    const unsigned char* pool;
    __nv_bfloat16* out;
    Head* head;
    Part* begins;                // [groups]
    float2* ml;                  // [2 groups tiles][row_cap]: reference and sum of a row; the first of a group's two slots for what others began
    float4* sums;                // [2 groups tiles][32][row_cap]
    int* status;
    float scale_log2;
    int groups, tiles, row_cap;  // tiles: of a group, 1 or 2
    uint32_t wait_limit;
    int starve;
};

__device__ __forceinline__ int blocks_of(const TreeSpan& s) { return (s.length + s.nodes + kKeys - 1) / kKeys; }
__device__ __forceinline__ int rounds_of(const AttentionParams& p, const TreeSpan& s) { return (s.nodes * p.t.group + kRows * p.tiles - 1) / (kRows * p.tiles); }
__device__ __forceinline__ long long units_of(const AttentionParams& p, const TreeSpan& s) { return s.nodes == 0 ? 0 : (long long)blocks_of(s) * rounds_of(p, s) * p.t.kv_heads; }
__device__ __forceinline__ long long begin_of(long long units, int groups, int j) { return units * j / groups; }

// The pieces of items that a group goes through, in order; each role walks for itself.
struct Walk {
    const AttentionParams& p;
    long long at, end, tree_first;
    int s, tile_of_group;
    TreeSpan span;
    int head, round, tile, kb0, kb1, blocks;
    long long first;             // unit of the item's first block
    __device__ __forceinline__ Walk(const AttentionParams& p_, long long at_, long long end_, long long tree_first_, int s_, int tile_)
        : p(p_), at(at_), end(end_), tree_first(tree_first_), s(s_), tile_of_group(tile_) { span = tree_span(p.t, s, p.status); }
    __device__ __forceinline__ bool next() {
        while (at < end) {
            long long mine = units_of(p, span);
            while (at >= tree_first + mine) {
                tree_first += mine;
                span = tree_span(p.t, ++s, p.status);
                mine = units_of(p, span);
            }
            blocks = blocks_of(span);
            const long long in_tree = at - tree_first, item = in_tree / blocks;
            const int rounds = rounds_of(p, span);
            kb0 = (int)(in_tree - item * blocks);
            kb1 = (int)min((long long)blocks, kb0 + (end - at));
            head = (int)(item / rounds);
            round = (int)(item - (long long)head * rounds);
            tile = round * p.tiles + tile_of_group;
            first = tree_first + item * blocks;
            at += kb1 - kb0;
            if (tile * kRows < span.nodes * p.t.group) return true;
        }
        return false;
    }
};

__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar_addr) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(smem_dst), "l"(map), "r"(x), "r"(y), "r"(z),
                 "r"(bar_addr)
                 : "memory");
}
// B operand with the contraction index as rows: atoms of 8 keys x 64 channels; the next 64 channels kHalf further on, the next 8 keys 1024 bytes.
__device__ __forceinline__ uint64_t make_smem_desc_mn(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(kHalf >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void tmem_ld_32_async(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, %0;\n" ::"n"(kRows) : "memory"); }
__device__ __forceinline__ bool not_finite(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }
// 32 bits from bit `at` (any) of a node's row of bits, ones in front of it
__device__ __forceinline__ uint32_t bits_from(const uint32_t* row, int at) {
    if (at <= -32) return 0xffffffffu;
    if (at >= kMostNodes) return 0;
    if (at < 0) return (row[0] << -at) | ((1u << -at) - 1u);
    const int w = at >> 5;
    return __funnelshift_r(row[w], w + 1 < kWords ? row[w + 1] : 0u, at & 31);
}

__global__ void __launch_bounds__(kThreads, 2) tree_attention_kernel(const __grid_constant__ AttentionParams p) {
    // f32 accumulator, bf16 operands, M = 128; N = 64, or 128 with B's contraction index as rows
    constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kRows >> 4) << 24);
    constexpr uint32_t kIdescS = kIdesc | ((uint32_t)(kKeys >> 3) << 17), kIdescO = kIdesc | ((uint32_t)(kTreeDim >> 3) << 17) | (1u << 16);
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2], q_full;
    __shared__ uint32_t tmem_holder;
    __shared__ long long s_sum[kThreads / 32], s_first;
    __shared__ int s_tree;
    __shared__ uint32_t s_bad[4];                       // of the blocks in flight: pages out of range
    __shared__ int s_up[kMostNodes];
    __shared__ uint32_t s_sees[kRows][kWords], s_odd[kWords];   // ancestors and itself of the tile's nodes; nodes with values that are not finite

    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sQ = smem, sK = smem + 2 * kQHalf, sV = sK + 2 * kStage;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = blockIdx.x / p.tiles, tile_of_group = blockIdx.x % p.tiles;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 1); mbar_init(&v_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_empty[i], 1); mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], kSoftmaxWarps);
        }
        mbar_init(&q_full, kSoftmaxWarps);
        mbar_fence_init();
    }
    pdl_wait();

    // ---- this group's units: every CTA adds up the trees' for itself -----------------------------------------------------------
    const int per = (p.t.n_trees + kThreads - 1) / kThreads;
    long long mine = 0;
    for (int s = tid * per; s < min((tid + 1) * per, p.t.n_trees); ++s) mine += units_of(p, tree_span(p.t, s, p.status));
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const long long other = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += other;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    long long units = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w == warp) upto += units;
        units += s_sum[w];
    }
    const int groups = (int)max(1ll, min((long long)p.groups, units / kMinUnits));
    if (blockIdx.x == 0 && tid == 0) { p.head->units = units; p.head->groups = units ? groups : 0; }
    if (units == 0 || group >= groups) return;          // the whole CTA
    const long long begin = begin_of(units, groups, group), end = begin_of(units, groups, group + 1);
    if (begin >= upto - mine && begin < upto) {
        long long first = upto - mine;
        for (int s = tid * per;; ++s) {
            const long long here = units_of(p, tree_span(p.t, s, p.status));
            if (begin < first + here) { s_tree = s; s_first = first; break; }
            first += here;
        }
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_holder)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_holder;
    pdl_launch_dependents();
    Walk walk(p, begin, end, s_first, s_tree, tile_of_group);
    bool failed = false;

    if (warp > kMmaWarp) {
        // ================= warps 5, 6: the pages of K and V ==========================================================================
        const int is_v = warp - kMmaWarp - 1;
        uint64_t* full = is_v ? v_full : k_full;
        uint64_t* empty = is_v ? v_empty : k_empty;
        const uint32_t base = is_v ? sV : sK;
        int g = 0;
        while (!failed && walk.next()) {
            const int last_page = (walk.span.length + walk.span.nodes - 1) / kTreePage;
            const int* table = p.t.table + (long long)walk.span.slot * p.t.max_pages;
            auto page_of = [&](int kb) { return lane < kPages && kb < walk.kb1 && kb * kPages + lane <= last_page ? table[kb * kPages + lane] : -2; };
            int coming = page_of(walk.kb0);
            for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++g) {
                const int page = coming;
                coming = page_of(kb + 1);
                if (g >= 2 && !mbar_wait_parked(smem_u32(&empty[g & 1]), (uint32_t)((g - 2) >> 1) & 1u, p.wait_limit)) failed = true;
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;
                const bool there = lane < kPages && kb * kPages + lane <= last_page, good = there && page >= 0 && page < p.t.n_pages;
                const uint32_t bar = smem_u32(&full[g & 1]), dst = base + (g & 1) * kStage;
                const uint32_t bad = __ballot_sync(0xffffffffu, there && !good), load = __ballot_sync(0xffffffffu, good);
                if (bad) {   // nothing is seen of them, but a value that is NaN would count in spite of its weight of 0
                    for (uint32_t b = bad; b; b &= b - 1)
                        for (int i = lane; i < 2 * kTreePage * 8; i += 32)
                            st_shared_v4(dst + (i >> 7) * kHalf + (__ffs(b) - 1) * (kTreePage * 128) + (i & 127) * 16, 0, 0, 0, 0);
                    fence_proxy_async();
                    if (lane == 0) atomicExch(p.status, 2);
                    __syncwarp();
                }
                if (lane == 0) {
                    if (!is_v) s_bad[g & 3] = bad;
                    mbar_expect_tx_addr(bar, (uint32_t)__popc(load) * 2 * kTreePage * 128);
                }
                __syncwarp();
                if (good && !(p.starve && g == 0 && !is_v)) {   // two copies a page: its halves of 64 channels
                    const int row0 = ((page * p.t.kv_heads + walk.head) * 2 + is_v) * kTreePage;
                    tma_load_3d(dst + lane * (kTreePage * 128), &p.map, 0, 0, row0, bar);
                    tma_load_3d(dst + kHalf + lane * (kTreePage * 128), &p.map, 0, 1, row0, bar);
                }
                __syncwarp();
            }
        }
        // copies still in flight write this CTA's shared memory
        for (int i = max(g - 2, 0); i < g; ++i) mbar_wait_parked(smem_u32(&full[i & 1]), (uint32_t)(i >> 1) & 1u, p.wait_limit);
        if (failed && lane == 0) atomicExch(p.status, 3);
    } else if (warp == kMmaWarp) {
        // ================= warp 4: one thread issues every product ===================================================================
        if (elect_one()) {
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                if (!failed && !mbar_wait_parked(smem_u32(bar), parity & 1u, p.wait_limit)) failed = true;
                return !failed;
            };
            auto scores = [&](int g) {
                if (!wait(&k_full[g & 1], (uint32_t)(g >> 1))) return;
                tc_fence_after();
                const uint64_t a = make_smem_desc(sQ), b = make_smem_desc(sK + (g & 1) * kStage);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    umma_bf16(tmem + (uint32_t)(g & 1) * kKeys, a + (uint64_t)((k >> 2) * (kQHalf >> 4) + 2 * (k & 3)), b + (uint64_t)((k >> 2) * (kHalf >> 4) + 2 * (k & 3)), kIdescS,
                              k > 0 ? 1u : 0u);
                umma_commit(&s_full[g & 1]);
                umma_commit(&k_empty[g & 1]);
            };
            int g = 0;
            for (int seg = 0; !failed && walk.next(); ++seg) {
                const int n = walk.kb1 - walk.kb0;
                if (!wait(&q_full, (uint32_t)seg)) break;
                tc_fence_after();
                scores(g);
                if (n > 1) scores(g + 1);
                for (int i = 0; i < n && !failed; ++i, ++g) {
                    if (!wait(&p_full[g & 1], (uint32_t)(g >> 1)) || !wait(&v_full[g & 1], (uint32_t)(g >> 1))) break;
                    tc_fence_after();
                    const uint64_t b = make_smem_desc_mn(sV + (g & 1) * kStage);
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        umma_bf16_ts(tmem + kOCol, tmem + (uint32_t)(g & 1) * kKeys + 8u * k, b + (uint64_t)(k * (16 * 128 >> 4)), kIdescO, (i > 0 || k > 0) ? 1u : 0u);
                    umma_commit(&v_empty[g & 1]);
                    if (i + 2 < n) scores(g + 2);
                }
            }
            if (failed) atomicExch(p.status, 3);
        }
        __syncwarp();
    } else {
        // ================= warps 0 - 3: softmax, a row per thread ====================================================================
        // After a timeout every warp still goes through all pieces, without waiting or working, so that the barriers of these warps are met.
        const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16), t_o = t_lane + kOCol;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (!failed && !mbar_wait_parked(smem_u32(bar), parity & 1u, p.wait_limit)) failed = true;
            failed = __any_sync(0xffffffffu, failed);
            return !failed;
        };
        int g = 0, tree = -1, tile = -1;
        if (tile_of_group == 0 && tid == 0) {   // the item that this group begins in, for the kernel that joins parts (whichever tiles it has)
            long long in_tree = begin - walk.tree_first, blocks = blocks_of(walk.span), item = in_tree / blocks, rounds = rounds_of(p, walk.span);
            p.begins[group] = {walk.tree_first + item * blocks, walk.tree_first + (item + 1) * blocks, walk.s, (int)(item / rounds), (int)(item % rounds), 0};
        }
        while (walk.next()) {
            const TreeSpan& span = walk.span;
            const int rows = span.nodes * p.t.group, rr = walk.tile * kRows + tid, node0 = walk.tile * kRows / p.t.group;
            const bool live = rr < rows;
            const int node = live ? rr / p.t.group : node0, head = walk.head * p.t.group + rr % p.t.group;
            // ---- the row's query, K-major with the 128-byte swizzle (the products that read the last one are complete: its output has been waited for)
            {
                const uint4* src = reinterpret_cast<const uint4*>(p.q + (long long)(span.row0 + node) * p.ldq + (long long)head * kTreeDim);
                const uint32_t dst = sQ + tid * 128;
                uint4 v[16];
#pragma unroll
                for (int c = 0; c < 16; ++c) v[c] = live ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int c = 0; c < 16; ++c) st_shared_v4(dst + (c >> 3) * kQHalf + (((c & 7) ^ (tid & 7)) << 4), v[c].x, v[c].y, v[c].z, v[c].w);
            }
            fence_proxy_async();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full);
            // ---- who sees whom
            softmax_sync();                                     // nobody reads the last piece's any more
            if (tid < kWords) s_odd[tid] = 0;
            if (walk.s != tree)
                for (int i = tid; i < span.nodes; i += kRows) s_up[i] = tree_parent(p.t, span, i, p.status);
            softmax_sync();
            if (walk.s != tree || walk.tile != tile) {
                const int i0 = node0 + tid;
#pragma unroll
                for (int w = 0; w < kWords; ++w) s_sees[tid][w] = 0;
                if (i0 < span.nodes && i0 * p.t.group < (walk.tile + 1) * kRows)
                    for (int i = i0; i >= 0; i = s_up[i]) s_sees[tid][i >> 5] |= 1u << (i & 31);
                tree = walk.s;
                tile = walk.tile;
                softmax_sync();
            }
            const uint32_t* sees = s_sees[node - node0];
            const bool idle = walk.tile * kRows + warp * 32 >= rows;   // no row of this warp is one
            float m = -INFINITY, l = 0.f;
            bool any = false;
            for (int kb = walk.kb0; kb < walk.kb1; ++kb, ++g) {
                const uint32_t t_s = t_lane + (uint32_t)(g & 1) * kKeys;
                wait(&s_full[g & 1], (uint32_t)(g >> 1));
                tc_fence_after();
                const bool tail = (kb + 1) * kKeys > span.length;
                if (!idle && !failed) {
                    uint32_t sr[kKeys];
                    tmem_ld_32_async(t_s, sr);
                    tmem_ld_32_async(t_s + 32, sr + 32);
                    tmem_wait_ld();
                    const uint32_t bad = s_bad[g & 3];
                    if (tail || bad) {
                        uint32_t vis[2];
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            vis[w] = bits_from(sees, kb * kKeys + 32 * w - span.length);
                            if (bad >> (2 * w) & 1) vis[w] &= 0xffff0000u;
                            if (bad >> (2 * w) & 2) vis[w] &= 0x0000ffffu;
                        }
                        any |= (vis[0] | vis[1]) != 0;
#pragma unroll
                        for (int j = 0; j < kKeys; ++j)
                            if (!(vis[j >> 5] >> (j & 31) & 1)) sr[j] = 0xff800000u;
                    } else {
                        any = true;
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < kKeys; ++j) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(sr[j]));
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
                    float keep = 1.f;
                    if (top > m + kLag || (kb == walk.kb0 && top > m)) {
                        keep = ex2(m - top);
                        m = top;
                    }
                    if (kb > walk.kb0 && __any_sync(0xffffffffu, keep != 1.f)) {   // O of the blocks in front, once their last product is complete
                        wait(&v_empty[(g - 1) & 1], (uint32_t)((g - 1) >> 1));
                        tc_fence_after();
                        if (!failed) {
#pragma unroll 1
                            for (int c = 0; c < 4; ++c) {
                                uint32_t r[32];
                                tmem_ld_32_async(t_o + 32u * c, r);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * keep);
                                tmem_st_32(t_o + 32u * c, r);
                            }
                        }
                    }
                    l *= keep;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
                    const float ref = m == -INFINITY ? 0.f : m;
                    if (__any_sync(0xffffffffu, fabsf(ref) > kLargeScore)) {
#pragma unroll
                        for (int j = 0; j < kKeys; ++j) sr[j] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(sr[j]), p.scale_log2), ref));
                    } else {
#pragma unroll
                        for (int j = 0; j < kKeys; ++j) sr[j] = __float_as_uint(fmaf(__uint_as_float(sr[j]), p.scale_log2, -ref));
                    }
#pragma unroll
                    for (int i = 0; i < kKeys / 2; ++i) {
                        const float w0 = ex2(__uint_as_float(sr[2 * i])), w1 = ex2(__uint_as_float(sr[2 * i + 1]));
                        sum[i & 3] += w0 + w1;
                        sr[i] = pack_bf16x2(w0, w1);
                    }
                    tmem_st_32(t_s, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                }
                if (tail && wait(&v_full[g & 1], (uint32_t)(g >> 1))) {
                    // values behind the last node, and those of nodes that are not finite: the product sees zeros
                    const int from = max(0, span.length - kb * kKeys), total = span.length + span.nodes;
                    for (int i = tid; i < (kKeys - from) * 16; i += kRows) {
                        const int r = from + (i >> 4), token = kb * kKeys + r;
                        const uint32_t at = sV + (g & 1) * kStage + (i >> 3 & 1) * kHalf + r * 128 + ((i & 7) << 4);
                        uint4 v = ld_shared_v4(at);
                        if (token >= total) {
                            st_shared_v4(at, 0, 0, 0, 0);
                        } else {
                            uint32_t *w = &v.x, odd = 0;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t none = __vcmpgeu2(w[k] & 0x7fff7fffu, 0x7f807f80u);
                                w[k] &= ~none;
                                odd |= none;
                            }
                            if (odd) {
                                st_shared_v4(at, v.x, v.y, v.z, v.w);
                                atomicOr(&s_odd[(token - span.length) >> 5], 1u << ((token - span.length) & 31));
                            }
                        }
                    }
                    fence_proxy_async();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[g & 1]);
            }
            // ---- O / l, or the row's part of it
            wait(&v_empty[(g - 1) & 1], (uint32_t)((g - 1) >> 1));
            tc_fence_after();
            if (!failed && !idle) {
                const bool whole = walk.kb0 == 0 && walk.kb1 == walk.blocks;
                const size_t slot = 2 * (size_t)blockIdx.x + (walk.kb0 == 0 ? 1 : 0);
                if (any && m == -INFINITY) l = NAN;             // scores of -inf alone
                const float inv = whole ? (any ? 1.f / l : 0.f) : 1.f;
                uint32_t odd = 0;
#pragma unroll
                for (int w = 0; w < kWords; ++w) odd |= s_odd[w] & sees[w];
                if (!whole && live) p.ml[slot * p.row_cap + tid] = make_float2(m, l);
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float o[32];
                    tmem_ld_32(t_o + 32u * c, o);
                    if (!live) continue;
                    if (odd) {
                        for (int i = 0; i < span.nodes; ++i) {
                            if (!(s_odd[i >> 5] & sees[i >> 5] & 1u << (i & 31))) continue;
                            const int at = span.length + i;
                            const long long place = tree_place(p.t, span.slot, at, p.status);
                            if (place < 0) continue;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const int chunk = 4 * c + (j >> 3);
                                const uint16_t v = *reinterpret_cast<const uint16_t*>(p.pool + place + (2 * walk.head + 1) * kTreeBlock + ((chunk ^ (at & 7)) << 4) + 2 * (j & 7));
                                if (not_finite(v)) o[j] += __uint_as_float((uint32_t)v << 16);
                            }
                        }
                    }
                    if (whole) {
                        uint4* dst = reinterpret_cast<uint4*>(p.out + ((long long)(span.row0 + node) * p.t.q_heads + head) * kTreeDim);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            dst[4 * c + i] = make_uint4(pack_bf16x2(o[8 * i] * inv, o[8 * i + 1] * inv), pack_bf16x2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                                        pack_bf16x2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack_bf16x2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            p.sums[(slot * 32 + 8 * c + i) * p.row_cap + tid] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                }
            }
        }
        if (failed && lane == 0) atomicExch(p.status, 3);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// Joins the parts of the items in which a group begins: one CTA per (group, tile, 32 rows, 64 channels); the first group that begins inside an item does it.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ AttentionParams p) {
    __shared__ __align__(16) __nv_bfloat16 s_out[32][64 + 8];
    pdl_launch_dependents();
    pdl_wait();
    const int groups = p.head->groups, j = blockIdx.x + 1, half = blockIdx.y & 1, quarter = (blockIdx.y >> 1) & 3, tile_of_group = blockIdx.y >> 3;
    if (j >= groups) return;
    const long long units = p.head->units;
    const Part item = p.begins[j];
    if (begin_of(units, groups, j) == item.first || begin_of(units, groups, j - 1) > item.first) return;
    const TreeSpan span = tree_span(p.t, item.tree, p.status);
    const int tile = item.round * p.tiles + tile_of_group, rows = span.nodes * p.t.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = quarter * 32 + lane, first_row = tile * kRows + quarter * 32;
    if (first_row >= rows) return;
    const bool live = tile * kRows + row < rows;
    const int last = (int)min((long long)groups, (item.end * groups + units - 1) / units) - 1;   // the last group that begins in front of the item's end
    auto slot = [&](int k) { return 2 * ((size_t)k * p.tiles + tile_of_group) + (k == j - 1 ? 1 : 0); };
    float top = -INFINITY, l = 0.f;
    float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    if (live) {
#pragma unroll 8
        for (int k = j - 1; k <= last; ++k) top = fmaxf(top, p.ml[slot(k) * p.row_cap + row].x);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll 4
        for (int k = j - 1; k <= last; ++k) {
            const float2 ml = p.ml[slot(k) * p.row_cap + row];
            const float f = ex2(ml.x - ref);
            l += ml.x == -INFINITY ? ml.y : ml.y * f;           // (without a score 0, or NaN)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float4 v = p.sums[(slot(k) * 32 + 16 * half + 8 * i + warp) * p.row_cap + row];
                o[i].x += v.x * f; o[i].y += v.y * f; o[i].z += v.z * f; o[i].w += v.w * f;
            }
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint2*>(&s_out[lane][4 * (8 * i + warp)]) = make_uint2(pack_bf16x2(o[i].x * inv, o[i].y * inv), pack_bf16x2(o[i].z * inv, o[i].w * inv));
    __syncthreads();
    const int r = threadIdx.x >> 3, rr = first_row + r;
    if (rr < rows)
        *reinterpret_cast<uint4*>(p.out + ((long long)(span.row0 + rr / p.t.group) * p.t.q_heads + item.head * p.t.group + rr % p.t.group) * kTreeDim + 64 * half + 8 * (threadIdx.x & 7)) =
            *reinterpret_cast<const uint4*>(&s_out[r][8 * (threadIdx.x & 7)]);
}

// The pool as rows of a token and head of 256 bytes (z), two halves (y) of 64 channels (x); a block (page, kv head, keys or values) begins at row
// ((page x kv heads + head) x 2 + is value) x 16. The kernel asks for pages below n_pages alone.
int encode_pool(const void* pool, const DraftTrees& t, CUtensorMap* map) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(GPTRS_EXECUTION, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[3] = {64, 2, (cuuint64_t)t.n_pages * t.kv_heads * 2 * kTreePage};
    cuuint64_t strides[2] = {128, 256};
    cuuint32_t box[3] = {64, 1, (cuuint32_t)kTreePage};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(pool), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GPTRS_EXECUTION, "cuTensorMapEncodeTiled failed for the pool (" + std::to_string((int)r) + ")");
    return GPTRS_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How a call is cut: groups of one CTA, or of two where trees may have more than 128 rows.
void cut(const gptrs_draft_trees* t, int* groups, int* tiles, int* row_cap) {
    const int rows = t->max_nodes * (t->q_heads / t->kv_heads);
    *tiles = rows > kRows ? 2 : 1;
    *groups = 2 * sm_count() / *tiles;
    *row_cap = rows < kRows ? (rows + 31) / 32 * 32 : kRows;
}
size_t head_bytes(int groups) { return sizeof(Head) + (size_t)groups * sizeof(Part); }

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" {

size_t gptrs_cuda_tree_scratch_bytes(const gptrs_draft_trees* t) {
    DraftTrees checked;
    if (draft_trees(t, &checked) != GPTRS_OK) return 0;
    int groups, tiles, row_cap;
    cut(t, &groups, &tiles, &row_cap);
    const size_t slots = 2 * (size_t)groups * tiles;
    return head_bytes(groups) + slots * row_cap * (sizeof(float2) + 32 * sizeof(float4));
}

int gptrs_cuda_tree_attention(const gptrs_draft_trees* t, const gptrs_tree_attention_step* s, void* stream) {
    AttentionParams p = {};
    const int rc = draft_trees(t, &p.t);
    if (rc) return rc;
    GPTRS_REQUIRE(s && s->d_pool && s->d_status && (t->rows == 0 || (s->d_q && s->d_out)), "null pointer");
    GPTRS_REQUIRE(aligned16(s->d_q) && aligned16(s->d_pool) && aligned16(s->d_out) && aligned16(s->d_scratch), "pointers must be 16-byte aligned");
    const int64_t width = (int64_t)t->q_heads * kTreeDim;
    p.ldq = s->ldq ? s->ldq : width;
    GPTRS_REQUIRE(p.ldq >= width && p.ldq % 8 == 0 && p.ldq < ((int64_t)1 << 31), "rows of queries overlap, or do not start at multiples of 16 bytes");
    GPTRS_REQUIRE(t->n_pages * t->kv_heads * 2 * kTreePage < ((int64_t)1 << 31), "the pool has too many pages");
    GPTRS_REQUIRE(s->d_scratch && s->scratch_bytes >= gptrs_cuda_tree_scratch_bytes(t), "scratch is too small");
    if (t->rows == 0) return GPTRS_OK;
    const char *q = static_cast<const char*>(s->d_q), *out = static_cast<const char*>(s->d_out);
    GPTRS_REQUIRE(out >= q + 2 * ((t->rows - 1) * p.ldq + width) || q >= out + 2 * t->rows * width, "the output lies in rows of queries");
    const int bad = encode_pool(s->d_pool, p.t, &p.map);
    if (bad) return bad;
    p.q = static_cast<const __nv_bfloat16*>(s->d_q);
    p.pool = static_cast<const unsigned char*>(s->d_pool);
    p.out = static_cast<__nv_bfloat16*>(s->d_out);
    p.status = s->d_status;
    p.scale_log2 = (t->scale != 0.f ? t->scale : 1.f / sqrtf((float)kTreeDim)) * kLog2e;
    cut(t, &p.groups, &p.tiles, &p.row_cap);
    const size_t slots = 2 * (size_t)p.groups * p.tiles;
    p.head = static_cast<Head*>(s->d_scratch);
    p.begins = reinterpret_cast<Part*>(p.head + 1);
    p.sums = reinterpret_cast<float4*>(static_cast<char*>(s->d_scratch) + head_bytes(p.groups));
    p.ml = reinterpret_cast<float2*>(p.sums + slots * 32 * p.row_cap);
    prefill_tc_fault(&p.starve, &p.wait_limit);
    static PerDeviceOnce attr_once;
    if (attr_once.first_time()) GPTRS_CUDA_OK(cudaFuncSetAttribute(tree_attention_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    const int failed = launch_kernel(tree_attention_kernel, dim3((unsigned)(p.groups * p.tiles)), dim3(kThreads), kSmem, as_stream(stream), 1, p);
    if (failed) return failed;
    // the second kernel waits for the first one itself (griddepcontrol.wait), so it may be launched ahead of its end
    const int pdl = g_use_pdl;
    g_use_pdl = 1;
    const int joined = launch_kernel(tree_join_kernel, dim3((unsigned)max(1, p.groups - 1), (unsigned)(8 * p.tiles)), dim3(kJoinThreads), 0, as_stream(stream), 1, p);
    g_use_pdl = pdl;
    return joined;
}

}  // extern "C"
