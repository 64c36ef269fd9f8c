// Attention of trees of drafted tokens over the paged bf16 cache: node i of a tree sees the sequence's tokens, its ancestors and itself.
//
// The rows of a tree and kv head (row = node x group + query head) share the keys that they see, all but the last few dozen, so they are the M side of
// tcgen05 products: a CTA holds a tile of 128 rows and walks over keys in blocks of 64 (four pages), two CTAs to an SM:
//   S[128 x 64] = Q . K^T      both from shared memory (K-major, 128-byte swizzle, which is how the pool holds a page), two accumulators in tensor memory
//   softmax                    warps 0 - 3, a thread per row, one pass over its scores: the reference stays until a block's weights add up to more than 2^14, so there is
//                              no pass for the maximum but in a row's first block; weights go over S as two bf16 terms each, since values are bf16 and a product has one
//                              type. With one term results were off by 0.0023 of their size, with two by 0.0017, which is their own rounding; it costs twice the
//                              products of P . V and two conversions a weight (64 trees 211 -> 236 us, two long ones 162 -> 175, six wide ones 70 -> 75)
//   O[128 x 128] += P . V      P's two terms from tensor memory, V as an MN-major operand
// Warp 4 issues the products, S two blocks ahead of P . V; warps 5 and 6 request the pages of K and V; warp 7 looks ahead: it finds the next piece of work, collects
// the ancestors of its nodes and requests its queries as soon as the products that read the last ones are complete.
// Blocks that reach behind the sequence's tokens are masked by a bit per node. In them values of nodes that are not finite are taken out of the stage by warp 6
// (a weight of 0 does not help there) and added to the rows that see them at the end.
//
// Work, where contexts may be long: an item is a (tree, kv head, row tile or pair of them), a unit a block of an item, and an item has some more that stand for what it costs
// beside its keys; every group of CTAs (one, or two for trees of more rows than a tile has, which then share the keys through L2) takes the same number of consecutive
// units, whatever the trees' lengths. Where an item is cut, its parts are counted in warp by warp (a warp has the same rows in all of them): the last warp to finish waits until
// the others' sums are in scratch and joins them with its own, four at a time, in the order of the keys, and such joins are joined again. Few items have many parts each: those a
// second kernel joins. So the result depends on the call alone, not on who was last. Where contexts are short (kSmall) a cluster of up to eight CTAs takes a (tree, kv head, row
// tile), a share of its keys each, and joins through distributed shared memory: nothing has to be added up or looked for in front.
//
// What bounds it (times of the kernels in a graph; calls from Python take 2 to 50 us more), 32 / 8 heads: 64 trees of 32 nodes at 512 to 8192 tokens 236 us for the 1.18 GB of the
// cache (181 at the rate of a copy), two trees at 100003 and 131072 175 us (145): HBM, the wait for the products in front of a stage's reuse, and the joins at the end. A block takes
// the softmax warps 1800 to 2100 cycles, of which 64 exponentials a thread, four lanes a cycle and scheduler, are 1024 for the two warps that a scheduler has. Where rows share keys (six trees
// of 250 nodes at 700 to 4000, 16 / 2 heads, 67 to 80 us) that is half of it: of the 82 to 114 thousand cycles of a CTA 43 to 57 are the softmax of 22 to 28 blocks, 9 to 13 waits for
// scores, 8 to 49 the ends of its pieces, where parts are joined; some CTAs have nothing, where the second tile of a pair is one too many. One tree of 26 nodes at 1500 tokens 13.0 us, a chain of latencies: tree, table, pages, three blocks of the CTA's share, and
// the cluster's join. Two threads to a row took 284 us where one took 207 (a barrier every block).
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
constexpr int kThreads = (kSoftmaxWarps + 4) * 32;
constexpr int kQHalf = kRows * 128;             // bytes of 64 channels of the queries
constexpr int kHalf = kKeys * 128;              // of a block's keys or values
constexpr int kStage = 2 * kHalf;
constexpr uint32_t kTmemCols = 256;             // two S, O
constexpr uint32_t kOCol = 128;
constexpr size_t kSmem = 2 * kQHalf + 4 * kStage + 1024;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMostSum = 16384.f;             // of a row's weights in a block: above it the reference is raised
constexpr float kLargeScore = 1048576.f;        // above it a product and a sum rounded once (fma) are further apart than an exponent may be off
constexpr int kMinUnits = 8;                    // of a group
constexpr int kORow = kTreeDim + 4;             // floats of a row of sums in shared memory
constexpr int kWords = kMostNodes / 32;
constexpr int kJoin = 4;                        // parts that are joined at a time
constexpr int kLevels = 5;                      // 4^5 groups
constexpr int kReaders = kSoftmaxWarps + 3;     // of a piece of work: the softmax's warps, the products' thread, the two that load

// An item that a CTA has the first part of, for the kernel that joins parts (0 or 1 of them: none).
struct Item { int parts, row0, nodes, head, tile, pad[3]; };

struct AttentionParams {
    CUtensorMap map, q_map;
    DraftTrees t;
    const unsigned char* pool;
    __nv_bfloat16* out;
    Item* items;                 // [groups tiles], where a second kernel joins the parts; NULL: the warps do
    uint32_t *done, *stored;     // [levels][2 groups tiles][4]: parts of a join that are worked out, and in scratch, by warp; 0 again when it is made
    float2* ml;                  // [2 groups tiles][row_cap]: reference and sum of a row; the first of a CTA's two slots is for items that others began
    float4* sums;                // [2 groups tiles][32][row_cap]
    int* status;
    float scale_log2;
    int groups, tiles, row_cap;  // tiles: of a group, 1 or 2
    int tile_nodes;              // of a tile: as many as 128 rows hold
    int cluster;                 // small calls: CTAs of a tile
    uint32_t wait_limit;
    int starve;
};

__device__ __forceinline__ int blocks_of(const TreeSpan& s) { return (s.length + s.nodes + kKeys - 1) / kKeys; }
__device__ __forceinline__ int rounds_of(const AttentionParams& p, const TreeSpan& s) {
    const int tiles = (s.nodes + p.tile_nodes - 1) / p.tile_nodes;
    return p.tiles == 2 ? (tiles + 1) >> 1 : tiles;
}
// What an item costs beside its blocks, in units: its queries, its output, and the masks of the blocks with nodes in them.
__device__ __forceinline__ int extra_of(const TreeSpan& s) { return 2 + (s.nodes + kKeys - 1) / kKeys; }
__device__ __forceinline__ uint32_t units_of(const AttentionParams& p, const TreeSpan& s) {   // (the host has made sure that they fit)
    return s.nodes == 0 ? 0u : (uint32_t)(blocks_of(s) + extra_of(s)) * (uint32_t)rounds_of(p, s) * (uint32_t)p.t.kv_heads;
}
// The first unit of group j, and the group that has a unit (at most 2^9 groups: 32 bits are enough for most calls).
__device__ __forceinline__ long long begin_of(long long units, int groups, int j) {
    return units < (1 << 22) ? (long long)((uint32_t)units * (uint32_t)j / (uint32_t)groups) : units * j / groups;
}
__device__ __forceinline__ int group_of(long long units, int groups, long long unit) {   // the last j with units j / groups < unit + 1
    const long long x = (unit + 1) * groups - 1;
    return units < (1 << 22) ? (int)((uint32_t)x / (uint32_t)units) : (int)(x / units);
}

// A piece of work: blocks kb0 .. kb1 - 1 of an item; kb1 0: there is none any more.
struct Piece { TreeSpan span; int head, tile, kb0, kb1, part, parts; };   // part: which of the item's

// The pieces that a group goes through, in order.
struct Walk {
    const AttentionParams& p;
    long long units, pos;        // of all; the one that comes next
    int groups, s, tile_of_group;
    TreeSpan span;
    uint32_t at, left;           // pos within the tree, units left
    uint32_t tree_units;
    int size, extra, rounds;     // an item's units, those in front of its blocks
    Piece piece;
    __device__ __forceinline__ Walk(const AttentionParams& p_, long long units_, int groups_, long long pos_, long long end, int s_, const TreeSpan& span_, uint32_t at_, int tile_)
        : p(p_), units(units_), pos(pos_), groups(groups_), s(s_), tile_of_group(tile_), span(span_), at(at_), left((uint32_t)(end - pos_)) { measure(); }
    __device__ __forceinline__ void measure() {
        extra = extra_of(span);
        size = blocks_of(span) + extra;
        rounds = rounds_of(p, span);
        tree_units = units_of(p, span);
    }
    __device__ __forceinline__ bool next() {
        while (left > 0) {
            if (at >= tree_units) {
                at -= tree_units;
                span = tree_span(p.t, ++s, p.status);
                measure();
                continue;
            }
            const uint32_t item = at / (uint32_t)size;
            const int in_item = (int)(at - item * (uint32_t)size), n = (int)min((uint32_t)(size - in_item), left);
            const long long first = pos - in_item;
            at += n; left -= n; pos += n;
            const int head = rounds == 1 ? (int)item : (int)(item / (uint32_t)rounds), tile = ((int)item - head * rounds) * p.tiles + tile_of_group;
            piece = {span, head, tile, max(0, in_item - extra), in_item + n - extra, 0, 1};
            if (piece.kb1 <= piece.kb0 || tile * p.tile_nodes >= span.nodes) continue;
            if (piece.kb1 - piece.kb0 < size - extra) {
                const int from = group_of(units, groups, first + extra);
                piece.part = group_of(units, groups, pos - 1) - from;
                piece.parts = group_of(units, groups, first + size - 1) - from + 1;
            }
            return true;
        }
        piece.kb1 = 0;
        return false;
    }
};

__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar_addr) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(smem_dst), "l"(map), "r"(x), "r"(y), "r"(z),
                 "r"(bar_addr)
                 : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar_addr) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(smem_dst), "l"(map), "r"(x), "r"(y),
                 "r"(z), "r"(w), "r"(bar_addr)
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
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        "tcgen05.wait::ld.sync.aligned;\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool not_finite(uint32_t half) { return (half & 0x7f80u) == 0x7f80u; }
// 32 bits from bit `at` (any) of a node's row of bits, ones in front of it
__device__ __forceinline__ uint32_t bits_from(const uint32_t* row, int at) {
    if (at <= -32) return 0xffffffffu;
    if (at >= kMostNodes) return 0;
    if (at < 0) return (row[0] << -at) | ((1u << -at) - 1u);
    const int w = at >> 5;
    return __funnelshift_r(row[w], w + 1 < kWords ? row[w + 1] : 0u, at & 31);
}

__device__ __forceinline__ bool mbar_ready(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok;
}
// Waits (bounded) until `n` parts of a join are in scratch, and sets the count back.
__device__ __forceinline__ bool parts_stored(uint32_t* at, uint32_t n, uint32_t limit) {
    for (uint32_t i = 0; i < 8 * limit; ++i) {
        uint32_t v;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];\n" : "=r"(v) : "l"(at) : "memory");
        if (v >= n) { *at = 0; return true; }
    }
    return false;
}
// A load that stays where it is written: the ones of several parts are all under way before the first is used (left to the compiler a join of four took 15000 cycles).
__device__ __forceinline__ float4 load_now(const float4* at) {
    float4 v;
    asm volatile("ld.global.cg.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(at) : "memory");
    return v;
}
// A part of a row has (m, l): its reference and its sum, or, where no score is above -inf, m = -inf and l = 0 (nothing is seen), 1 (scores of -inf) or NaN (some are NaN). Keys whose
// scores are -inf weigh nothing beside finite ones of other parts; whether a row has none is known where all of its parts meet.
// What a part adds to the sum of parts whose largest reference is top; f = 2^(m - that).
__device__ __forceinline__ float share_of(float2 ml, float f, float top) { return ml.x == -INFINITY ? (top == -INFINITY ? ml.y : ml.y * 0.f) : ml.y * f; }
__device__ __forceinline__ float inverse_of(float top, float sum) { return top == -INFINITY ? (sum == 0.f ? 0.f : NAN) : 1.f / sum; }
__device__ __forceinline__ void store_part(const AttentionParams& p, size_t slot, bool live, uint32_t t_o, float m, float l) {
    float4* to = p.sums + slot * 32 * p.row_cap + threadIdx.x;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        float o[32];
        __syncwarp();
        tmem_ld_32(t_o + 32u * c, o);
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i) to[(8 * c + i) * p.row_cap] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
    }
    if (live) p.ml[slot * p.row_cap + threadIdx.x] = make_float2(m, l);
}
// A warp's part of an item: to scratch, unless this warp is the last of its join's four; then it joins them, to the first one's place or, all of the item, to the output. Returns
// false if a wait ran out.
__device__ __forceinline__ bool join_parts(const AttentionParams& p, const Piece& piece, bool live, uint32_t t_o, float m, float l, uint4* dst) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, from = blockIdx.x / p.tiles - piece.part;
    const size_t slots = 2 * (size_t)p.groups * p.tiles;
    auto slot = [&](int part) { return 2 * ((size_t)(from + part) * p.tiles + blockIdx.x % p.tiles) + (part == 0 ? 1 : 0); };
    int n = p.items ? 1 : piece.parts, at = piece.part, apart = 1;   // parts of this level, this one's number, how far they lie apart
    bool mine = true;                                  // the sums are in tensor memory; else in scratch
    if (p.items) store_part(p, slot(at), live, t_o, m, l);
    for (int level = 0; n > 1; ++level) {
        const int first = at / kJoin * kJoin, members = min(kJoin, n - first), me = mine ? at - first : kJoin;
        const size_t count = ((size_t)level * slots + slot(first * apart)) * kSoftmaxWarps + warp;
        uint32_t before = members - 1;
        if (members > 1) {
            if (lane == 0) before = atomicInc(p.done + count, members - 1);   // (back to 0 by the last one)
            before = __shfl_sync(0xffffffffu, before, 0);
        }
        const bool last = before == members - 1;
        if (mine && (!last || members == 1)) {
            store_part(p, slot(at), live, t_o, m, l);
            mine = false;
        }
        if (members > 1) {
            if (!last) {
                __threadfence();
                __syncwarp();
                if (lane == 0) atomicAdd(p.stored + count, 1u);
                return true;
            }
            bool there = true;
            if (lane == 0) there = parts_stored(p.stored + count, members - 1, p.wait_limit);
            if (!__shfl_sync(0xffffffffu, (int)there, 0)) return false;
            __threadfence();
            const bool all = n <= kJoin;
            // (loads without conditions, so that they are under way together: the first part's where there is none, or the own one is taken)
            const float4* part[kJoin];
            float2 ml[kJoin];
            float f[kJoin], top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < kJoin; ++k) {
                const size_t at_k = slot((first + (k < members ? k : 0)) * apart);
                part[k] = p.sums + at_k * 32 * p.row_cap + tid;
                ml[k] = __ldcg(p.ml + at_k * p.row_cap + tid);
            }
#pragma unroll
            for (int k = 0; k < kJoin; ++k) {
                if (k == me) ml[k] = make_float2(m, l);
                if (k >= members) ml[k] = make_float2(-INFINITY, 0.f);
                top = fmaxf(top, ml[k].x);
            }
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int k = 0; k < kJoin; ++k) {
                f[k] = ex2(ml[k].x - ref);
                sum += share_of(ml[k], f[k], top);
            }
            const float inv = inverse_of(top, sum);
            float4* to = p.sums + slot(first * apart) * 32 * p.row_cap + tid;
            const int cap = p.row_cap;
#pragma unroll 1
            for (int c = 0; c < 32; c += 4) {
                float4 v[kJoin][4], o[4];
                uint32_t own[16];
#pragma unroll
                for (int k = 0; k < kJoin; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[k][i] = load_now(part[k] + (c + i) * cap);
                __syncwarp();
                if (mine) tmem_ld_16(t_o + 4u * c, own);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int k = 0; k < kJoin; ++k) {
                        if (k >= members) break;
                        if (k == me) v[k][i] = make_float4(__uint_as_float(own[4 * i]), __uint_as_float(own[4 * i + 1]), __uint_as_float(own[4 * i + 2]), __uint_as_float(own[4 * i + 3]));
                        o[i].x += v[k][i].x * f[k]; o[i].y += v[k][i].y * f[k]; o[i].z += v[k][i].z * f[k]; o[i].w += v[k][i].w * f[k];
                    }
                }
                if (!live) continue;
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    if (all) dst[(c + i) / 2] = make_uint4(pack_bf16x2(o[i].x * inv, o[i].y * inv), pack_bf16x2(o[i].z * inv, o[i].w * inv), pack_bf16x2(o[i + 1].x * inv, o[i + 1].y * inv),
                                                           pack_bf16x2(o[i + 1].z * inv, o[i + 1].w * inv));
                    else { to[(c + i) * cap] = o[i]; to[(c + i + 1) * cap] = o[i + 1]; }
                }
            }
            if (!all && live) p.ml[slot(first * apart) * p.row_cap + tid] = make_float2(top, sum);
            mine = false;
            m = top;
            l = sum;
        }
        at /= kJoin;
        n = (n + kJoin - 1) / kJoin;
        apart *= kJoin;
    }
    return true;
}

// Values behind the last node, and those of nodes that are not finite: the product sees zeros, and `odd` says which nodes they are. By the warp that has asked for them, while the
// softmax is at the block in front (by the softmax's own warps a block took 4900 cycles instead of 2900).
__device__ __forceinline__ void clean_values(uint32_t stage, const TreeSpan& span, int kb, uint32_t* odd) {
    const int lane = threadIdx.x & 31, from = max(0, span.length - kb * kKeys), total = span.length + span.nodes - kb * kKeys;   // rows of nodes
#pragma unroll 1
    for (int k0 = from / 4 & ~3; k0 < kKeys / 4; k0 += 4) {   // 16 rows, of both halves: a row is eight lanes'
        uint4 v[8];
        bool any = false;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t at = stage + (k >> 2) * kHalf + (k0 + (k & 3)) * 512 + lane * 16;
            v[k] = ld_shared_v4(at);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {   // an exponent of ones and one more reach the sign's place
            constexpr uint32_t kExponents = 0x7f807f80u, kOnes = 0x00800080u;
            const uint32_t found = ((v[k].x & kExponents) + kOnes) | ((v[k].y & kExponents) + kOnes) | ((v[k].z & kExponents) + kOnes) | ((v[k].w & kExponents) + kOnes);
            any |= (found & 0x80008000u) != 0;
        }
        if (!__any_sync(0xffffffffu, any) && total >= 4 * k0 + 16) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int row = 4 * (k0 + (k & 3)) + (lane >> 3);
            const uint32_t at = stage + (k >> 2) * kHalf + (k0 + (k & 3)) * 512 + lane * 16;
            uint32_t* w = &v[k].x;
            uint32_t found = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t m = (((w[j] & 0x7f807f80u) + 0x00800080u) & 0x80008000u) >> 15;
                found |= m;
                w[j] &= ~(m * 0xffffu);
            }
            if (row >= total) st_shared_v4(at, 0, 0, 0, 0);
            else if (found && row >= from) {
                st_shared_v4(at, w[0], w[1], w[2], w[3]);
                const int node = kb * kKeys + row - span.length;
                atomicOr(&odd[node >> 5], 1u << (node & 31));
            }
        }
    }
    fence_proxy_async();
    __syncwarp();
}

template <bool kSmall>
__global__ void __launch_bounds__(kThreads, 2) tree_attention_kernel(const __grid_constant__ AttentionParams p) {
    // f32 accumulator, bf16 operands, M = 128; N = 64, or 128 with B's contraction index as rows
    constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(kRows >> 4) << 24);
    constexpr uint32_t kIdescS = kIdesc | ((uint32_t)(kKeys >> 3) << 17), kIdescO = kIdesc | ((uint32_t)(kTreeDim >> 3) << 17) | (1u << 16);
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_full[2], q_full, q_empty, piece_full[2], piece_empty[2], sees_full[2];
    __shared__ uint32_t tmem_holder;
    __shared__ long long s_sum[kSoftmaxWarps], s_first;
    __shared__ float2 s_ml[kSmall ? kRows : 1];         // of the rows of a share
    __shared__ int s_tree;
    __shared__ TreeSpan s_span;
    __shared__ Piece s_piece[2];                        // this one and the next
    __shared__ uint32_t s_bad[4];                       // of the blocks in flight: pages out of range
    __shared__ int s_up[kMostNodes];
    __shared__ __align__(16) uint32_t s_sees[2][kRows][kWords];   // ancestors and itself of a piece's nodes
    __shared__ uint32_t s_odd[2][kWords];               // nodes with values that are not finite

    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sQ = smem, sK = smem + 2 * kQHalf, sV = sK + 2 * kStage;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 1); mbar_init(&v_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_empty[i], 1); mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], kSoftmaxWarps + 1); mbar_init(&piece_full[i], 1); mbar_init(&piece_empty[i], kReaders); mbar_init(&sees_full[i], 1);
        }
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 1);
        mbar_fence_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_holder)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    pdl_wait();

    // ---- this CTA's work
    const int per = (p.t.n_trees + kRows - 1) / kRows;
    const int rank = kSmall && p.cluster > 1 ? (int)cluster_ctarank() : 0, group = blockIdx.x / p.tiles, tile_of_group = blockIdx.x % p.tiles;
    TreeSpan last = {-1, 0, 0, 0};
    Piece only = {};                                    // a small call's
    int first_page = -2;
    int groups = 1;
    long long units = 0, begin = 0, end = 0, mine = 0, upto = 0;
    bool idles = false;
    if constexpr (kSmall) {
        only.span = tree_span(p.t, blockIdx.z, p.status);
        only.head = blockIdx.y;
        only.tile = blockIdx.x >> (31 - __clz(p.cluster));
        only.parts = 1;
        idles = only.tile * p.tile_nodes >= only.span.nodes;
        if (!idles) {
            const int blocks = blocks_of(only.span);
            only.kb0 = (int)((uint32_t)blocks * (uint32_t)rank >> (31 - __clz(p.cluster)));
            only.kb1 = (int)((uint32_t)blocks * (uint32_t)(rank + 1) >> (31 - __clz(p.cluster)));
            // the first block's pages, which the loads of keys and values wait for
            const int page = only.kb0 * kPages + lane;
            if (warp > kMmaWarp && lane < kPages && only.kb0 < only.kb1 && page <= (only.span.length + only.span.nodes - 1) / kTreePage)
                first_page = p.t.table[(long long)only.span.slot * p.t.max_pages + page];
        }
    } else if (warp < kSoftmaxWarps) {   // warps 0 - 3 add up the trees' units
        for (int s = tid * per; s < min((tid + 1) * per, p.t.n_trees); ++s) {
            last = tree_span(p.t, s, p.status);
            mine += units_of(p, last);
        }
        upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        if (lane == 31) s_sum[warp] = upto;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_holder;
    if constexpr (!kSmall) {
#pragma unroll
        for (int w = 0; w < kSoftmaxWarps; ++w) {
            if (w == warp) upto += units;
            units += s_sum[w];
        }
        groups = (int)max(1ll, min((long long)p.groups, units / kMinUnits));
        idles = units == 0 || group >= groups;
        if (!idles) {
            begin = begin_of(units, groups, group);
            end = begin_of(units, groups, group + 1);
        }
        if (warp < kSoftmaxWarps && !idles && begin >= upto - mine && begin < upto) {
            long long first = upto - mine;
            int s = tid * per;
            if (per > 1) {
                for (;; ++s) {
                    last = tree_span(p.t, s, p.status);
                    const long long here = units_of(p, last);
                    if (begin < first + here) break;
                    first += here;
                }
            }
            s_tree = s;
            s_first = first;
            s_span = last;
        }
        __syncthreads();
    }
    pdl_launch_dependents();
    bool failed = false;
    // A piece's place in the ring, for those that read it: the i-th of this CTA.
    auto take = [&](int i, Piece* piece) {
        if constexpr (kSmall) {
            *piece = only;
            return i == 0 && only.kb1 > only.kb0;
        }
        if (idles) return false;
        if (!failed && !mbar_wait_parked(smem_u32(&piece_full[i & 1]), (uint32_t)(i >> 1) & 1u, p.wait_limit)) failed = true;
        if (failed) return false;
        *piece = s_piece[i & 1];
        return piece->kb1 > 0;
    };

    if (warp == kMmaWarp + 3) {
        // ================= warp 7: the next piece, its queries, and who sees whom =====================================================
        Walk walk(p, units, groups, begin, end, kSmall ? 0 : s_tree, kSmall ? only.span : s_span, kSmall ? 0u : (uint32_t)(begin - s_first), tile_of_group);
        if constexpr (kSmall) walk.piece = only;
        int tree = -1;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (!failed && !mbar_wait_parked(smem_u32(bar), parity & 1u, p.wait_limit)) failed = true;
            failed = __any_sync(0xffffffffu, failed);
            return !failed;
        };
        int asked = 0;
        Item told = {};
        for (int i = 0; !idles; ++i) {
            bool more = kSmall && i == 0 && only.kb1 > only.kb0;
            if constexpr (!kSmall) {
                more = walk.next();
                if (more && walk.piece.part == 0) told = {walk.piece.parts, walk.piece.span.row0, walk.piece.span.nodes, walk.piece.head, walk.piece.tile};   // (only the last one can have more)
            }
            if (i >= 2 && !wait(&piece_empty[i & 1], (uint32_t)((i >> 1) - 1))) break;
            if (!kSmall && lane == 0) {
                s_piece[i & 1] = walk.piece;
                mbar_arrive(&piece_full[i & 1]);
            }
            __syncwarp();
            if (!more) break;
            auto ask = [&]() {   // the queries: rows of the tile's nodes x the head's queries, in the order of the tile's rows
                if (lane == 0) {
                    const uint32_t bar = smem_u32(&q_full);
                    mbar_expect_tx_addr(bar, (uint32_t)(p.tile_nodes * p.t.group) * 256u);
                    for (int h = 0; h < 2; ++h)
                        tma_load_4d(sQ + h * kQHalf, &p.q_map, 0, h, walk.piece.head * p.t.group, walk.piece.span.row0 + walk.piece.tile * p.tile_nodes, bar);
                }
                ++asked;
                __syncwarp();
            };
            if (i == 0) ask();
            const TreeSpan& span = walk.piece.span;
            if (walk.s != tree) {
                int up[kWords];   // (asked for together)
#pragma unroll
                for (int j = 0; j < kWords; ++j) up[j] = 32 * j + lane < span.nodes ? p.t.parent[span.row0 + 32 * j + lane] : -1;
#pragma unroll
                for (int j = 0; j < kWords; ++j) s_up[32 * j + lane] = tree_parent_of(up[j], 32 * j + lane, p.status);
                tree = walk.s;
                __syncwarp();
            }
            const int node0 = walk.piece.tile * p.tile_nodes, nodes = min(p.tile_nodes, span.nodes - node0);
            for (int k = lane; k < nodes; k += 32) {
                uint32_t bits[kWords] = {};
                for (int up = node0 + k; up >= 0; up = s_up[up])
#pragma unroll
                    for (int w = 0; w < kWords; ++w) bits[w] |= up >> 5 == w ? 1u << (up & 31) : 0u;
                uint4* to = reinterpret_cast<uint4*>(s_sees[i & 1][k]);
                to[0] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
                to[1] = make_uint4(bits[4], bits[5], bits[6], bits[7]);
            }
            if (lane < kWords) s_odd[i & 1][lane] = 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sees_full[i & 1]);
            if (i > 0) {
                if (!wait(&q_empty, (uint32_t)(i - 1))) break;   // the products with the last piece's queries are complete
                ask();
            }
        }
        if (!kSmall && p.items && lane == 0) p.items[blockIdx.x] = told;
        if (asked) mbar_wait_parked(smem_u32(&q_full), (uint32_t)(asked - 1) & 1u, p.wait_limit);   // (queries in flight write this CTA's shared memory)
        if (failed && lane == 0) atomicExch(p.status, 3);
    } else if (warp > kMmaWarp) {
        // ================= warps 5, 6: the pages of K and V ==========================================================================
        const int is_v = warp - kMmaWarp - 1;
        uint64_t* full = is_v ? v_full : k_full;
        uint64_t* empty = is_v ? v_empty : k_empty;
        const uint32_t base = is_v ? sV : sK;
        int g = 0;
        Piece piece;
        for (int i = 0; __all_sync(0xffffffffu, take(i, &piece)); ++i) {
            __syncwarp();
            if (lane == 0) mbar_arrive(&piece_empty[i & 1]);
            const int last_page = (piece.span.length + piece.span.nodes - 1) / kTreePage;
            const int* table = p.t.table + (long long)piece.span.slot * p.t.max_pages;
            auto page_of = [&](int kb) { return lane < kPages && kb < piece.kb1 && kb * kPages + lane <= last_page ? table[kb * kPages + lane] : -2; };
            int coming = kSmall ? first_page : page_of(piece.kb0);
            bool due = false;                                 // values of the block in front are to be looked through, before the product with them
            auto clean = [&](int g, int kb) {
                if (!mbar_wait_parked(smem_u32(&v_full[g & 1]), (uint32_t)(g >> 1) & 1u, p.wait_limit) ||
                    !mbar_wait_parked(smem_u32(&sees_full[i & 1]), (uint32_t)(i >> 1) & 1u, p.wait_limit))
                    failed = true;
                failed = __any_sync(0xffffffffu, failed);
                if (failed) return;
                clean_values(base + (g & 1) * kStage, piece.span, kb, s_odd[i & 1]);
                if (lane == 0) mbar_arrive(&p_full[g & 1]);
            };
            for (int kb = piece.kb0; kb < piece.kb1; ++kb, ++g) {
                const int page = coming;
                coming = page_of(kb + 1);
                if (g >= 2) {
                    if (due && !__all_sync(0xffffffffu, mbar_ready(&empty[g & 1], (uint32_t)((g - 2) >> 1) & 1u))) {
                        clean(g - 1, kb - 1);
                        due = false;
                    }
                    if (!mbar_wait_parked(smem_u32(&empty[g & 1]), (uint32_t)((g - 2) >> 1) & 1u, p.wait_limit)) failed = true;
                }
                failed = __any_sync(0xffffffffu, failed);
                if (failed) break;
                const bool there = lane < kPages && kb * kPages + lane <= last_page, good = there && page >= 0 && page < p.t.n_pages;
                const uint32_t bar = smem_u32(&full[g & 1]), dst = base + (g & 1) * kStage;
                const uint32_t bad = __ballot_sync(0xffffffffu, there && !good), load = __ballot_sync(0xffffffffu, good);
                if (bad) {   // nothing is seen of them, but a value that is NaN would count in spite of its weight of 0
                    for (uint32_t b = bad; b; b &= b - 1)
                        for (int k = lane; k < 2 * kTreePage * 8; k += 32)
                            st_shared_v4(dst + (k >> 7) * kHalf + (__ffs(b) - 1) * (kTreePage * 128) + (k & 127) * 16, 0, 0, 0, 0);
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
                    const int row0 = ((page * p.t.kv_heads + piece.head) * 2 + is_v) * kTreePage;
                    tma_load_3d(dst + lane * (kTreePage * 128), &p.map, 0, 0, row0, bar);
                    tma_load_3d(dst + kHalf + lane * (kTreePage * 128), &p.map, 0, 1, row0, bar);
                }
                __syncwarp();
                if (is_v) {
                    if (due) clean(g - 1, kb - 1);
                    due = (kb + 1) * kKeys > piece.span.length;
                    if (!due && lane == 0) mbar_arrive(&p_full[g & 1]);
                }
            }
            if (!failed && due) clean(g - 1, piece.kb1 - 1);
            if (failed) break;
        }
        // copies still in flight write this CTA's shared memory
        for (int k = max(g - 2, 0); k < g; ++k) mbar_wait_parked(smem_u32(&full[k & 1]), (uint32_t)(k >> 1) & 1u, p.wait_limit);
        if (__any_sync(0xffffffffu, failed) && lane == 0) atomicExch(p.status, 3);
    } else if (warp == kMmaWarp) {
        // ================= warp 4: one thread issues every product ===================================================================
        if (elect_one()) {
            auto wait = [&](uint64_t* bar, uint32_t parity) {
                if (!failed && !mbar_wait_parked(smem_u32(bar), parity & 1u, p.wait_limit)) failed = true;
                return !failed;
            };
            int issued = 0, piece_at = 0, in_piece = 0;   // blocks whose scores are under way; pieces taken; blocks of the last one that are left
            int coming[2] = {0, 0}, taken = 0;            // blocks of the pieces that P . V has yet to begin
            bool more = true;
            auto scores = [&]() {                         // of the next block, whichever piece it belongs to
                if (in_piece == 0) {
                    Piece piece;
                    if (!take(piece_at, &piece)) { more = false; return; }
                    mbar_arrive(&piece_empty[piece_at & 1]);
                    in_piece = piece.kb1 - piece.kb0;
                    coming[piece_at & 1] = in_piece;
                    if (!wait(&q_full, (uint32_t)piece_at)) return;
                    ++piece_at;
                }
                const int g = issued;
                if (!wait(&k_full[g & 1], (uint32_t)(g >> 1))) return;
                tc_fence_after();
                const uint64_t a = make_smem_desc(sQ), b = make_smem_desc(sK + (g & 1) * kStage);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    umma_bf16(tmem + (uint32_t)(g & 1) * kKeys, a + (uint64_t)((k >> 2) * (kQHalf >> 4) + 2 * (k & 3)), b + (uint64_t)((k >> 2) * (kHalf >> 4) + 2 * (k & 3)), kIdescS,
                              k > 0 ? 1u : 0u);
                umma_commit(&s_full[g & 1]);
                umma_commit(&k_empty[g & 1]);
                if (--in_piece == 0) umma_commit(&q_empty);
                ++issued;
            };
            scores();
            if (more) scores();
            int left = 0;
            for (int g = 0; !failed && g < issued; ++g) {
                const bool begins = left == 0;
                if (begins) left = coming[taken++ & 1];
                if (!wait(&p_full[g & 1], (uint32_t)(g >> 1)) || !wait(&v_full[g & 1], (uint32_t)(g >> 1))) break;
                tc_fence_after();
                const uint64_t b = make_smem_desc_mn(sV + (g & 1) * kStage);
#pragma unroll
                for (int k = 0; k < kKeys / 8; ++k)   // 16 keys: the weights' upper terms, and their lower ones
                    umma_bf16_ts(tmem + kOCol, tmem + (uint32_t)(g & 1) * kKeys + (k & 1) * (kKeys / 2) + 8u * (k >> 1), b + (uint64_t)((k >> 1) * (16 * 128 >> 4)), kIdescO,
                                 (!begins || k > 0) ? 1u : 0u);
                umma_commit(&v_empty[g & 1]);
                --left;
                if (more) scores();
            }
            if (failed) atomicExch(p.status, 3);
        }
        __syncwarp();
    } else {
        // ================= warps 0 - 3: softmax, a row per thread ====================================================================
        const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16), t_o = t_lane + kOCol;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (!failed && !mbar_wait_parked(smem_u32(bar), parity & 1u, p.wait_limit)) failed = true;
            failed = __any_sync(0xffffffffu, failed);
            return !failed;
        };
        const int my_node = tid / p.t.group, my_head = tid - my_node * p.t.group;
        int g = 0;
        Piece piece;
        if constexpr (kSmall) s_ml[tid] = make_float2(-INFINITY, 0.f);
        for (int at = 0; __all_sync(0xffffffffu, take(at, &piece)); ++at) {
            const TreeSpan& span = piece.span;
            const int node0 = piece.tile * p.tile_nodes, node = node0 + my_node;
            const bool live = my_node < p.tile_nodes && node < span.nodes;
            const uint32_t* sees = s_sees[at & 1][live ? my_node : 0];
            const bool idle = !__any_sync(0xffffffffu, live);   // no row of this warp is one
            float m = -INFINITY, l = 0.f;
            bool any = false, large = false, fresh = true, masked = false;
            for (int kb = piece.kb0; kb < piece.kb1; ++kb, ++g) {
                const uint32_t t_s = t_lane + (uint32_t)(g & 1) * kKeys;
                const bool tail = (kb + 1) * kKeys > span.length;
                if (!wait(&s_full[g & 1], (uint32_t)(g >> 1))) break;
                tc_fence_after();
                const uint32_t bad = s_bad[g & 3];
                if ((tail || bad) && !masked) {
                    if (!wait(&sees_full[at & 1], (uint32_t)(at >> 1))) break;
                    masked = true;
                }
                if (!idle) {
                    uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
                    if (tail || bad) {
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            vis[w] = bits_from(sees, kb * kKeys + 32 * w - span.length);
                            if (bad >> (2 * w) & 1) vis[w] &= 0xffff0000u;
                            if (bad >> (2 * w) & 2) vis[w] &= 0x0000ffffu;
                        }
                    }
                    any |= (vis[0] | vis[1]) != 0;
                    float sum = 0.f;
                    for (bool look = live && m == -INFINITY;;) {
                        uint32_t sr[kKeys], low[kKeys / 2];
                        if (fresh) {   // a new reference for some rows: the maximum of this block
                            tmem_ld_32_begin(t_s, sr);
                            tmem_ld_32_begin(t_s + 32, sr + 32);
                            tmem_ld_32_end(sr);
                            tmem_ld_32_end(sr + 32);
                            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                            for (int j = 0; j < kKeys; ++j)
                                if (vis[j >> 5] >> (j & 31) & 1) mx[j & 3] = fmaxf(mx[j & 3], __uint_as_float(sr[j]));
                            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
                            const float keep = look && top > m ? ex2(m - top) : 1.f;
                            if (look && top > m) m = top;
                            large = __any_sync(0xffffffffu, m > kLargeScore || (m < -kLargeScore && m > -INFINITY));
                            l *= keep;
                            if (kb > piece.kb0 && __any_sync(0xffffffffu, keep != 1.f)) {   // O of the blocks in front, once their last product is complete
                                if (!wait(&v_empty[(g - 1) & 1], (uint32_t)((g - 1) >> 1))) break;
                                tc_fence_after();
#pragma unroll 1
                                for (int c = 0; c < 4; ++c) {
                                    uint32_t r[32];
                                    tmem_ld_32_begin(t_o + 32u * c, r);
                                    tmem_ld_32_end(r);
#pragma unroll
                                    for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * keep);
                                    tmem_st_32(t_o + 32u * c, r);
                                }
                            }
                            fresh = __any_sync(0xffffffffu, live && m == -INFINITY);   // (a row that has seen nothing looks again)
                        }
                        // ---- the weights, one pass over the scores: half of them on their way while the other half is worked on
                        const float ref = m == -INFINITY ? 0.f : m;
                        const uint64_t scale2 = pair_of(p.scale_log2, p.scale_log2), ref2 = pair_of(-ref, -ref);
                        uint64_t sums[2] = {0, 0};
                        tmem_ld_32_begin(t_s, sr);
                        tmem_ld_32_end(sr);
                        tmem_ld_32_begin(t_s + 32, sr + 32);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t* x = sr + 32 * h;
                            if (h) tmem_ld_32_end(x);
                            if (tail || bad) {
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (!(vis[h] >> j & 1)) x[j] = 0xff800000u;
                            }
                            if (large) {
#pragma unroll
                                for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(x[i]), p.scale_log2), ref));
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; ++i) {
                                    const float2 e = split(fma2(pair_of(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale2, ref2));
                                    x[2 * i] = __float_as_uint(e.x);
                                    x[2 * i + 1] = __float_as_uint(e.y);
                                }
                            }
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float w0 = ex2(__uint_as_float(x[2 * i])), w1 = ex2(__uint_as_float(x[2 * i + 1]));
                                sums[i & 1] = add2(sums[i & 1], pair_of(w0, w1));
                                const uint32_t high = pack_bf16x2(w0, w1);
                                const float2 rest = split(fma2(pair_of(__uint_as_float(high << 16), __uint_as_float(high & 0xffff0000u)), pair_of(-1.f, -1.f), pair_of(w0, w1)));
                                sr[16 * h + i] = high;   // (the places of scores that are done with)
                                low[16 * h + i] = pack_bf16x2(rest.x, rest.y);
                            }
                        }
                        const float2 s01 = split(add2(sums[0], sums[1]));
                        sum = s01.x + s01.y;
                        look = live && sum > kMostSum;
                        if (!__any_sync(0xffffffffu, look)) {
                            tmem_st_16(t_s, sr);
                            tmem_st_16(t_s + 16, sr + 16);
                            tmem_st_16(t_s + 32, low);
                            tmem_st_16(t_s + 48, low + 16);
                            break;
                        }
                        fresh = true;
                    }
                    l += sum;
                    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                }
                if (failed) break;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[g & 1]);
            }
            // ---- O / l, or the row's part of it
            if (failed || !wait(&v_empty[(g - 1) & 1], (uint32_t)((g - 1) >> 1))) break;
            tc_fence_after();
            if (!idle) {
                if (any && m == -INFINITY && l == 0.f) l = 1.f;  // scores of -inf alone
                uint32_t odd = 0;
                if (masked) {   // (the wait is over: it orders what the values' warp has found before the reads)
                    if (!wait(&p_full[(g - 1) & 1], (uint32_t)((g - 1) >> 1))) break;
#pragma unroll
                    for (int w = 0; w < kWords; ++w) odd |= s_odd[at & 1][w] & sees[w];
                }
                if (__any_sync(0xffffffffu, live && odd)) {     // the values that the products left out, for the rows that see them
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        uint32_t o[32];
                        __syncwarp();
                        tmem_ld_32_begin(t_o + 32u * c, o);
                        tmem_ld_32_end(o);
                        for (int i = 0; live && i < span.nodes; ++i) {
                            if (!(s_odd[at & 1][i >> 5] & sees[i >> 5] & 1u << (i & 31))) continue;
                            const int where = span.length + i;
                            const long long place = tree_place(p.t, span.slot, where, p.status);
                            if (place < 0) continue;
#pragma unroll
                            for (int j = 0; j < 32; ++j) {
                                const int chunk = 4 * c + (j >> 3);
                                const uint16_t v = *reinterpret_cast<const uint16_t*>(p.pool + place + (2 * piece.head + 1) * kTreeBlock + ((chunk ^ (where & 7)) << 4) + 2 * (j & 7));
                                if (not_finite(v)) o[j] = __float_as_uint(__uint_as_float(o[j]) + __uint_as_float((uint32_t)v << 16));
                            }
                        }
                        __syncwarp();
                        tmem_st_32(t_o + 32u * c, o);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                }
                uint4* dst = reinterpret_cast<uint4*>(p.out + ((long long)(span.row0 + node) * p.t.q_heads + piece.head * p.t.group + my_head) * kTreeDim);
                if (kSmall && p.cluster > 1) {                  // (the share's sums go to the other CTAs, see below)
                    if (live) s_ml[kSmall ? tid : 0] = make_float2(m, l);
                } else if (piece.parts == 1) {
                    const float inv = inverse_of(m, l);
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        float o[32];
                        __syncwarp();
                        tmem_ld_32(t_o + 32u * c, o);
                        if (!live) continue;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            dst[4 * c + i] = make_uint4(pack_bf16x2(o[8 * i] * inv, o[8 * i + 1] * inv), pack_bf16x2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                                        pack_bf16x2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack_bf16x2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                    }
                } else if constexpr (!kSmall) {
                    if (!join_parts(p, piece, live, t_o, m, l, dst)) {
                        failed = true;
                        break;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&piece_empty[at & 1]);
        }
        if (__any_sync(0xffffffffu, failed) && lane == 0) atomicExch(p.status, 3);
    }
    __syncwarp();
    tc_fence_before();
    if (kSmall && p.cluster > 1) {
        // ---- the share's sums to shared memory, where the stages and the queries were: two warps for 32 rows, half of the channels each
        const TreeSpan& span = only.span;
        const int node0 = only.tile * p.tile_nodes, rows = idles ? 0 : min(p.tile_nodes, span.nodes - node0) * p.t.group;
        __syncthreads();
        tc_fence_after();
        if (only.kb1 > only.kb0 && (warp & 3) * 32 < rows) {
            const int row = (warp & 3) * 32 + lane, c0 = (warp >> 2) * (kTreeDim / 2);
#pragma unroll 1
            for (int c = c0; c < c0 + kTreeDim / 2; c += 32) {
                float o[32];
                __syncwarp();
                tmem_ld_32(tmem + ((uint32_t)((warp & 3) * 32) << 16) + kOCol + (uint32_t)c, o);
                if (row >= rows) continue;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    st_shared_v4(sQ + (row * kORow + c + 4 * i) * 4, __float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]), __float_as_uint(o[4 * i + 2]), __float_as_uint(o[4 * i + 3]));
            }
            __syncwarp();
        }
        tc_fence_before();
        // ---- the shares of the cluster's task, in the order of the keys: a CTA takes every cluster-th row, a warp a row at a time, four channels a lane
        cluster_sync_all();
        const uint32_t ml_at = smem_u32(s_ml);
        for (int row = rank + p.cluster * warp; row < rows; row += p.cluster * (kThreads / 32)) {
            float2 ml[8];
            float4 v[8];
            float top = -INFINITY, l = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                ml[k] = make_float2(-INFINITY, 0.f);
                if (k < p.cluster) {
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];\n" : "=f"(ml[k].x), "=f"(ml[k].y) : "r"(map_to_cta(ml_at + 8 * row, k)));
                    v[k] = ld_dsmem_f4(map_to_cta(sQ + (row * kORow + 4 * lane) * 4, k));
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;   // (a share without keys has no sums)
                const float f = ex2(ml[k].x - ref);
                l += share_of(ml[k], f, top);
                if (k < p.cluster) { o.x += v[k].x * f; o.y += v[k].y * f; o.z += v[k].z * f; o.w += v[k].w * f; }
            }
            const float inv = inverse_of(top, l);
            const int node = row / p.t.group;
            *reinterpret_cast<uint2*>(p.out + ((long long)(span.row0 + node0 + node) * p.t.q_heads + only.head * p.t.group + (row - node * p.t.group)) * kTreeDim + 4 * lane) =
                make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        }
        cluster_sync_all();   // nobody leaves while its sums are read
    }
    __syncthreads();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

// Joins the parts of items. A piece of work is (item, 32 rows, 32 channels), dealt out in turn: every CTA lists the items for itself.
constexpr int kJoinThreads = 256, kMostItems = 512;
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(const __grid_constant__ AttentionParams p) {
    __shared__ __align__(16) __nv_bfloat16 s_out[32][32 + 8];
    __shared__ int s_cta[kMostItems], s_count[kMostItems / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int per = p.row_cap / 32 * 4, ctas = p.groups * p.tiles, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t has[kMostItems / kJoinThreads];
#pragma unroll
    for (int i = 0; i < kMostItems / kJoinThreads; ++i) {
        const int cta = i * kJoinThreads + threadIdx.x;
        has[i] = __ballot_sync(0xffffffffu, cta < ctas && p.items[cta].parts > 1);
        if (lane == 0) s_count[i * (kJoinThreads / 32) + warp] = __popc(has[i]);
    }
    __syncthreads();
    int items = 0;
#pragma unroll
    for (int i = 0; i < kMostItems / 32; ++i) {
        if (i % (kJoinThreads / 32) == warp && (has[i / (kJoinThreads / 32)] >> lane & 1)) s_cta[items + __popc(has[i / (kJoinThreads / 32)] & ((1u << lane) - 1u))] = i * 32 + lane;
        items += s_count[i];
    }
    __syncthreads();
    for (int w = blockIdx.x; w < items * per; w += gridDim.x) {
        const int cta = s_cta[w / per], quarter = w & 3, row = w % per / 4 * 32 + lane;
        const Item item = p.items[cta];
        const int rows = min(p.tile_nodes, item.nodes - item.tile * p.tile_nodes) * p.t.group;
        if (row - lane >= rows) continue;   // the whole CTA
        float top = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        constexpr int kAtOnce = 16;   // (with four at a time the loads' latencies of 18 parts added up to 15 us)
        for (int k0 = 0; k0 < item.parts && row < rows; k0 += kAtOnce) {
            float2 ml[kAtOnce];
            float4 v[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int part = min(k0 + k, item.parts - 1);
                const size_t slot = 2 * ((size_t)cta + (size_t)part * p.tiles) + (part == 0 ? 1 : 0);
                v[k] = load_now(p.sums + (slot * 32 + 8 * quarter + warp) * p.row_cap + row);
                ml[k] = p.ml[slot * p.row_cap + row];
            }
            float to = top;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (k0 + k >= item.parts) ml[k] = make_float2(-INFINITY, 0.f);
                to = fmaxf(to, ml[k].x);
            }
            const float ref = to == -INFINITY ? 0.f : to, keep = to == top ? 1.f : ex2(top - ref);
            l = share_of(make_float2(top, l), keep, to);
            top = to;
            o.x *= keep; o.y *= keep; o.z *= keep; o.w *= keep;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (k0 + k >= item.parts) break;
                const float f = ex2(ml[k].x - ref);
                l += share_of(ml[k], f, to);
                o.x += v[k].x * f; o.y += v[k].y * f; o.z += v[k].z * f; o.w += v[k].w * f;
            }
        }
        const float inv = inverse_of(top, l);
        *reinterpret_cast<uint2*>(&s_out[lane][4 * warp]) = make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        __syncthreads();
        const int r = threadIdx.x >> 2, rr = row - lane + r, chunk = 8 * (threadIdx.x & 3);
        if (r < 32 && rr < rows)
            *reinterpret_cast<uint4*>(p.out + ((long long)(item.row0 + item.tile * p.tile_nodes + rr / p.t.group) * p.t.q_heads + item.head * p.t.group + rr % p.t.group) * kTreeDim +
                                      32 * quarter + chunk) = *reinterpret_cast<const uint4*>(&s_out[r][chunk]);
        __syncthreads();
    }
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

// The queries: rows (w), heads (z), halves (y) of 64 channels (x); a copy brings a kv head's queries of a tile's nodes, node by node.
int encode_queries(const void* q, int64_t ldq, const DraftTrees& t, int tile_nodes, CUtensorMap* map) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return fail(GPTRS_EXECUTION, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[4] = {64, 2, (cuuint64_t)t.q_heads, (cuuint64_t)t.rows};
    cuuint64_t strides[3] = {128, 256, (cuuint64_t)ldq * 2};
    cuuint32_t box[4] = {64, 1, (cuuint32_t)t.group, (cuuint32_t)tile_nodes};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GPTRS_EXECUTION, "cuTensorMapEncodeTiled failed for the queries (" + std::to_string((int)r) + ")");
    return GPTRS_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How a call is cut. The host does not know the lengths, but the page table's width bounds them. Small: a cluster per (tree, kv head, row tile), with as many CTAs (8, 4, 2, 1) as
// leave a processor, or half of one, to each; taken where the longest context can cost no more than equal shares of all of them and their joins, which take as long as
// twenty blocks. Others: as many CTAs as there are places, in groups of one, or of two where trees may have more rows than a tile.
struct Cut { int cluster, ctas, groups, tiles, row_cap, tile_nodes, most_tiles; bool small, joined_after; };
Cut cut(const gptrs_draft_trees* t) {
    Cut c;
    const int group = t->q_heads / t->kv_heads, rows = t->max_nodes * group;
    c.tile_nodes = kRows / group;
    c.most_tiles = ceil_div(t->max_nodes, c.tile_nodes);
    const int64_t sms = sm_count(), tasks = t->n_trees * t->kv_heads * c.most_tiles, longest = ceil_div(t->max_pages * kTreePage, kKeys);
    c.cluster = tasks * 8 <= sms ? 8 : tasks * 4 <= sms ? 4 : tasks * 2 <= 2 * sms ? 2 : 1;
    c.small = tasks * c.cluster <= 2 * sms ? longest / c.cluster <= tasks * longest / (2 * sms) + 20 : tasks < (1 << 24) && longest <= 20;
    c.tiles = !c.small && c.most_tiles > 1 ? 2 : 1;
    c.ctas = c.small ? c.most_tiles * c.cluster : (int)(2 * sms < kMostItems ? 2 * sms : kMostItems);
    // a level of joins by warps takes 6 to 8 us at the end of a call, the second kernel 7 us, but while others still work on their keys the former cost nothing
    c.joined_after = !c.small && t->n_trees * t->kv_heads * ceil_div(c.most_tiles, c.tiles) * 4 <= 2 * sms / c.tiles;
    c.groups = (int)(2 * sms < kMostItems ? 2 * sms : kMostItems) / c.tiles;
    c.row_cap = rows < kRows ? (rows + 31) / 32 * 32 : kRows;
    return c;
}
size_t count_words(int groups, int tiles) { return (size_t)kLevels * 2 * groups * tiles * kSoftmaxWarps; }

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" {

size_t gptrs_cuda_tree_scratch_bytes(const gptrs_draft_trees* t) {
    DraftTrees checked;
    if (draft_trees(t, &checked) != GPTRS_OK) return 0;
    const Cut c = cut(t);
    if (c.small) return 0;
    const size_t slots = 2 * (size_t)c.groups * c.tiles;
    return 2 * count_words(c.groups, c.tiles) * sizeof(uint32_t) + slots * c.row_cap * (sizeof(float2) + 32 * sizeof(float4));
}

int gptrs_cuda_tree_attention(const gptrs_draft_trees* t, const gptrs_tree_attention_step* s, void* stream) {
    AttentionParams p = {};
    const int rc = draft_trees(t, &p.t);
    if (rc) return rc;
    GPTRS_REQUIRE(s && s->d_pool && s->d_status && (t->rows == 0 || (s->d_q && s->d_out)), "null pointer");
    GPTRS_REQUIRE(aligned16(s->d_q) && aligned16(s->d_pool) && aligned16(s->d_out) && aligned16(s->d_scratch), "pointers must be 16-byte aligned");
    const int64_t width = (int64_t)t->q_heads * kTreeDim;
    const int64_t ldq = s->ldq ? s->ldq : width;
    GPTRS_REQUIRE(ldq >= width && ldq % 8 == 0 && ldq < ((int64_t)1 << 31), "rows of queries overlap, or do not start at multiples of 16 bytes");
    GPTRS_REQUIRE(t->n_pages * t->kv_heads * 2 * kTreePage < ((int64_t)1 << 31), "the pool has too many pages");
    GPTRS_REQUIRE(t->max_pages * kTreePage / kKeys + 8 < (((int64_t)1 << 31) / ceil_div(t->max_nodes, kRows / (t->q_heads / t->kv_heads)) / t->kv_heads), "the page table is too long for so many rows");
    const size_t scratch = gptrs_cuda_tree_scratch_bytes(t);
    GPTRS_REQUIRE(scratch == 0 || (s->d_scratch && s->scratch_bytes >= scratch), "scratch is too small");
    if (t->rows == 0) return GPTRS_OK;
    const char *q = static_cast<const char*>(s->d_q), *out = static_cast<const char*>(s->d_out);
    GPTRS_REQUIRE(out >= q + 2 * ((t->rows - 1) * ldq + width) || q >= out + 2 * t->rows * width, "the output lies in rows of queries");
    static PerDeviceOnce attr_once;
    if (attr_once.first_time()) {
        GPTRS_CUDA_OK(cudaFuncSetAttribute(tree_attention_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
        GPTRS_CUDA_OK(cudaFuncSetAttribute(tree_attention_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem));
    }
    const Cut c = cut(t);
    p.cluster = c.cluster; p.groups = c.groups; p.tiles = c.tiles; p.row_cap = c.row_cap; p.tile_nodes = c.tile_nodes;
    int bad = encode_pool(s->d_pool, p.t, &p.map);
    if (!bad) bad = encode_queries(s->d_q, ldq, p.t, p.tile_nodes, &p.q_map);
    if (bad) return bad;
    p.pool = static_cast<const unsigned char*>(s->d_pool);
    p.out = static_cast<__nv_bfloat16*>(s->d_out);
    p.status = s->d_status;
    p.scale_log2 = (t->scale != 0.f ? t->scale : 1.f / sqrtf((float)kTreeDim)) * kLog2e;
    const size_t slots = 2 * (size_t)p.groups * p.tiles;
    p.done = static_cast<uint32_t*>(s->d_scratch);
    if (c.joined_after) p.items = reinterpret_cast<Item*>(p.done);   // (the counts are not used then; they take more room)
    p.stored = p.done + count_words(p.groups, p.tiles);
    p.sums = reinterpret_cast<float4*>(p.stored + count_words(p.groups, p.tiles));
    p.ml = reinterpret_cast<float2*>(p.sums + slots * 32 * p.row_cap);
    prefill_tc_fault(&p.starve, &p.wait_limit);
    if (c.small) return launch_kernel(tree_attention_kernel<true>, dim3((unsigned)c.ctas, (unsigned)t->kv_heads, (unsigned)t->n_trees), dim3(kThreads), kSmem, as_stream(stream), 1, p, c.cluster);
    bad = launch_kernel(tree_attention_kernel<false>, dim3((unsigned)c.ctas), dim3(kThreads), kSmem, as_stream(stream), 1, p);
    if (bad || !c.joined_after) return bad;
    // the second kernel waits for the first one itself (griddepcontrol.wait), so it may be launched ahead of its end
    const int pdl = g_use_pdl;
    g_use_pdl = 1;
    bad = launch_kernel(tree_join_kernel, dim3((unsigned)(2 * sm_count())), dim3(kJoinThreads), 0, as_stream(stream), 1, p);
    g_use_pdl = pdl;
    return bad;
}

}  // extern "C"
