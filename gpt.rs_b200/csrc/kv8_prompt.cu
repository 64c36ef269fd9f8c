// Attention over the 8-bit cache for tiles of rows of one sequence (prompts), on the tcgen05 tensor cores.
//
// The formula of kv8_attention.cu: t = (s_K scale log2 e) q . a + log2 s_V, w = 2^(t - M), out = sum w b / sum (w / s_V). Whole numbers of 8 bits
// become f16 in shared memory (exact), the scales of a block of 16 keys meet the scores of its 16 columns, so the matrix products see no scale.
//
// One CTA (one per SM) takes the rows of a tile x the query heads of one kv head, as two row tiles of 128 (row = token x group + head), and walks
// the visible keys in blocks of 128 (8 pages), two halves of 64 keys in flight on their own (h):
//   S_ih[128 x 64] = Q_i . K_h^T   both operands f16 in shared memory (K-major, 128-byte swizzle), accumulator in tensor memory
//   softmax                        warps 4 i .. 4 i + 3, a thread per row, in one pass over its scores: the reference M stays what it is until a weight would
//                                  no longer be an f16 (a page's weights add up to more than 65504), so there is no pass for the maximum. It is set
//                                  to 2 below a maximum: a row's largest weight is 2^2 or more, others have 11 bits down to 2^-16 of it and are off
//                                  by at most 2^-27 of it below (the 2^19 tokens of a tail lose 2^-8 of the sum at most, as much as the result's rounding).
//                                  Weights go as f16 over the first 32 columns of S_ih
//   O_i[128 x dim] += P_ih . V_h   A = P_ih from tensor memory, B = V^T in shared memory (keys contiguous), accumulator in tensor memory
// Warps 8 - 11 widen the pages, two of a block each: bytes from global memory to registers ahead of time, f16 into the stage when the products that read
// it are complete. A thread of theirs takes the 16 bytes that the row kernel's lane would; which 16 is chosen so that eight (K) or sixteen (V) threads
// store to different banks. The order of the keys inside a page is the cache's (pairs 0, 1, 8, 9, 2, 3, ...): P's columns are written in the same
// order. Warps 12 and 13 issue the products of a row tile each: behind P_ih come O_i += P_ih . V_h and the next block's S_ih, while the softmax is at the
// other half. One thread for both tiles had the one wait for the other's weights (547 us for the prompt below).
//
// One prompt of 8192 tokens, 32 / 8 heads of 128: 521 us, 1055 TFLOP/s (64 % of what a large bf16 product of the library reaches), where the reference is hardly
// ever raised, 552 us where blocks' scales and scores scatter widely; 500 tokens behind 32768 282 and 311 us; seven ragged prompts of 91 - 1777 tokens, 12 heads
// of 64: 54.5 us. What bounds long ones is the softmax warps' chain: a half takes a warp
// about 1700 cycles (1150 of weights, 230 until the scores are seen, 150 of storing them), of which the special function unit needs 512 for each of the two
// warps of a scheduler; it issues in 39 % of the cycles, a third of that for the loaders, and the tensor pipe is busy for 38 %. Short ones pay 8.5 us per CTA
// beside their keys: 2 of loads that depend on each other (tile, slot, length), 2 until the first scores, 2 for these (maximum and masks), 1.5 for the
// output and 1 between CTAs; a half is 0.95 us. Measured and left: two threads a row (16 softmax warps, 667 us where one had 606), eight loader warps (539
// where four had 518), an eighth of the exponentials as a polynomial on the multiply-add units (519 and, for the chunk, 292, where all on the special
// function unit took 524 and 288), whole blocks of scores instead of halves (690), first halves without masks where all see them (no difference).
// Every wait is bounded: on a timeout code 3 goes to the status word and every role leaves its loop.
#include <type_traits>

#include "kv8_attention.cuh"
#include "umma_common.cuh"

namespace gptrs {

void prefill_tc_fault(int* starve, uint32_t* wait_limit);   // the test switch of paged_prefill_tc.cu

namespace {

constexpr int kRows = 128;                 // of a row tile = lanes of tensor memory
constexpr int kTiles = 2;
constexpr int kSoftmaxThreads = kTiles * kRows;
constexpr int kLoadWarps = 4;
constexpr int kLoadWarp = kSoftmaxThreads / 32, kMmaWarp = kLoadWarp + kLoadWarps;
constexpr int kThreads = kSoftmaxThreads + kLoadWarps * 32 + 128;   // two warps for the products and two that only make their group whole
// Registers of a thread at launch, and what the groups of four warps make of them: the shares add up to what the block has, so every request ends.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 160, kLoadRegs = kLaunchRegs, kMmaRegs = 64;
static_assert(kThreads == 512 && 2 * kSoftmaxRegs + kLoadRegs + kMmaRegs <= 4 * kLaunchRegs, "more registers than the block is launched with");
constexpr int kKeys = 128;                 // of a block
constexpr int kPages = kKeys / kKv8Tokens;
constexpr int kHalfBytes = 128 * 128;      // 128 rows x 64 f16
constexpr uint32_t kTmemCols = 512;        // S_0, S_1, O_0, O_1
constexpr uint32_t kOCol = 256;
constexpr float kLargestSum = 65504.f;     // of a page's weights: each is an f16 then
// log2 of the largest weight behind a new reference: bits for the tail, which scores that grow along the keys cannot use (the reference is raised more often). us
// of 8192 tokens, 32 / 8 heads of 128, with 0 / 2 / 3 / 4: scores with a standard deviation of 2 520 for all, of 4 542 / 556 / 581 / 620; keys of scales that differ 541 / 547 / 553 / 561.
constexpr float kHeadroom = 2.f;
constexpr int kScaleSlots = 4;             // blocks whose scales may be in use at a time are three at most

struct PromptParams {
    Kv8Attention a;
    int starve;
    uint32_t wait_limit;
};

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) { umma_bf16(d, a, b, idesc, accumulate); }

__device__ __forceinline__ void tmem_ld_32_async(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                 "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ void st_shared_v2(uint32_t addr, uint32_t a, uint32_t b) {
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};\n" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
    const uint4 v = ld_shared_v4(addr);
    return make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
}

template <int kDim>
constexpr size_t prompt_smem() { return (size_t)(kTiles + 2) * kRows * kDim * 2 + 2 * (size_t)kDim * kKeys * 2 + 1024; }

template <int kDim>
__global__ void __launch_bounds__(kThreads, 1) kv8_prompt_kernel(const __grid_constant__ PromptParams params) {
    const Kv8Attention& p = params.a;
    constexpr int kQBytes = kRows * kDim * 2, kKBytes = kKeys * kDim * 2, kVHalf = kDim * 128;   // a half of V^T: 64 keys
    constexpr int kC = kDim / 32;
    constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kRows >> 4) << 24);                       // f32 accumulator, f16 operands, M = 128
    constexpr uint32_t kIdescS = kIdesc | ((uint32_t)(kKeys / 2 >> 3) << 17), kIdescO = kIdesc | ((uint32_t)(kDim >> 3) << 17);

    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t k_first, k_read, full[2], empty[2], s_full[kTiles][2], p_full[kTiles][2], o_first[kTiles], o_full[kTiles], drained[kTiles];
    __shared__ uint32_t tmem_holder;
    __shared__ int s_begin[kSoftmaxThreads / 32], s_end[kSoftmaxThreads / 32];
    __shared__ __align__(16) float scales[kScaleSlots][kPages][4];   // s_K scale log2 e, log2 s_V, 1 / s_V

    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t sQ = smem, sK = sQ + kTiles * kQBytes, sV = sK + 2 * kKBytes;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool is_softmax = tid < kSoftmaxThreads;
    const int ti = is_softmax ? tid >> 7 : 0, row = tid & (kRows - 1);
    const int group = p.group, tq = kRows / group;
    const int kv_head = blockIdx.x, tile = (int)gridDim.y - 1 - (int)blockIdx.y;   // the longest contexts come last in a chunk: start them first

    pdl_wait();
    const int row0 = kv8_row(p, tile * p.tile_tokens);   // (tile_tokens: 2 tq)
    if (row0 < 0) return;
    const int n_rows = p.tile_rows[tile];
    int slot = p.slot[row0];
    if (slot >= p.n_slots) slot = -1;   // (the rows' spans report it)

    if (tid == 0) {
        mbar_init(&k_first, kLoadWarps);
        mbar_init(&k_read, kTiles);
        for (int i = 0; i < 2; ++i) { mbar_init(&full[i], kLoadWarps); mbar_init(&empty[i], kTiles); }
        for (int i = 0; i < kTiles; ++i) {
            for (int h = 0; h < 2; ++h) { mbar_init(&s_full[i][h], 1); mbar_init(&p_full[i][h], kRows); }
            mbar_init(&o_first[i], 1);
            mbar_init(&o_full[i], 1);
            mbar_init(&drained[i], 1);
        }
        mbar_fence_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_holder)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    // ---- a softmax thread's row ------------------------------------------------------------------------------------------------------------
    const int in_tile = ti * tq + row / group, my_row = row0 + in_tile, my_head = kv_head * group + row % group;
    bool live = is_softmax && row < tq * group && in_tile < n_rows;   // the output of this row is this thread's
    int begin = 0, end = 0;
    float q_scale = 0.f;
    if (is_softmax) {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + (live ? my_row : row0) * p.ldq + (long long)my_head * kDim);
        uint4 v[kDim / 8];
#pragma unroll
        for (int c = 0; c < kDim / 8; ++c) v[c] = live ? __ldg(src + c) : make_uint4(0, 0, 0, 0);   // (on its way beside the span)
        if (live) {
            const Kv8Span s = kv8_span(p, my_row);
            live = s.slot >= 0 && s.slot == slot;
            if (s.slot >= 0 && s.slot != slot) atomicExch(p.status, 2);   // a tile is of one sequence
            if (live) { begin = s.begin; end = s.end; }
        }
        const int warp_begin = __reduce_min_sync(0xffffffffu, end > begin ? begin : 0x7fffffff), warp_end = __reduce_max_sync(0xffffffffu, end > begin ? end : 0);
        if (lane == 0) { s_begin[warp] = warp_begin; s_end[warp] = warp_end; }
        // ---- its query: f16 with a power of two in front (kv8_cache.cuh) -> shared memory --------------------------------------------------------
        uint32_t big = 0;
#pragma unroll
        for (int c = 0; c < kDim / 8; ++c) {
            if (!live) v[c] = make_uint4(0, 0, 0, 0);
            big = __vmaxu2(big, __vmaxu2(abs_bits_max2(v[c].x, v[c].y), abs_bits_max2(v[c].z, v[c].w)));
        }
        const int e = pow2_exponent(widest_half(big));
        const float factor = e == 128 ? 0.f : pow2(-e);
        q_scale = e == 128 ? __uint_as_float(0x7fc00000u) : pow2(e);
        const uint32_t dst = sQ + ti * kQBytes + row * 128;
#pragma unroll
        for (int c = 0; c < kDim / 8; ++c)
            st_shared_v4(dst + (c >> 3) * kHalfBytes + (((c & 7) ^ (row & 7)) << 4), bf16x2_to_f16x2(v[c].x, factor), bf16x2_to_f16x2(v[c].y, factor),
                         bf16x2_to_f16x2(v[c].z, factor), bf16x2_to_f16x2(v[c].w, factor));
        fence_proxy_async();
    }
    // ---- what a loader's thread does (warps 8 - 11: pages 2 w, 2 w + 1 of every block) -------------------------------------------------------
    int first_key = 0x7fffffff, last_key = 0, n_blocks = 0, length = 0, end_block = 0;   // of this CTA: keys [first_key, last_key), blocks of 128; tokens, blocks of 16
    // whole blocks of the split's share of a tile's keys
    auto cut = [&](int from, int to) {
        first_key = from; last_key = to; n_blocks = 0;
        if (last_key <= 0) return;
        first_key = first_key / kKv8Tokens * kKv8Tokens;
        const int all = (last_key - first_key + kKeys - 1) / kKeys, per = (all + p.splits - 1) / p.splits, skip = min((int)blockIdx.z * per, all);
        n_blocks = min(per, all - skip);
        first_key += skip * kKeys;
        end_block = (last_key + kKv8Tokens - 1) / kKv8Tokens;
    };
    const int w = warp - kLoadWarp;
    const int kg = lane >> 3, kc = (lane >> 2) & 1, t = lane & 3;           // K: token, chunk of 32 channels, eight channels
    const int vg = 2 * ((lane & 15) >> 2) + (lane >> 4);                    // V: channel, four tokens
    enum { kNone, kClosed, kOpen };
    struct Page { const unsigned char* at; int block, kind; };
    auto block_of = [&](int kb, int j) { return first_key / kKv8Tokens + kb * kPages + 2 * w + j; };
    // entry of the page table, asked for a block before it is needed (the load is not waited for here)
    auto number = [&](int kb, int j) {
        const int block = block_of(kb, j);
        return block < end_block && (block + 1) * kKv8Tokens <= length ? p.table[slot * p.max_pages + block] : 0;
    };
    auto find = [&](int kb, int j, int page) {
        Page pg = {nullptr, block_of(kb, j), kNone};
        if (pg.block >= end_block) return pg;
        if ((pg.block + 1) * kKv8Tokens > length) { pg.kind = kOpen; return pg; }
        if (page < 0 || page >= p.n_pages) { atomicExch(p.status, 2); return pg; }
        pg.at = p.pool + ((long long)page * p.kv_heads + kv_head) * kv8_block_bytes(kDim);
        pg.kind = kClosed;
        return pg;
    };
    uint4 kb_[2][kC], vb_[2][kC];
    float2 sc[2];
    auto load_k = [&](const Page (&pg)[2]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (pg[j].kind != kClosed) continue;
            sc[j] = __ldg(reinterpret_cast<const float2*>(pg[j].at + 32 * kDim));
#pragma unroll
            for (int i = 0; i < kC; ++i)   // two channel chunks and tokens kg, kg + 4 of them
                kb_[j][i] = __ldg(reinterpret_cast<const uint4*>(pg[j].at + ((i >> 1) * 2 + kc) * 512 + ((kg + 4 * (i & 1)) * 4 + t) * 16));
        }
    };
    auto load_v = [&](const Page (&pg)[2]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (pg[j].kind != kClosed) continue;
#pragma unroll
            for (int i = 0; i < kC; ++i) vb_[j][i] = __ldg(reinterpret_cast<const uint4*>(pg[j].at + 16 * kDim + i * 512 + (vg * 4 + t) * 16));
        }
    };
    Page pages[2], next[2];
    int numbers[2];
    int asked_first = -1, asked_last = -1;
    auto ask_first = [&] {   // for block 0
#pragma unroll
        for (int j = 0; j < 2; ++j) pages[j] = find(0, j, number(0, j));
        load_k(pages);
        load_v(pages);
        asked_first = first_key;
        asked_last = last_key;
    };
    if (warp >= kLoadWarp && warp < kMmaWarp && slot >= 0) {
        // Pages of block 0 are asked for beside the queries: rows come at consecutive positions, so the keys go from the first row's to the last row's. Asked
        // for again where the rows say otherwise.
        const int last_row = row0 + n_rows - 1, last_slot = p.slot[last_row];
        length = p.length[slot];
        const int first_end = min(min(p.ctx_len[row0], p.max_len), length), last_end = min(min(p.ctx_len[last_row], p.max_len), length);
        if (last_slot == slot && first_end > 0 && last_end >= first_end) {
            cut(p.window > 0 ? max(0, first_end - p.window) : 0, last_end);
            if (n_blocks > 0) ask_first();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_holder;
    pdl_launch_dependents();   // every CTA of this grid holds its tensor memory (or has left)
    int tile_end[kTiles], from = 0x7fffffff, to = 0, nb_t[kTiles] = {0, 0};   // blocks of row tile i
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
        tile_end[i] = max(max(s_end[4 * i], s_end[4 * i + 1]), max(s_end[4 * i + 2], s_end[4 * i + 3]));
        to = max(to, tile_end[i]);
        from = min(from, min(min(s_begin[4 * i], s_begin[4 * i + 1]), min(s_begin[4 * i + 2], s_begin[4 * i + 3])));
    }
    cut(from, to);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) nb_t[i] = min(n_blocks, max(0, (tile_end[i] - first_key + kKeys - 1) / kKeys));
    bool failed = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {   // whole warp
        if (!failed && !mbar_wait_parked(smem_u32(bar), parity, params.wait_limit)) failed = true;
        failed = __any_sync(0xffffffffu, failed);
        return !failed;
    };

    if (warp >= kMmaWarp + kTiles) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kMmaRegs));
    } else if (warp >= kLoadWarp && warp < kMmaWarp) {
        // ================= warps 8 - 11: pages 2 w, 2 w + 1 of every block ===================================================================
        auto open_rows = [&](int block, int is_value) {
            return p.open + (long long)slot * kv8_open_elems(p.kv_heads, kDim) + kv8_open_at(block, p.kv_heads, kv_head, is_value, kDim);
        };
        // The block that is not complete: exponents of its largest finite key and value, and its tokens with one that is not finite. Their keys go as NaN, so that
        // their weights are none for the rows that see them, and values that are not finite as zero, or 0 x infinity would reach the other rows.
        struct Open { int key, value; uint32_t none; };
        auto look_at = [&](const __nv_bfloat16* rows, int have) {
            uint32_t big = 0, big_v = 0, none = 0;
#pragma unroll 1
            for (int i = lane; i < have * (kDim / 2); i += 32) {
                uint32_t x = reinterpret_cast<const uint32_t*>(rows)[i], y = reinterpret_cast<const uint32_t*>(rows)[i + kKv8Tokens * (kDim / 2)];
                if (drop_not_finite(x) | drop_not_finite(y)) none |= 1u << (i / (kDim / 2));
                big = __vmaxu2(big, x & 0x7fff7fffu);
                big_v = __vmaxu2(big_v, y & 0x7fff7fffu);
            }
            return Open{pow2_exponent(__reduce_max_sync(0xffffffffu, widest_half(big))), pow2_exponent(__reduce_max_sync(0xffffffffu, widest_half(big_v))),
                        __reduce_or_sync(0xffffffffu, none)};
        };
        auto store_k = [&](const Page& pg, int j, int kb, uint32_t base) {
            float k_scale = 0.f, v_scale = 1.f;
            const int page = 2 * w + j;
            auto at = [&](int i, int r) {   // 16 bytes of token g + 8 r
                const int g = kg + 4 * (i & 1), key = page * kKv8Tokens + g + 8 * r;
                return base + (i >> 1) * kHalfBytes + key * 128 + (((4 * kc + t) ^ (key & 7)) << 4);
            };
            if (pg.kind == kClosed) {
                k_scale = sc[j].x; v_scale = sc[j].y;
#pragma unroll
                for (int i = 0; i < kC; ++i) {
                    uint32_t x[8];
                    kv8_widen(kb_[j][i].x, &x[0], &x[1]); kv8_widen(kb_[j][i].y, &x[2], &x[3]);
                    kv8_widen(kb_[j][i].z, &x[4], &x[5]); kv8_widen(kb_[j][i].w, &x[6], &x[7]);
                    st_shared_v4(at(i, 0), x[0], x[1], x[2], x[3]);
                    st_shared_v4(at(i, 1), x[4], x[5], x[6], x[7]);
                }
            } else {
                // the rows of the block that is not complete, or nothing: zeros (once in a sequence: short code rather than fast)
                const int have = pg.kind == kOpen ? length - pg.block * kKv8Tokens : 0;
                const __nv_bfloat16* src = open_rows(pg.block, 0);
                const Open o = look_at(src, have);
                const float factor = pow2(-o.key);
                if (pg.kind == kOpen) { k_scale = pow2(o.key); v_scale = pow2(o.value); }
#pragma unroll 1
                for (int i = 0; i < 2 * kC; ++i) {
                    const int token = kg + 4 * ((i >> 1) & 1) + 8 * (i & 1), d = ((i >> 2) * 2 + kc) * 32 + 8 * t;
                    uint4 x = token < have ? *reinterpret_cast<const uint4*>(src + token * kDim + d) : make_uint4(0, 0, 0, 0);
                    if ((o.none >> token) & 1) x = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
                    st_shared_v4(at(i >> 1, i & 1), bf16x2_to_f16x2(x.x, factor), bf16x2_to_f16x2(x.y, factor), bf16x2_to_f16x2(x.z, factor), bf16x2_to_f16x2(x.w, factor));
                }
            }
            if (lane == 0) {
                float* s = scales[kb % kScaleSlots][page];
                s[0] = k_scale * p.scale_log2;
                s[1] = pg.kind == kNone ? -INFINITY : __log2f(v_scale);   // tokens of a page that is none do not count
                s[2] = k_scale == k_scale ? __fdividef(1.f, v_scale) : k_scale;
            }
        };
        auto store_v = [&](const Page& pg, int j, uint32_t base) {
            const int page = 2 * w + j;
            auto at = [&](int d) {   // four keys of channel d (d % 8 = vg)
                return base + (page >> 2) * kVHalf + d * 128 + (((2 * (page & 3) + (t >> 1)) ^ (d & 7)) << 4) + (t & 1) * 8;
            };
            if (pg.kind == kClosed) {
#pragma unroll
                for (int i = 0; i < kC; ++i) {
                    const uint32_t b[4] = {vb_[j][i].x, vb_[j][i].y, vb_[j][i].z, vb_[j][i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t lo, hi;
                        kv8_widen(b[k], &lo, &hi);
                        st_shared_v2(at(32 * i + 8 * k + vg), lo, hi);
                    }
                }
            } else {
                const int have = pg.kind == kOpen ? length - pg.block * kKv8Tokens : 0;
                const unsigned short* src = reinterpret_cast<const unsigned short*>(open_rows(pg.block, 1));
                const float factor = pow2(-look_at(open_rows(pg.block, 0), have).value);
#pragma unroll 1
                for (int i = 0; i < 4 * kC; ++i) {
                    const int d = 8 * i + vg;
                    uint32_t x[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int token = 2 * t + 8 * r;
                        const uint32_t lo = token < have ? src[token * kDim + d] : 0u, hi = token + 1 < have ? src[(token + 1) * kDim + d] : 0u;
                        uint32_t both = lo | hi << 16;
                        drop_not_finite(both);
                        x[r] = bf16x2_to_f16x2(both, factor);
                    }
                    st_shared_v2(at(d), x[0], x[1]);
                }
            }
        };
        // Round kb stores V of block kb (stage kb & 1) and K of block kb + 1 (the other stage). What lies there, V of block kb - 2 and K of block kb - 1, is read
        // by the products of round kb - 2, whose end `empty` tells; only K of block 0 is read in front of all rounds: `k_read` tells the end of the first
        // scores, before K of block 2 takes its place.
        auto store_keys = [&](const Page (&pg)[2], int kb) {
#pragma unroll
            for (int j = 0; j < 2; ++j) store_k(pg[j], j, kb, sK + (kb & 1) * kKBytes);
        };
        if (n_blocks > 0) {
            if (first_key != asked_first || last_key != asked_last) ask_first();
#pragma unroll
            for (int j = 0; j < 2; ++j) numbers[j] = number(1, j);
            store_keys(pages, 0);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0 && !params.starve) mbar_arrive(&k_first);
        }
        for (int kb = 0; kb < n_blocks; ++kb) {
            const int st = kb & 1;
#pragma unroll
            for (int j = 0; j < 2; ++j) { next[j] = find(kb + 1, j, numbers[j]); numbers[j] = number(kb + 2, j); }
            if (kb + 1 < n_blocks) load_k(next);
            if (kb >= 2 && !wait(&empty[st], (uint32_t)((kb - 2) >> 1) & 1u)) break;
            if (kb == 1 && n_blocks > 2 && !wait(&k_read, 0)) break;
#pragma unroll
            for (int j = 0; j < 2; ++j) { store_v(pages[j], j, sV + st * 2 * kVHalf); pages[j] = next[j]; }
            if (kb + 1 < n_blocks) {
                load_v(pages);
                store_keys(pages, kb + 1);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[st]);
        }
        if (failed && lane == 0) atomicExch(p.status, 3);
    } else if (warp >= kMmaWarp) {
        // ================= warps 12, 13: the products of a tile each, so that neither waits for the other's weights ================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kMmaRegs));
        if (elect_one()) {
            const int i = warp - kMmaWarp, my_blocks = nb_t[i];
            auto wait_one = [&](uint64_t* bar, uint32_t parity) { return !failed && !(failed = !mbar_wait_parked(smem_u32(bar), parity, params.wait_limit)); };
            const uint64_t q_desc = make_smem_desc(sQ + i * kQBytes), k_desc = make_smem_desc(sK), v_desc = make_smem_desc(sV);
            const uint32_t t_s = tmem + (uint32_t)(i * kKeys), t_o = tmem + kOCol + (uint32_t)(i * kDim);
            auto issue_s = [&](int h, int kb) {   // 64 keys
                const uint64_t b_desc = k_desc + (uint64_t)(((kb & 1) * kKBytes + h * (kKeys / 2) * 128) >> 4);
#pragma unroll
                for (int ks = 0; ks < kDim / 16; ++ks) {
                    const uint64_t off = (uint64_t)((ks >> 2) * (kHalfBytes >> 4) + 2 * (ks & 3));
                    umma_f16(t_s + (uint32_t)(h * (kKeys / 2)), q_desc + off, b_desc + off, kIdescS, ks > 0 ? 1u : 0u);
                }
                umma_commit(&s_full[i][h]);
            };
            if (my_blocks > 0 && wait_one(&k_first, 0)) {
                tc_fence_after();
                for (int h = 0; h < 2; ++h) issue_s(h, 0);
                umma_commit(&k_read);
            } else if (!failed) {
                mbar_arrive(&k_read);
            }
            for (int kb = 0; kb < n_blocks && !failed; ++kb) {
                const int st = kb & 1;
                if (!wait_one(&full[st], (uint32_t)(kb >> 1) & 1u)) break;
#pragma unroll 1
                for (int h = 0; h < 2 && kb < my_blocks; ++h) {
                    if (!wait_one(&p_full[i][h], (uint32_t)kb & 1u)) break;
                    tc_fence_after();
                    const uint64_t b_desc = v_desc + (uint64_t)(((2 * st + h) * kVHalf) >> 4);
#pragma unroll
                    for (int ks = 0; ks < kKeys / 32; ++ks)
                        umma_bf16_ts(t_o, t_s + (uint32_t)(h * (kKeys / 2)) + 8u * ks, b_desc + (uint64_t)(2 * ks), kIdescO, (kb > 0 || h > 0 || ks > 0) ? 1u : 0u);
                    if (kb == my_blocks - 1) umma_commit(h ? &o_full[i] : &o_first[i]);
                    if (kb + 1 < my_blocks) issue_s(h, kb + 1);
                }
                if (!failed) umma_commit(&empty[st]);
            }
            if (failed) {   // products in flight read shared and tensor memory: let them end before the CTA does
                umma_commit(&drained[i]);
                mbar_wait_parked(smem_u32(&drained[i]), 0, params.wait_limit);
                atomicExch(p.status, 3);
            }
        }
        __syncwarp();
    } else {
        // ================= warps 0 - 7: a row per thread =========================================================================================
        const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t t_s = t_lane + (uint32_t)ti * kKeys, t_o = t_lane + kOCol + (uint32_t)ti * kDim;
        const int my_blocks = nb_t[ti];
        const uint32_t s_bar = smem_u32(&s_full[ti][0]), p_bar = smem_u32(&p_full[ti][0]), sc0 = smem_u32(&scales[0][0][0]);
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
        // Halves of blocks (64 keys; steps, two of a block) that all rows of this warp see: most. Rows that are nobody's see what the others do.
        const int seen_from = __reduce_max_sync(0xffffffffu, live ? begin : 0) - first_key, seen_to = __reduce_min_sync(0xffffffffu, live ? end : 0x7fffffff) - first_key;
        const int steps = 2 * my_blocks, whole_from = max(1, (seen_from + kKeys / 2 - 1) / (kKeys / 2)), whole_to = min(steps, seen_to / (kKeys / 2));
        float m_run = live ? -3e38f : 0.f, l_run = 0.f;
        int step = 0;
        auto scores_there = [&] {   // of this step; whole warp
            if (!mbar_wait_parked(s_bar + 8u * (step & 1), (uint32_t)(step >> 1) & 1u, params.wait_limit)) failed = true;
            failed = __any_sync(0xffffffffu, failed);
            tc_fence_after();
            return !failed;
        };
#pragma unroll 1   // (the code of a half is long: copies of it do not stay in the instruction cache)
        while (step < steps) {
            uint32_t sc, t_h;   // this step's scales; its scores, later its weights
            auto place = [&] {
                sc = sc0 + (uint32_t)((step >> 1) % kScaleSlots) * (kPages * 16) + (step & 1) * (kPages / 2 * 16);
                t_h = t_s + (uint32_t)(step & 1) * (kKeys / 2);
            };
            uint32_t s[64], weights[32];   // scores of half a block; two weights each
            auto load = [&] {
                tmem_ld_32_async(t_h, s);
                tmem_ld_32_async(t_h + 32u, s + 32);
                tmem_wait_ld();   // straight behind: nothing may touch the registers before
            };
            // Raises the reference of rows whose weights of a half came out too large, to kHeadroom below that half's maximum: what was computed with the old one
            // (output and sum) is scaled down. Rare behind a sequence's first keys.
            auto raise = [&](bool over) {
                const int kb = step >> 1, half = step & 1, key0 = first_key + step * (kKeys / 2);
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 64; ++j) {
                    const float4 x = ld_shared_f4(sc + (j / 16) * 16);
                    const int key = key0 + j;
                    if (over && key >= begin && key < end) top = fmaxf(top, fmaf(__uint_as_float(s[j]), x.x * q_scale, x.y));
                }
                top = fmaxf(m_run, top - kHeadroom);
                const float alpha = kv8_exp2(m_run - top);   // (0 the first time)
                m_run = top;
                l_run *= alpha;
                if (kb == 0 && half == 0) return;
                // The products with V so far have to be complete. Those of this half came before these scores; of the other half, behind its next scores (or the
                // last block's: o_first).
                const bool last = half == 1 && kb + 1 == my_blocks;
                if (!mbar_wait_parked(last ? smem_u32(&o_first[ti]) : s_bar + 8u * (half ^ 1), last ? 0u : (uint32_t)(kb + half) & 1u, params.wait_limit)) failed = true;
                failed = __any_sync(0xffffffffu, failed);
                tc_fence_after();
#pragma unroll 1
                for (int i = 0; i < kDim / 16; ++i) {
                    uint32_t r[16];
                    tmem_ld_16(t_o + 16u * i, r);
#pragma unroll
                    for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
                    tmem_st_16(t_o + 16u * i, r);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
            };
            // Scores of a half -> weights, packed in the order of V's keys, and their share of the sum; returns whether a page's weights add up to more
            // than keeps each an f16 (or to no number). The usual way takes the reference off inside the multiply-add. Scores of 2^27 and more are rounded to steps
            // that are exponents of their own, so where the reference has just been set it is taken off the rounded score, whose maximum it is.
            auto weigh = [&](auto all_seen, float& share) {
                constexpr bool kWhole = decltype(all_seen)::value;
                const int key0 = first_key + step * (kKeys / 2);
                bool fits = true;
                share = 0.f;
#pragma unroll
                for (int pg = 0; pg < 4; ++pg) {
                    const float4 x = ld_shared_f4(sc + pg * 16);
                    const float cq = x.x * q_scale, b = kWhole ? x.y - m_run : x.y;
                    const uint64_t c2 = pair_of(cq, cq), b2 = pair_of(b, b), m2 = pair_of(-m_run, -m_run);
                    uint64_t part = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {   // keys 2 i, 2 i + 1
                        const uint64_t t2 = fma2(pair_of(__uint_as_float(s[16 * pg + 2 * i]), __uint_as_float(s[16 * pg + 2 * i + 1])), c2, b2);
                        const float2 t = split(kWhole ? t2 : add2(t2, m2));
                        float2 w = make_float2(kv8_exp2(t.x), kv8_exp2(t.y));
                        if (!kWhole) {
                            const int key = key0 + 16 * pg + 2 * i;
                            w.x = key >= begin && key < end ? w.x : 0.f;
                            w.y = key + 1 >= begin && key + 1 < end ? w.y : 0.f;
                        }
                        part = add2(part, pair_of(w.x, w.y));
                        weights[8 * pg + (i < 4 ? 2 * i : 2 * (i - 4) + 1)] = pack_f16x2(w.x, w.y);
                    }
                    const float2 both = split(part);
                    const float page_sum = both.x + both.y;
                    // 1 / s_V that is not a number belongs to a page that is none: of rows that see all of it. Others find that in their weights.
                    share = fmaf(page_sum, kWhole || x.z == x.z ? x.z : 1.f, share);
                    fits &= page_sum <= kLargestSum;
                }
                return !fits && live;
            };
            float share;
            auto hand_over = [&] {
                l_run += share;
                tmem_st_32(t_h, weights);
                asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                tc_fence_before();
                mbar_arrive_addr(p_bar + 8u * (step & 1));
                ++step;
            };
            bool over = true, raises = step == 0;   // the first scores of all have their maximum taken first; others only where the weights turn out too large
#pragma unroll 1
            while (step >= whole_from && step < whole_to) {   // the usual way, apart from the other one so that their registers need not meet
                if (!scores_there()) break;
                place();
                load();
                over = weigh(std::true_type{}, share);
                if (__any_sync(0xffffffffu, over)) { raises = true; break; }
                hand_over();
            }
            if (failed || step == steps || !scores_there()) break;
            place();
#pragma unroll 1
            for (int pass = 0; pass < 2; ++pass) {
                load();   // the weights have not been stored over the scores yet
                if (raises) raise(over);
                over = weigh(std::false_type{}, share);
                if (!__any_sync(0xffffffffu, over)) break;   // (behind a raise: of rows that fitted in the usual way, or that are none)
                raises = true;
            }
            hand_over();
        }
        // ---- the output, or this split's part of it --------------------------------------------------------------------------------------------
        if (my_blocks > 0 && !failed) {
            if (!mbar_wait_parked(smem_u32(&o_full[ti]), 0, params.wait_limit)) failed = true;
            failed = __any_sync(0xffffffffu, failed);
        }
        // a query that is not a number, or scores that are infinite: the row is none
        if (end > begin && my_blocks > 0 && (q_scale != q_scale || m_run == INFINITY)) l_run = __uint_as_float(0x7fc00000u);
        const long long at = (long long)my_row * p.q_heads + my_head;
        if (!failed && p.splits == 1) {
            tc_fence_after();
            const float inv = l_run == 0.f ? 0.f : __fdividef(1.f, l_run);
            uint4* dst = reinterpret_cast<uint4*>(p.out + at * kDim);
#pragma unroll 1
            for (int c = 0; c < kDim / 32; ++c) {
                float o[32];
                if (my_blocks > 0) {
                    tmem_ld_32(t_o + 32u * c, o);
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0.f;
                }
                if (live) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        dst[4 * c + i] = make_uint4(pack_bf16x2(o[8 * i] * inv, o[8 * i + 1] * inv), pack_bf16x2(o[8 * i + 2] * inv, o[8 * i + 3] * inv),
                                                    pack_bf16x2(o[8 * i + 4] * inv, o[8 * i + 5] * inv), pack_bf16x2(o[8 * i + 6] * inv, o[8 * i + 7] * inv));
                }
            }
        } else if (!failed) {
            tc_fence_after();
            const long long part = at * p.splits + blockIdx.z;
            const bool seen = my_blocks > 0 && (l_run != 0.f);
            if (live) { p.part_ml[2 * part] = seen ? m_run : -INFINITY; p.part_ml[2 * part + 1] = seen ? l_run : 0.f; }
            if (my_blocks > 0) {
                float4* dst = reinterpret_cast<float4*>(p.part_o + part * kDim);
#pragma unroll 1
                for (int c = 0; c < kDim / 32; ++c) {
                    float o[32];
                    tmem_ld_32(t_o + 32u * c, o);
                    if (live) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) dst[8 * c + i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
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

template <int kDim>
int launch_prompt(const PromptParams& p, cudaStream_t stream) {
    // a kernel compiled for fewer registers than its groups ask for would wait for them without end
    static const int regs = [] {
        cudaFuncAttributes attr;
        return cudaFuncGetAttributes(&attr, kv8_prompt_kernel<kDim>) == cudaSuccess ? attr.numRegs : 0;
    }();
    if (regs != kLaunchRegs) return fail(GPTRS_EXECUTION, "kv8_prompt_kernel has " + std::to_string(regs) + " registers a thread, not those that its warps share out");
    static PerDeviceOnce attr_once;
    if (attr_once.first_time())
        GPTRS_CUDA_OK(cudaFuncSetAttribute(kv8_prompt_kernel<kDim>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)prompt_smem<kDim>()));
    return launch_kernel(kv8_prompt_kernel<kDim>, dim3((unsigned)p.a.kv_heads, (unsigned)p.a.n_tiles, (unsigned)p.a.splits), dim3(kThreads), prompt_smem<kDim>(), stream, 1, p);
}

}  // namespace

int kv8_prompt_attention(const Kv8Attention& a, int dim, cudaStream_t stream) {
    PromptParams p = {};
    p.a = a;
    prefill_tc_fault(&p.starve, &p.wait_limit);
    return dim == 64 ? launch_prompt<64>(p, stream) : launch_prompt<128>(p, stream);
}

}  // namespace gptrs
