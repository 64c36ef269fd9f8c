// Attention of trees of drafted tokens over the paged bf16 cache: node i of a tree sees the sequence's tokens, its ancestors and itself.
//
// A warp per node and query head walks over what the node sees, four channels a lane, with the running maximum and sum of the softmax.
#include "draft_tree.cuh"

namespace gptrs {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 8;

struct AttentionParams {
    DraftTrees t;
    const __nv_bfloat16* q;
    long long ldq;
    const unsigned char* pool;
    __nv_bfloat16* out;
    int* status;
    float scale_log2;
};

__global__ void __launch_bounds__(kWarps * 32) tree_attention_kernel(const AttentionParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int node = blockIdx.x, head = blockIdx.z * kWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const TreeSpan s = tree_span(p.t, blockIdx.y, p.status);
    if (node >= s.nodes || head >= p.t.q_heads) return;
    const long long row = s.row0 + node;
    const uint2 qw = *reinterpret_cast<const uint2*>(p.q + row * p.ldq + head * kTreeDim + 4 * lane);
    const float q[4] = {bf16_lo(qw.x) * p.scale_log2, bf16_hi(qw.x) * p.scale_log2, bf16_lo(qw.y) * p.scale_log2, bf16_hi(qw.y) * p.scale_log2};
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    bool any = false;
    auto see = [&](int position) {
        const long long place = tree_place(p.t, s.slot, position, p.status);
        if (place < 0) return;
        any = true;
        const unsigned char* at = p.pool + place + 2 * (head / p.t.group) * kTreeBlock + (((lane >> 1) ^ (position & 7)) << 4) + 8 * (lane & 1);
        const uint2 k = *reinterpret_cast<const uint2*>(at), v = *reinterpret_cast<const uint2*>(at + kTreeBlock);
        const float z = warp_sum(q[0] * bf16_lo(k.x) + q[1] * bf16_hi(k.x) + q[2] * bf16_lo(k.y) + q[3] * bf16_hi(k.y));
        const float to = fmaxf(m, z), keep = m == to ? 1.f : exp2f(m - to), w = exp2f(z - to);
        m = to;
        l = l * keep + w;
        o[0] = o[0] * keep + w * bf16_lo(v.x); o[1] = o[1] * keep + w * bf16_hi(v.x);
        o[2] = o[2] * keep + w * bf16_lo(v.y); o[3] = o[3] * keep + w * bf16_hi(v.y);
    };
    for (int i = 0; i < s.length; ++i) see(i);
    for (int i = node; i >= 0; i = tree_parent(p.t, s, i, p.status)) see(s.length + i);
    const float inv = any ? 1.f / l : 0.f;
    *reinterpret_cast<uint2*>(p.out + (row * p.t.q_heads + head) * kTreeDim + 4 * lane) = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace gptrs

using namespace gptrs;

extern "C" {

size_t gptrs_cuda_tree_scratch_bytes(const gptrs_draft_trees* t) { return 0; }

int gptrs_cuda_tree_attention(const gptrs_draft_trees* t, const gptrs_tree_attention_step* s, void* stream) {
    AttentionParams p = {};
    const int rc = draft_trees(t, &p.t);
    if (rc) return rc;
    GPTRS_REQUIRE(s && s->d_pool && s->d_status && (t->rows == 0 || (s->d_q && s->d_out)), "null pointer");
    GPTRS_REQUIRE(aligned16(s->d_q) && aligned16(s->d_pool) && aligned16(s->d_out) && aligned16(s->d_scratch), "pointers must be 16-byte aligned");
    const int64_t width = (int64_t)t->q_heads * kTreeDim;
    p.ldq = s->ldq ? s->ldq : width;
    GPTRS_REQUIRE(p.ldq >= width && p.ldq % 8 == 0 && p.ldq < ((int64_t)1 << 31), "rows of queries overlap, or do not start at multiples of 16 bytes");
    const size_t scratch = gptrs_cuda_tree_scratch_bytes(t);
    GPTRS_REQUIRE(scratch == 0 || (s->d_scratch && s->scratch_bytes >= scratch), "scratch is too small");
    if (t->rows == 0) return GPTRS_OK;
    const char *q = static_cast<const char*>(s->d_q), *out = static_cast<const char*>(s->d_out);
    GPTRS_REQUIRE(out >= q + 2 * ((t->rows - 1) * p.ldq + width) || q >= out + 2 * t->rows * width, "the output lies in rows of queries");
    p.q = static_cast<const __nv_bfloat16*>(s->d_q);
    p.pool = static_cast<const unsigned char*>(s->d_pool);
    p.out = static_cast<__nv_bfloat16*>(s->d_out);
    p.status = s->d_status;
    p.scale_log2 = (t->scale != 0.f ? t->scale : 1.f / sqrtf((float)kTreeDim)) * kLog2e;
    return launch_kernel(tree_attention_kernel, dim3((unsigned)t->max_nodes, (unsigned)t->n_trees, (unsigned)ceil_div(t->q_heads, kWarps)), dim3(kWarps * 32), 0, as_stream(stream), 1, p);
}

}  // extern "C"
