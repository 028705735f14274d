// Attention of drafted trees over the compressed cache: the kernels of
// attend.cuh over a sequence's whole context and the drafted tokens that a
// node's mask names (its ancestors and itself).
#include "attend.cuh"

namespace ins {

constexpr int TREE_MAX_NODES = 256;          // drafted tokens of one sequence

// 32 visibility bits of node `mk` from drafted offset d on (d < 0: context).
__device__ __forceinline__ uint32_t seen32(const uint64_t *mk, int nodes, int d) {
    auto word = [&](int at) -> uint64_t { return at * 64 < nodes ? mk[at] : 0ull; };
    uint32_t bits;
    if (d <= -32) return 0xffffffffu;
    if (d < 0) bits = (uint32_t)(word(0) << -d) | ((1u << -d) - 1u);
    else {
        const int sh = d & 63;
        bits = (uint32_t)(word(d >> 6) >> sh);
        if (sh > 32) bits |= (uint32_t)(word((d >> 6) + 1) << (64 - sh));
    }
    const int live = nodes - d;                      // bits at and beyond the tree's end are no tokens
    return live >= 32 ? bits : live <= 0 ? 0u : bits & ((1u << live) - 1u);
}

struct TreeView {
    using Seq = AttendSeq;
    static constexpr bool SHARES = false;
    const uint64_t *mask;
    int32_t words;
    struct Row {
        const uint64_t *mk;
        int32_t nodes, context;
        __device__ __forceinline__ bool sees(int p) const {
            const int d = p - context;
            return d < 0 || ((mk[d >> 6] >> (d & 63)) & 1);
        }
        __device__ __forceinline__ uint32_t bits(int p) const { return seen32(mk, nodes, p - context); }
    };
    __host__ __device__ __forceinline__ int span(const Seq &s) const { return s.context + s.nodes; }
    __device__ __forceinline__ int at(const Seq &, int i) const { return i; }
    __device__ __forceinline__ Row row(const Seq &s, int node) const {
        return Row{mask + (int64_t)(s.node0 + node) * words, s.nodes, s.context};
    }
    __device__ __forceinline__ bool whole(const Seq &s, int p, int n) const { return p + n <= s.context; }
};

namespace {

using TreePlan = AttendPlan<TreeView>;

int make_plan(const CacheBase *c, int32_t B, const int32_t *seq, const int32_t *nodes, int sms, const TreeView &v,
              TreePlan &p) {
    const Geo &g = c->g;
    int64_t all = 0;
    p.seqs.reserve((size_t)B);
    for (int32_t b = 0; b < B; ++b) {
        if (seq[b] < 0 || seq[b] >= c->cfg.max_seqs)
            return fail(INS_EINVAL, "sequence id " + std::to_string(seq[b]) + " out of range");
        const int64_t len = c->h_seq_lens[seq[b]];
        if (nodes[b] < 0 || nodes[b] > TREE_MAX_NODES)
            return fail(INS_EINVAL, "a tree holds 0 to " + std::to_string(TREE_MAX_NODES) + " nodes, not " +
                                        std::to_string(nodes[b]));
        if (nodes[b] > len)
            return fail(INS_EBADLEN, "sequence " + std::to_string(seq[b]) + " holds " + std::to_string(len) +
                                         " tokens, fewer than its tree's " + std::to_string(nodes[b]));
        if (nodes[b])
            p.seqs.push_back(AttendSeq{seq[b], (int32_t)(len - nodes[b]), nodes[b], (int32_t)all, 1, 0, 0});
        all += nodes[b];
    }
    if (all > INT32_MAX / (g.n_kv * g.H)) return fail(INS_EBADLEN, "too many nodes in one call");
    return cut_plan(g, v, sms, p);
}

int tree_body(CacheBase *c, int32_t B, const int32_t *seq, const int32_t *nodes, const uint64_t *mask, int32_t words,
              const int32_t *q, void *out, void *workspace, int64_t workspace_bytes, int64_t *need, cudaStream_t s) {
    int sms = 0;
    if (int rc = device_sms(c->device, &sms)) return rc;
    const TreeView v{mask, words};
    TreePlan p;
    if (int rc = make_plan(c, B, seq, nodes, sms, v, p)) return rc;
    if (need) {
        *need = (int64_t)p.acc_bytes();
        return INS_OK;
    }
    if (p.seqs.empty()) return INS_OK;
    if (int rc = check_formats(c, "tree scan")) return rc;
    for (const AttendSeq &t : p.seqs)
        if (t.nodes > 64 * words) return fail(INS_EINVAL, "the mask's words are too few for a tree's nodes");
    if (!mask || !q || !out) return fail(INS_EINVAL, "tree scan: NULL buffer");
    if (((uintptr_t)mask & 7u) || ((uintptr_t)q & 15u) || ((uintptr_t)out & 15u))
        return fail(INS_EINVAL, "tree scan: mask 8-byte, q and out 16-byte aligned");
    if ((int64_t)p.acc_bytes() > workspace_bytes || (p.acc_bytes() && (!workspace || ((uintptr_t)workspace & 15u))))
        return fail(INS_EINVAL, "tree scan: a 16-byte aligned workspace of " + std::to_string(p.acc_bytes()) +
                                    " bytes is needed");
    return run_plan(c, p, attend_args(c, p, q, out, workspace), v, s);
}

}  // namespace
}  // namespace ins

using namespace ins;

extern "C" {

int64_t ins_tree_workspace(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int32_t *nodes) {
    if (!cache || B < 0 || (B > 0 && (!seq_ids || !nodes))) return fail(INS_EINVAL, "tree scan arguments"), -1;
    int64_t need = 0;
    CacheBase *c = cache_base(cache);
    const int rc = guarded([&] {
        return tree_body(c, B, seq_ids, nodes, nullptr, 0, nullptr, nullptr, nullptr, 0, &need, nullptr);
    });
    return rc ? -1 : need;
}

int ins_tree_scan(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int32_t *nodes, const uint64_t *mask,
                  int32_t words, const int32_t *q_rot, void *out, void *workspace, int64_t workspace_bytes,
                  void *stream) {
    if (!cache) return fail(INS_EINVAL, "cache is NULL");
    if (B < 0 || (B > 0 && (!seq_ids || !nodes))) return fail(INS_EINVAL, "tree scan arguments");
    if (B == 0) return INS_OK;
    CacheBase *c = cache_base(cache);
    return guarded([&] {
        DeviceGuard dg(c->device);
        return tree_body(c, B, seq_ids, nodes, mask, words, q_rot, out, workspace, workspace_bytes, nullptr,
                         (cudaStream_t)stream);
    });
}

}  // extern "C"
