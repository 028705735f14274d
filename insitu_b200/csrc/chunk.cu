// Attention of chunks of new tokens over the compressed cache: causal, over
// everything or over a sliding window and the first tokens of the sequence
// (sinks).
//
// The new token at position p attends position t where t <= p and, under a
// window of w, t > p - w or t < sinks.
#include "attend.cuh"

namespace ins {

// A sequence's walk: its first `early` tokens (those that hold the sinks), then
// the tokens from position early + skip on (those that its first new token's
// window reaches). Both are multiples of 128 tokens, so that a tile of either
// is a run of positions.
struct ChunkSeq : AttendSeq {
    int32_t early, skip;
};

struct ChunkView {
    using Seq = ChunkSeq;
    int32_t window, sinks;                   // no window: one larger than any position
    struct Row {
        int32_t p, from, sinks;              // sees `from` to p, and what is below sinks
        __device__ __forceinline__ bool sees(int t) const { return t <= p && (t >= from || t < sinks); }
        __device__ __forceinline__ uint32_t bits(int t) const {
            auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? FULL : (1u << n) - 1u; };
            return below(p + 1 - t) & (~below(from - t) | below(sinks - t));
        }
    };
    __host__ __device__ __forceinline__ int span(const Seq &s) const { return s.context + s.nodes - s.skip; }
    __device__ __forceinline__ int at(const Seq &s, int i) const { return i < s.early ? i : i + s.skip; }
    __device__ __forceinline__ Row row(const Seq &s, int node) const {
        return Row{s.context + node, s.context + node + 1 - window, sinks};
    }
    __device__ __forceinline__ bool whole(const Seq &s, int t, int n) const {
        return t + n - 1 <= s.context && (t >= s.context + s.nodes - window || t + n <= sinks);
    }
};

namespace {

using ChunkPlan = AttendPlan<ChunkView>;

// Walks are cut at multiples of this.
constexpr int WALK = 128;
// Positions, and ends of tiles beyond them, stay well inside 32 bits.
constexpr int32_t MAX_LENGTH = 1 << 30;
static_assert(WALK % FEW_TILE == 0 && WALK % MANY_TILE == 0, "a tile of a walk is a run of positions");

ChunkSeq walk_of(const ChunkView &v, int32_t seq, int64_t len, int32_t n, int64_t node0) {
    ChunkSeq s{};
    s.seq = seq;
    s.context = (int32_t)(len - n);
    s.nodes = n;
    s.node0 = (int32_t)node0;
    s.splits = 1;
    const int32_t first = std::max(0, s.context + 1 - v.window) / WALK * WALK;
    const int32_t early = (int32_t)(((int64_t)std::min(v.sinks, s.context + n) + WALK - 1) / WALK * WALK);
    if (first > early) s.early = early, s.skip = first - early;
    return s;
}

int make_plan(const CacheBase *c, int32_t B, const int32_t *seq, const int32_t *counts, int sms, const ChunkView &v,
              ChunkPlan &p) {
    const Geo &g = c->g;
    int64_t all = 0;
    p.seqs.reserve((size_t)B);
    for (int32_t b = 0; b < B; ++b) {
        if (seq[b] < 0 || seq[b] >= c->cfg.max_seqs)
            return fail(INS_EINVAL, "sequence id " + std::to_string(seq[b]) + " out of range");
        const int64_t len = c->h_seq_lens[seq[b]];
        if (counts[b] < 0 || counts[b] > len)
            return fail(INS_EBADLEN, "sequence " + std::to_string(seq[b]) + " holds " + std::to_string(len) +
                                         " tokens; its chunk cannot be " + std::to_string(counts[b]));
        if (counts[b] && len > MAX_LENGTH)
            return fail(INS_EBADLEN, "chunk scan: sequences of up to 2^30 tokens are supported");
        if (counts[b]) p.seqs.push_back(walk_of(v, seq[b], len, counts[b], all));
        all += counts[b];
    }
    if (all > INT32_MAX / (g.n_kv * g.H)) return fail(INS_EBADLEN, "too many tokens in one call");
    return cut_plan(g, v, sms, p);
}

int chunk_body(CacheBase *c, int32_t B, const int32_t *seq, const int32_t *counts, int32_t window, int32_t sinks,
               const int32_t *q, void *out, void *workspace, int64_t workspace_bytes, int64_t *need, cudaStream_t s) {
    if (window < 0 || sinks < 0) return fail(INS_EINVAL, "chunk scan: a negative window or number of sinks");
    int sms = 0;
    if (int rc = device_sms(c->device, &sms)) return rc;
    const ChunkView v{window ? std::min(window, MAX_LENGTH) : MAX_LENGTH, window ? std::min(sinks, MAX_LENGTH) : 0};
    ChunkPlan p;
    if (int rc = make_plan(c, B, seq, counts, sms, v, p)) return rc;
    if (need) {
        *need = (int64_t)p.acc_bytes();
        return INS_OK;
    }
    if (p.seqs.empty()) return INS_OK;
    if (int rc = check_formats(c, "chunk scan")) return rc;
    if (!q || !out) return fail(INS_EINVAL, "chunk scan: NULL buffer");
    if (((uintptr_t)q & 15u) || ((uintptr_t)out & 15u))
        return fail(INS_EINVAL, "chunk scan: q and out 16-byte aligned");
    if ((int64_t)p.acc_bytes() > workspace_bytes || (p.acc_bytes() && (!workspace || ((uintptr_t)workspace & 15u))))
        return fail(INS_EINVAL, "chunk scan: a 16-byte aligned workspace of " + std::to_string(p.acc_bytes()) +
                                    " bytes is needed");
    return run_plan(c, p, attend_args(c, p, q, out, workspace), v, s);
}

}  // namespace
}  // namespace ins

using namespace ins;

extern "C" {

int64_t ins_chunk_workspace(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int32_t *counts, int32_t window,
                            int32_t sinks) {
    if (!cache || B < 0 || (B > 0 && (!seq_ids || !counts))) return fail(INS_EINVAL, "chunk scan arguments"), -1;
    int64_t need = 0;
    CacheBase *c = cache_base(cache);
    const int rc = guarded([&] {
        return chunk_body(c, B, seq_ids, counts, window, sinks, nullptr, nullptr, nullptr, 0, &need, nullptr);
    });
    return rc ? -1 : need;
}

int ins_chunk_scan(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int32_t *counts, int32_t window,
                   int32_t sinks, const int32_t *q_rot, void *out, void *workspace, int64_t workspace_bytes,
                   void *stream) {
    if (!cache) return fail(INS_EINVAL, "cache is NULL");
    if (B < 0 || (B > 0 && (!seq_ids || !counts))) return fail(INS_EINVAL, "chunk scan arguments");
    if (B == 0) return INS_OK;
    CacheBase *c = cache_base(cache);
    return guarded([&] {
        DeviceGuard dg(c->device);
        return chunk_body(c, B, seq_ids, counts, window, sinks, q_rot, out, workspace, workspace_bytes, nullptr,
                          (cudaStream_t)stream);
    });
}

}  // extern "C"
