// Attention of chunks of new tokens over the compressed cache: causal, over
// everything or over a sliding window and the first tokens of the sequence
// (sinks).
//
// The new token at position p attends position t where t <= p and, under a
// window of w, t > p - w or t < sinks.
#include "chunk_tiles.cuh"

namespace ins {
namespace {

// How a call is cut: the walks of its sequences, for the kernels of attend.cuh
// (few) or, `tiles`, for k_chunk_tiles.
struct ChunkPlan {
    AttendPlan<ChunkView> few;
    std::vector<ChunkSeq> seqs;
    bool tiles = false;
    int64_t units = 0, row_tiles = 0, walk_tiles = 0;
    int splits = 1;                          // the most pieces of a row tile
    int64_t image_bytes(const Geo &g) const { return (row_tiles + walk_tiles) * g.n_kv * 2 * TL_IMAGE; }
    int64_t bytes(const Geo &g) const {
        if (!tiles) return (int64_t)few.acc_bytes();
        return 256 + image_bytes(g) + (splits > 1 ? units * TL_ROWS * (64 + 2) * (int64_t)sizeof(float) : 0);
    }
};

// Positions, and ends of tiles beyond them, stay well inside 32 bits.
constexpr int32_t MAX_LENGTH = 1 << 30;

// Row tiles, units and pieces of k_chunk_tiles. Units are whole row tiles unless
// that leaves SMs idle: a row tile's KV tiles are then cut so that the units
// fill rounds of one an SM evenly. Counted in KV tiles' times (1.26 us measured):
// what a unit costs besides its tiles (4.5), and the join of pieces (1,024 units:
// 44 us). False: the images would take too much.
constexpr int64_t TILES_MOST = (int64_t)8 << 30;
constexpr double UNIT_TILES = 4.5, JOIN_TILES = 0.034;
bool cut_tiles(const Geo &g, const ChunkView &v, int sms, ChunkPlan &p) {
    std::sort(p.seqs.begin(), p.seqs.end(), [](const ChunkSeq &a, const ChunkSeq &b) {
        return a.context + a.nodes != b.context + b.nodes ? a.context + a.nodes > b.context + b.nodes : a.node0 < b.node0;
    });
    const int per = TL_ROWS / g.H;
    std::vector<int64_t> most(p.seqs.size());
    int64_t longest = 0;
    double work = 0;
    for (size_t i = 0; i < p.seqs.size(); ++i) {
        ChunkSeq &s = p.seqs[i];
        s.rts = (s.nodes + per - 1) / per;
        s.group0 = (int32_t)p.row_tiles;
        s.tile0 = (int32_t)p.walk_tiles;
        p.row_tiles += s.rts;
        p.walk_tiles += (v.span(s) + TL_TILE - 1) / TL_TILE;
        const int64_t first = row_tile(v, s, g.H, 0).tiles, last = row_tile(v, s, g.H, s.rts - 1).tiles;
        most[i] = std::max(first, last);
        longest = std::max(longest, most[i]);
        work += 0.5 * (double)(first + last) * s.rts * g.n_kv;
    }
    if (p.image_bytes(g) > TILES_MOST) return false;
    double best = 0;
    int64_t piece = longest;
    for (int k = 1; k <= 64; ++k) {
        const int64_t size = (longest + k - 1) / k;
        if (k > 1 && size < 4) break;
        double n = 0;
        for (size_t i = 0; i < p.seqs.size(); ++i)
            n += (double)p.seqs[i].rts * g.n_kv * (double)((most[i] + size - 1) / size);
        const double rounds = std::ceil(n / sms), each = work / n + UNIT_TILES;
        const double time = std::max(rounds * each, size + UNIT_TILES) + (k > 1 ? n * JOIN_TILES : 0.0);
        if (k == 1 || time < 0.97 * best) best = time, piece = size;
    }
    for (size_t i = 0; i < p.seqs.size(); ++i) {
        ChunkSeq &s = p.seqs[i];
        s.splits = (int32_t)((most[i] + piece - 1) / piece);
        s.unit0 = (int32_t)p.units;
        p.units += (int64_t)s.rts * g.n_kv * s.splits;
        p.splits = std::max(p.splits, (int)s.splits);
    }
    return p.units <= INT32_MAX;
}

// k_chunk_tiles takes over where a KV head has more than TILES_FROM query rows in
// some sequence: 8 KV heads of 4 query heads, k_attend_many (or few) against it, of
// 32,768 tokens and of 16 x 8,192: 64 tokens 53 : 60 us and 139 : 164, 96 tokens
// 71 : 76 and 227 : 241, 128 tokens 77 : 77 and 247 : 248, 160 tokens 97 : 92 and
// 345 : 318, 256 tokens 123 : 118 and 479 : 410. Not where its images would take
// more than TILES_MOST bytes, nor in formats whose scores need a factor above 2^5
// (k_attend_few takes those, at any number of rows).
constexpr int64_t TILES_FROM = 512;

int make_plan(const CacheBase *c, int32_t B, const int32_t *seq, const int32_t *counts, int sms, const ChunkView &v,
              ChunkPlan &p) {
    const Geo &g = c->g;
    int64_t all = 0, most = 0;
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
        most = std::max<int64_t>(most, (int64_t)counts[b] * g.H);
    }
    if (all > INT32_MAX / (g.n_kv * g.H)) return fail(INS_EBADLEN, "too many tokens in one call");
    if (p.seqs.empty()) return INS_OK;
    p.few.seqs = p.seqs;
    if (most > TILES_FROM && score_shift(g) <= MANY_SHIFT) {
        p.tiles = cut_tiles(g, v, sms, p);
        if (p.tiles) return INS_OK;
    }
    return cut_plan(g, v, sms, p.few);
}

template <int KB, int VB>
int launch_expand(CacheBase *c, const ChunkPlan &p, const Plan &plan, const TilesArgs &a, const ChunkView &v,
                  cudaStream_t s) {
    return plan.run(c, s, [&](const auto &src) -> cudaError_t {
        *c->launches += 1;
        return launch_after(k_chunk_expand<KB, VB, std::decay_t<decltype(src)>>,
                            (unsigned)((p.walk_tiles + p.row_tiles) * c->g.n_kv), 256u, 0, s, c->g, a, v, src);
    });
}

int run_tiles(CacheBase *c, const ChunkPlan &p, const ChunkView &v, const int32_t *q, void *out, void *workspace,
              int sms, cudaStream_t s) {
    const Geo &g = c->g;
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    TilesArgs a{};
    a.tb = c->d_tables;
    a.pool = c->d_pool;
    a.table = c->d_page_table;
    a.q = q;
    a.out = static_cast<__nv_bfloat16 *>(out);
    a.ticket = reinterpret_cast<int32_t *>(ws);
    a.q_images = ws + 256;
    a.kv_images = a.q_images + p.row_tiles * g.n_kv * 2 * TL_IMAGE;
    a.acc = reinterpret_cast<float *>(a.kv_images + p.walk_tiles * g.n_kv * 2 * TL_IMAGE);
    a.ml = a.acc + p.units * TL_ROWS * 64;
    a.status = c->d_status;
    a.n_seqs = (int32_t)p.seqs.size();
    a.units = (int32_t)p.units;
    a.kv_ctas = (int32_t)(p.walk_tiles * g.n_kv);
    a.poll_limit = std::min(c->wait.poll_limit, WAIT_POLLS);
    a.hold_cta = c->wait.item;
    a.hold_tile = c->wait.chunk;
    const float unit = std::ldexp(1.0f, score_shift(g));
    a.q_scale = std::min(unit, 1.0f);
    a.k_scale = std::max(unit, 1.0f);
    a.out_unit = std::ldexp(1.0f, 9 - g.norm_frac);
    Plan plan;
    plan.add(p.seqs);
    const int rc = g.kb == 4 && g.vb == 2   ? launch_expand<4, 2>(c, p, plan, a, v, s)
                   : g.kb == 3 && g.vb == 3 ? launch_expand<3, 3>(c, p, plan, a, v, s)
                                            : launch_expand<0, 0>(c, p, plan, a, v, s);
    if (rc) return rc;
    if (int rc2 = plan.run(c, s, [&](const auto &src) -> cudaError_t {
            auto fn = k_chunk_tiles<std::decay_t<decltype(src)>>;
            const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, TL_SMEM);
            if (e != cudaSuccess) return e;
            *c->launches += 1;
            return launch_after(fn, (unsigned)std::min<int64_t>(sms, p.units), (unsigned)TL_THREADS, (size_t)TL_SMEM, s, g,
                                a, v, src);
        }))
        return rc2;
    if (p.splits == 1) return INS_OK;
    const size_t smem = (size_t)8 * p.splits * sizeof(float);
    return plan.run(c, s, [&](const auto &src) -> cudaError_t {
        *c->launches += 1;
        return launch_after(k_chunk_join<std::decay_t<decltype(src)>>,
                            (unsigned)(p.row_tiles * g.n_kv * (TL_ROWS / 8)), 128u, smem, s, g, a, v, src);
    });
}

int chunk_body(CacheBase *c, int32_t B, const int32_t *seq, const int32_t *counts, int32_t window, int32_t sinks,
               const int32_t *q, void *out, void *workspace, int64_t workspace_bytes, int64_t *need, cudaStream_t s) {
    if (window < 0 || sinks < 0) return fail(INS_EINVAL, "chunk scan: a negative window or number of sinks");
    int sms = 0;
    if (int rc = device_sms(c->device, &sms)) return rc;
    const ChunkView v{window ? std::min(window, MAX_LENGTH) : MAX_LENGTH, window ? std::min(sinks, MAX_LENGTH) : 0};
    ChunkPlan p;
    if (int rc = make_plan(c, B, seq, counts, sms, v, p)) return rc;
    const int64_t bytes = p.bytes(c->g);
    if (need) {
        *need = bytes;
        return INS_OK;
    }
    if (p.seqs.empty()) return INS_OK;
    if (int rc = check_formats(c, "chunk scan")) return rc;
    if (!q || !out) return fail(INS_EINVAL, "chunk scan: NULL buffer");
    if (((uintptr_t)q & 15u) || ((uintptr_t)out & 15u))
        return fail(INS_EINVAL, "chunk scan: q and out 16-byte aligned");
    if (bytes > workspace_bytes || (bytes && (!workspace || ((uintptr_t)workspace & 127u))))
        return fail(INS_EINVAL, "chunk scan: a 128-byte aligned workspace of " + std::to_string(bytes) + " bytes is needed");
    if (p.tiles) return run_tiles(c, p, v, q, out, workspace, sms, s);
    AttendArgs a = attend_args(c, p.few, q, out, workspace);
    a.k_unit = c->k_unit;
    a.v_unit = c->v_unit;
    a.score_unit /= a.k_unit;
    a.k_scale /= a.k_unit;
    a.out_unit /= a.v_unit;
    return run_plan(c, p.few, a, v, s);
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
