// Chunks of many query rows: the cache's tiles expanded once, then a flash
// attention on the tensor cores.
//
// A chunk of n tokens has n x groups query rows a KV head. In row tiles of 256,
// each cached tile would be decoded by every row tile; from a few row tiles on
// it costs less to expand the rows that the call walks once, into fp16 tiles
// of 128 tokens in a workspace (k_chunk_expand: 52 bytes read, 256 written a row
// and head), laid out as shared memory holds them, so that k_chunk_tiles fetches
// a tile's keys and values by one bulk copy. The queries are converted there too.
//
// k_chunk_tiles: one CTA an SM, persistent, takes units (a row tile of a KV
// head, or a piece of its KV tiles) from a ticket in order of falling size. One
// warp loads, two groups of eight warps (a stream each: 128 rows, two threads a
// row) turn S = Q K^T into P, one warp issues the products S and one a stream O +=
// P V. P replaces S in tensor memory, so that there is room for three score buffers
// of 128 columns next to two outputs of 64: while both streams work on a buffer
// each, the third already holds the scores of the one that finishes first.
//
// 2,048 tokens on each of 4 sequences of 34,816 in all (8 KV heads of 4 query
// heads, 2.27 TFLOP) take 2.69 ms, 0.84 PFLOP/s, in a run long enough for the power
// cap, 2.35 ms, 0.97 PFLOP/s, in a short one (as the steps below). Bound by the exponentials and what surrounds them: of 2,200 clocks
// a KV tile the special function unit works 70 %, the issue slots 61 %, the tensor
// pipe 47 %. The steps there: one thread a row and one warp that issued all
// products 2,814 us, as that warp's waits and issues (some 200 clocks each) followed
// one another; two threads a row then 2,999, with a warp for the score products and
// one a stream for the value products 2,565. Steps of 64 columns with three score
// buffers a stream: 3,332 to 4,453, each step's fixed 700 clocks counting twice.
#pragma once

#include "attend.cuh"

namespace ins {

// A sequence's walk: its first `early` tokens (those that hold the sinks), then
// the tokens from position early + skip on (those that its first new token's
// window reaches). Both are multiples of 128 tokens, so that a tile of either
// is a run of positions.
struct ChunkSeq : AttendSeq {
    int32_t early, skip;
    int32_t tile0, rts;                      // its first expanded tile; its row tiles
};

struct ChunkView {
    using Seq = ChunkSeq;
    static constexpr bool SHARES = true;
    int32_t window, sinks;                   // no window: one larger than any position
    struct Row {
        int32_t p, from, sinks;              // sees `from` to p, and what is below sinks
        __host__ __device__ __forceinline__ bool sees(int t) const { return t <= p && (t >= from || t < sinks); }
        __host__ __device__ __forceinline__ uint32_t bits(int t) const {
            auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? FULL : (1u << n) - 1u; };
            return below(p + 1 - t) & (~below(from - t) | below(sinks - t));
        }
    };
    __host__ __device__ __forceinline__ int span(const Seq &s) const { return s.context + s.nodes - s.skip; }
    __host__ __device__ __forceinline__ int at(const Seq &s, int i) const { return i < s.early ? i : i + s.skip; }
    __host__ __device__ __forceinline__ Row row(const Seq &s, int node) const {
        return Row{s.context + node, s.context + node + 1 - window, sinks};
    }
    __host__ __device__ __forceinline__ bool whole(const Seq &s, int t, int n) const {
        return t + n - 1 <= s.context && (t >= s.context + s.nodes - window || t + n <= sinks);
    }
};

constexpr int TL_ROWS = 256, TL_TILE = 128, TL_IMAGE = TL_TILE * 128;      // an image: 128 rows of 64 fp16
constexpr int TL_STAGES = 4, TL_THREADS = 20 * 32;
constexpr int TL_Q_AT = 0, TL_KV_AT = 2 * 2 * TL_IMAGE, TL_UNIT_AT = TL_KV_AT + TL_STAGES * 2 * TL_IMAGE;
constexpr int TL_HALVES_AT = TL_UNIT_AT + 128, TL_BARS_AT = TL_HALVES_AT + 2048, TL_SMEM = TL_BARS_AT + 256;

// Pairs of 16 whose exponentials are polynomials, where no mask applies: 2,048
// tokens of 4 x 34,816 take 2,539 us with none, 2,369, 2,341, 2,356 and 2,409 with
// 3, 4, 5 and 6 (short runs, before the power cap).
constexpr int TL_POLY = 4;

struct TilesArgs {
    const DevTables *tb;
    const uint8_t *pool;
    const int32_t *table;
    const int32_t *q;
    __nv_bfloat16 *out;
    int32_t *ticket;
    uint8_t *q_images, *kv_images;           // [row tile][KV head][2 TL_IMAGE], [walk tile][KV head][keys, values]
    float *acc, *ml;                         // partials: [unit][TL_ROWS][64], [unit][TL_ROWS][2]
    int32_t *status;
    int32_t n_seqs, units, kv_ctas;
    int32_t poll_limit, hold_cta, hold_tile;
    float q_scale, k_scale, out_unit;
};

// A row tile's KV tiles, of positions 128 P on: P = j below `early`, j + jump
// from there on, j below `tiles`.
struct RowTile {
    int32_t first, n;                        // its tokens: new ones [first, first + n)
    int32_t early, jump, tiles;
};
__host__ __device__ __forceinline__ RowTile row_tile(const ChunkView &v, const ChunkSeq &s, int groups, int rt) {
    RowTile t;
    const int per = TL_ROWS / groups;
    t.first = rt * per;
    t.n = s.nodes - t.first < per ? s.nodes - t.first : per;
    const int lo = s.context + t.first, hi = lo + t.n - 1;
    const int from = lo + 1 > v.window ? (lo + 1 - v.window) / TL_TILE : 0;
    const int early = ((v.sinks < hi + 1 ? v.sinks : hi + 1) + TL_TILE - 1) / TL_TILE;
    t.early = from > early ? early : 0;
    t.jump = from > early ? from - early : 0;
    t.tiles = hi / TL_TILE + 1 - t.jump;
    return t;
}

// The KV tiles j of a row tile that all its rows see whole: those below `held` (of
// sinks), and from `from` to below `to`.
struct WholeTiles {
    int32_t held, from, to;
    __host__ __device__ __forceinline__ bool operator()(int j) const { return j < held || (j >= from && j < to); }
};
__host__ __device__ __forceinline__ WholeTiles whole_tiles(const ChunkView &v, int p_lo, int p_hi, int early, int jump) {
    const int sunk = v.sinks / TL_TILE, left = p_hi - v.window, from = left < 0 ? 0 : left / TL_TILE + 1 - jump;
    return WholeTiles{sunk < early ? sunk : early, from > early ? from : early, (p_lo + 1) / TL_TILE - jump};
}

// The walk of a sequence of `len` tokens whose last n are the chunk.
constexpr int WALK = 128;
static_assert(WALK % FEW_TILE == 0 && WALK % MANY_TILE == 0 && WALK % TL_TILE == 0, "a tile of a walk is a run of positions");
inline ChunkSeq walk_of(const ChunkView &v, int32_t seq, int64_t len, int32_t n, int64_t node0) {
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

// ---------------------------------------------------------------------------
// expanding: queries and cached rows into images
// ---------------------------------------------------------------------------

// Where 16 bytes c (of 8) of row r lie in an image: the 128-byte swizzle of the
// products' operands.
__device__ __forceinline__ int image_at(int r, int c) { return r * 128 + ((c ^ (r & 7)) * 16); }

// One CTA per (walk tile, KV head), then one per (row tile, KV head); a thread
// makes 16 bytes at a time. Bound by the bytes written.
template <int KB, int VB, class Src>
__global__ void __launch_bounds__(256) k_chunk_expand(Geo g, TilesArgs a, ChunkView view, const __grid_constant__ Src src) {
    __shared__ float cent[2][256];
    const int tid = threadIdx.x;
    const float cunit = exp2f((float)-g.centroid_frac);
    for (int i = tid; i < (1 << g.kb); i += 256) cent[0][i] = (float)a.tb->k_cent[i] * cunit;
    for (int i = tid; i < (1 << g.vb); i += 256) cent[1][i] = (float)a.tb->v_cent[i] * cunit;
    wait_prior_grid();
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) *a.ticket = 0;
    const ChunkSeq *seqs = reinterpret_cast<const ChunkSeq *>(src.data());
    if ((int)blockIdx.x < a.kv_ctas) {
        const int tile = blockIdx.x / g.n_kv, head = blockIdx.x % g.n_kv;
        int lo = 0, hi = a.n_seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (seqs[mid].tile0 <= tile) lo = mid;
            else hi = mid - 1;
        }
        const ChunkSeq sq = seqs[lo];
        const int i0 = (tile - sq.tile0) * TL_TILE, live = min(TL_TILE, view.span(sq) - i0), p0 = view.at(sq, i0);
        uint8_t *to = a.kv_images + (int64_t)blockIdx.x * 2 * TL_IMAGE;
#pragma unroll 2
        for (int i = tid; i < TL_TILE * 8; i += 256) {
            const int r = i / 8, c = i % 8;
            uint4 k = make_uint4(0, 0, 0, 0), v = k;     // past the end: zeros
            if (r < live) {
                const int p = p0 + r, page = page_of(g, p), in = row_in_page(g, p);
                const uint8_t *region = a.pool + region_off(g, a.table[(int64_t)sq.seq * g.max_pages + page], head);
                const uint32_t norms = __ldg(reinterpret_cast<const uint32_t *>(region + nplane_off(g)) + in);
                auto eight = [&](auto width, const uint8_t *codes, int bits_any, const float *cent8, float norm) {
                    constexpr int BITS = decltype(width)::value;
                    const int bits = BITS ? BITS : bits_any;
                    const uint8_t *at = codes + c * bits;
                    uint64_t w = 0;
                    if constexpr (BITS == 4) w = *reinterpret_cast<const uint32_t *>(at);
                    else if constexpr (BITS == 2) w = *reinterpret_cast<const uint16_t *>(at);
                    else
                        for (int b = 0; b < bits; ++b) w |= (uint64_t)at[b] << (8 * b);
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[j] = cent8[(uint32_t)(w >> (j * bits)) & ((1u << bits) - 1u)] * norm;
                    return make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]),
                                      pack_half2(x[6], x[7]));
                };
                k = eight(std::integral_constant<int, KB>(), region + (int64_t)in * g.kbytes, g.kb, cent[0],
                          norm_value(norms & 0xffffu, NORM_UNIT) * a.k_scale);
                v = eight(std::integral_constant<int, VB>(), region + vplane_off(g) + (int64_t)in * g.vbytes, g.vb,
                          cent[1], norm_value(norms >> 16, NORM_UNIT));
            }
            *reinterpret_cast<uint4 *>(to + image_at(r, c)) = k;
            *reinterpret_cast<uint4 *>(to + TL_IMAGE + image_at(r, c)) = v;
        }
        return;
    }
    // a row tile's queries, in log2 units
    const int unit = blockIdx.x - a.kv_ctas, item = unit / g.n_kv, head = unit % g.n_kv;
    int lo = 0, hi = a.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (seqs[mid].group0 <= item) lo = mid;
        else hi = mid - 1;
    }
    const ChunkSeq sq = seqs[lo];
    const RowTile t = row_tile(view, sq, g.H, item - sq.group0);
    uint8_t *to = a.q_images + (int64_t)unit * 2 * TL_IMAGE;
    const float u = Q_UNIT * a.q_scale;
#pragma unroll 4
    for (int i = tid; i < TL_ROWS * 8; i += 256) {
        const int r = i / 8, c = i % 8;
        uint4 w = make_uint4(0, 0, 0, 0);
        if (r < t.n * g.H) {
            const int4 *p = reinterpret_cast<const int4 *>(
                a.q + (((int64_t)(sq.node0 + t.first + r / g.H) * g.n_kv + head) * g.H + r % g.H) * D + 8 * c);
            const int4 y = p[0], z = p[1];
            w = make_uint4(pack_half2((float)y.x * u, (float)y.y * u), pack_half2((float)y.z * u, (float)y.w * u),
                           pack_half2((float)z.x * u, (float)z.y * u), pack_half2((float)z.z * u, (float)z.w * u));
        }
        *reinterpret_cast<uint4 *>(to + r / 128 * TL_IMAGE + image_at(r % 128, c)) = w;
    }
}

// ---------------------------------------------------------------------------
// the attention
// ---------------------------------------------------------------------------

// What a CTA works on, in shared memory (two: the loader is one ahead).
struct TilesUnit {
    int32_t end;                             // no more units
    int32_t node0, head, first, rows;        // its row tile: the sequence's and its first new token, query rows
    int32_t p_lo, p_hi;                      // its tokens' positions
    int32_t early, jump, lo, hi;             // its KV tiles [lo, hi) of the row tile's
    int32_t slot;                            // partial slot, -1: all of the row tile's KV tiles
};

// 2^v of two values by additions and multiplications: the special function unit
// makes 16 exponentials a clock and SM, and bounds the kernel where it makes all.
// With n the integer nearest to v and f = v - n, 2^f is a polynomial of degree
// 3 (of least largest relative error on [-1/2, 1/2]: 2^-13.7, below P's rounding
// to fp16, and the same in P and in its sum), and n is added to the exponent's
// bits: for |v| up to 126.
constexpr float POLY0 = 0.9999280571937561f, POLY1 = 0.6932609677314758f, POLY2 = 0.2426111251115799f,
                POLY3 = 0.0551716685295105f, POLY_RANGE = 126.0f;
__device__ __forceinline__ float2 exp2_pair(uint64_t v) {
    auto both = [](float c) { return pair64(__float_as_uint(c), __float_as_uint(c)); };
    const uint64_t t = add_pair(v, both(12582912.0f));           // 1.5 * 2^23: n in the low bits
    const uint64_t f = fma_pair(add_pair(t, both(-12582912.0f)), both(-1.0f), v);
    uint64_t r = fma_pair(f, both(POLY3), both(POLY2));
    r = fma_pair(r, f, both(POLY1));
    r = fma_pair(r, f, both(POLY0));
    const float2 n = split64(t), y = split64(r);
    return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(n.x) << 23)),
                       __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(n.y) << 23)));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// P = exp2(S - ref) of 64 columns of a row in fp16 pairs, with a factor of 2^7
// (as sum has). ref is the largest score of some that the row has seen: under
// the row's own maximum the weights sum to 2^13 at most; true if they exceed
// 2^15, or a polynomial's range (P and sum are then not valid). Up to there
// every weight is inside fp16, which keeps them down to 2^-31 of the maximum,
// and no comparison of all scores is needed. A row that has seen nothing yet
// (-inf: a window leaves its unit's first tiles out) has no such ref, and its
// sum says nothing: true too. POLY of 16 pairs go by polynomials.
template <bool MASKED, int POLY, class Row>
__device__ __forceinline__ bool weigh_half(uint32_t S, float ref, float &sum, uint32_t (&p)[32], const Row &row, int t0) {
    const float sub = (ref > -INFINITY ? -ref : 0.0f) + 7.0f;
    const uint64_t sub2 = pair64(__float_as_uint(sub), __float_as_uint(sub));
    uint64_t acc[2] = {0, 0};
    float far = 0.0f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        uint32_t x[32];
        tc_load32(x, S + 32 * c);
        tc_wait_load(x);
        if (MASKED) {
            const uint32_t see = row.bits(t0 + 32 * c);
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = (see >> j) & 1 ? x[j] : 0xff800000u;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const uint64_t v2 = add_pair(pair64(x[2 * j], x[2 * j + 1]), sub2);
            const float2 v = split64(v2);
            float2 e;
            if (j * POLY / 16 != (j + 1) * POLY / 16) {
                e = exp2_pair(v2);
                far = max3(far, fabsf(v.x), fabsf(v.y));
            } else {
                e = make_float2(ex2(v.x), ex2(v.y));
            }
            acc[j & 1] = add_pair(acc[j & 1], pair64(__float_as_uint(e.x), __float_as_uint(e.y)));
            p[16 * c + j] = pack_half2(e.x, e.y);
        }
    }
    const float2 v = split64(add_pair(acc[0], acc[1]));
    sum = v.x + v.y;
    return !(ref > -INFINITY) || sum > 32768.0f || (POLY && far > POLY_RANGE);
}
// The largest of a row's 64 columns that it sees, and of `m`.
template <class Row>
__device__ __noinline__ float largest_half(uint32_t S, float m, const Row row, int t0) {
    uint32_t x[32];
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
        tc_load32(x, S + 32 * c);
        tc_wait_load(x);
        hide<true>(x, row, t0 + 32 * c);
        m = largest(x, m);
    }
    return m;
}
// 32 output columns times f.
__device__ __noinline__ void scale_half(uint32_t O, float f) {
    uint32_t x[32];
    tc_load32(x, O);
    tc_wait_load(x);
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * f);
    tc_store16(O, x);
    tc_store16(O + 16, x + 16);
    tc_wait_st();
}
// True for both warps of a pair if `x` is for one of their threads. They wait
// for one another: each comes here as often as the other.
__device__ __forceinline__ bool pair_any(int pair, bool x) {
    uint32_t r;
    asm volatile(
        "{ .reg .pred p, q; setp.ne.u32 p, %1, 0; barrier.cta.red.or.pred q, %2, 64, p; selp.u32 %0, 1, 0, q; }"
        : "=r"(r)
        : "r"((uint32_t)x), "r"(1 + pair)
        : "memory");
    return r;
}

// bar_wait of a whole warp: the first look is all that most waits need.
__device__ __forceinline__ bool warp_wait(uint32_t bar, int phase, int limit) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done)
                 : "r"(bar), "r"((uint32_t)phase & 1u)
                 : "memory");
    if (__all_sync(FULL, done)) return true;
    return __all_sync(FULL, bar_wait(bar, (uint32_t)phase & 1u, limit));
}

template <class Src>
__global__ void __launch_bounds__(TL_THREADS, 1) k_chunk_tiles(Geo g, TilesArgs a, ChunkView view,
                                                               const __grid_constant__ Src src) {
    extern __shared__ __align__(1024) uint8_t tiles_smem[];
    uint8_t *const sm = tiles_smem;
    const uint32_t sm0 = smem_u32(sm);
    const int tid = threadIdx.x, warp = __shfl_sync(FULL, tid / 32, 0), lane = tid % 32;
    const uint32_t bars = sm0 + TL_BARS_AT;
    auto kv_full = [&](int i) { return bars + 8 * i; };
    auto kv_empty = [&](int i) { return bars + 32 + 8 * i; };
    auto q_full = [&](int i) { return bars + 64 + 8 * i; };
    auto q_empty = [&](int i) { return bars + 80 + 8 * i; };
    // of step k, k % 6: its stream is k % 2, its score buffer k % 3
    auto s_ready = [&](int k) { return bars + 96 + 8 * k; };
    auto p_ready = [&](int k) { return bars + 144 + 8 * k; };
    auto pv_done = [&](int k) { return bars + 192 + 8 * k; };
    const uint32_t fin = bars + 240;
    volatile uint32_t *tmem_at = reinterpret_cast<uint32_t *>(sm + TL_BARS_AT + 248);
    TilesUnit *unit_sm = reinterpret_cast<TilesUnit *>(sm + TL_UNIT_AT);
    static_assert(2 * sizeof(TilesUnit) <= 128, "two units");

    if (tid == 0) {
        for (int i = 0; i < TL_STAGES; ++i) bar_init(kv_full(i), 1), bar_init(kv_empty(i), 2);
        for (int i = 0; i < 2; ++i) {
            bar_init(q_full(i), 1), bar_init(q_empty(i), 19);
        }
        for (int k = 0; k < 6; ++k) bar_init(s_ready(k), 1), bar_init(p_ready(k), 8), bar_init(pv_done(k), 1);
        bar_init(fin, 3);
        bar_init_fence();
    }
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32((void *)tmem_at))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    wait_prior_grid();
    __syncthreads();
    tc_fence_after();
    constexpr uint32_t tmem = 0;                     // all columns are this CTA's
    if (*tmem_at != tmem || (sm0 & 1023)) {          // never: reported, not worked around
        if (tid == 0) atomicOr(a.status, ST_INTERNAL);
        __syncthreads();
        if (warp == 16)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(*tmem_at) : "memory");
        return;
    }
    // score buffer b at column 128 b, output of stream i at 384 + 64 i

    bool lost = false;                               // a wait gave up: the same for all lanes of a warp
    auto wait = [&](uint32_t bar, int phase) {
        if (!warp_wait(bar, phase, a.poll_limit)) {
            lost = true;
            if (lane == 0) atomicOr(a.status, ST_TIMEOUT);
        }
    };

    if (warp == 19) {
        // ---- loads
        const ChunkSeq *seqs = reinterpret_cast<const ChunkSeq *>(src.data());
        int kt = 0, n = 0;                           // KV tiles, units so far
        for (;;) {
            int u = 0;
            if (lane == 0) u = atomicAdd(a.ticket, 1);
            u = __shfl_sync(FULL, u, 0);
            const int slot = n & 1;
            if (n >= 2) wait(q_empty(slot), n / 2 - 1);
            if (lost) break;
            if (u >= a.units) {
                if (lane == 0) {
                    unit_sm[slot].end = 1;
                    bar_arrive(q_full(slot));
                }
                break;
            }
            const ChunkSeq sq = seqs[find_seq<false>(seqs, a.n_seqs, u)];
            // (row tile, falling; KV head; piece)
            const int local = u - sq.unit0, piece = local % sq.splits, item = local / sq.splits;
            const int head = item % g.n_kv, rt = sq.rts - 1 - item / g.n_kv;
            const RowTile t = row_tile(view, sq, g.H, rt);
            const int lo = (int)((int64_t)t.tiles * piece / sq.splits), hi = (int)((int64_t)t.tiles * (piece + 1) / sq.splits);
            if (lo == hi) {                          // a piece of a row tile of few tiles: nothing
                for (int r = lane; r < TL_ROWS; r += 32)
                    *reinterpret_cast<float2 *>(a.ml + ((int64_t)u * TL_ROWS + r) * 2) = make_float2(-INFINITY, 0.0f);
                continue;
            }
            if (lane == 0) {
                TilesUnit &w = unit_sm[slot];
                w.end = 0;
                w.node0 = sq.node0, w.head = head, w.first = t.first, w.rows = t.n * g.H;
                w.p_lo = sq.context + t.first, w.p_hi = w.p_lo + t.n - 1;
                w.early = t.early, w.jump = t.jump, w.lo = lo, w.hi = hi;
                w.slot = sq.splits > 1 ? u : -1;
                bar_expect(q_full(slot), 2 * TL_IMAGE);
                copy_bulk(sm0 + TL_Q_AT + slot * 2 * TL_IMAGE,
                          a.q_images + ((int64_t)(sq.group0 + rt) * g.n_kv + head) * 2 * TL_IMAGE, 2 * TL_IMAGE, q_full(slot));
            }
            for (int j = lo; j < hi && !lost; ++j, ++kt) {
                const int st = kt % TL_STAGES;
                if (kt >= TL_STAGES) wait(kv_empty(st), kt / TL_STAGES - 1);
                if (lost) break;
                const int tile = j < t.early ? j : j + t.jump;
                const int walk = tile < sq.early / TL_TILE ? tile : tile - sq.skip / TL_TILE;
                if (lane == 0) {
                    const bool held = (int)blockIdx.x == a.hold_cta && kt == a.hold_tile;
                    bar_expect(kv_full(st), 2 * TL_IMAGE + (held ? 16 : 0));
                    copy_bulk(sm0 + TL_KV_AT + st * 2 * TL_IMAGE,
                              a.kv_images + ((int64_t)(sq.tile0 + walk) * g.n_kv + head) * 2 * TL_IMAGE, 2 * TL_IMAGE,
                              kv_full(st));
                }
                __syncwarp();
            }
            ++n;
            if (lost) break;
        }
        // copies in flight land before the CTA goes
        if (lost) {
            for (int k = max(0, kt - TL_STAGES); k < kt; ++k)
                bar_wait(kv_full(k % TL_STAGES), (k / TL_STAGES) & 1, a.poll_limit);
            for (int k = max(0, n - 2); k < n; ++k) bar_wait(q_full(k & 1), (k / 2) & 1, a.poll_limit);
        }
    } else if (warp >= 16) {
        // ---- products: one warp issues the score products, one a stream its value
        // products. All lanes walk the same steps, one elected lane issues. Step k
        // (of all units, one after another) is stream k % 2's of a KV tile and uses
        // score buffer k % 3.
        int kt = 0, k6 = 0, use = 0;                 // KV tiles so far; the next step: k % 6, k / 6
        if (warp == 16) {
            constexpr uint32_t idesc = tc_idesc(128, false);
            const uint64_t q_desc = tc_desc(sm0 + TL_Q_AT), k_desc = tc_desc(sm0 + TL_KV_AT);
            for (int n = 0; !lost; ++n) {
                wait(q_full(n & 1), n >> 1);
                if (lost) break;
                const TilesUnit un = unit_sm[n & 1];
                if (un.end) break;
                const uint64_t q = q_desc + (uint64_t)((n & 1) * (2 * TL_IMAGE >> 4));
                for (int j = un.lo; j < un.hi && !lost; ++j, ++kt) {
                    const int st = kt % TL_STAGES;
                    wait(kv_full(st), kt / TL_STAGES);
                    const uint64_t k = k_desc + (uint64_t)(st * (2 * TL_IMAGE >> 4));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // its buffer's last step was k - 3
                        if (!lost && (use || k6 >= 3)) wait(pv_done(k6 >= 3 ? k6 - 3 : k6 + 3), k6 >= 3 ? use : use - 1);
                        if (lost) break;
                        tc_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                tc_mma_ss(tmem + 128 * (k6 % 3), q + (uint64_t)(i * (TL_IMAGE >> 4)) + 2 * x, k + 2 * x, idesc,
                                          x > 0);
                            tc_commit(s_ready(k6));
                        }
                        __syncwarp();
                        k6 = k6 == 5 ? 0 : k6 + 1;
                        use += k6 == 0;
                    }
                }
                if (elect_one()) tc_commit(q_empty(n & 1));
                __syncwarp();
            }
        } else {
            const int i = warp - 17;
            constexpr uint32_t idesc = tc_idesc(64, true);
            const uint64_t v_desc = tc_desc(sm0 + TL_KV_AT + TL_IMAGE);
            k6 = i;
            for (int n = 0; !lost; ++n) {
                wait(q_full(n & 1), n >> 1);
                if (lost) break;
                const TilesUnit un = unit_sm[n & 1];
                if (un.end) break;
                for (int j = un.lo; j < un.hi && !lost; ++j, ++kt) {
                    const int st = kt % TL_STAGES;
                    wait(kv_full(st), kt / TL_STAGES);
                    if (!lost) wait(p_ready(k6), use);
                    if (lost) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t v = v_desc + (uint64_t)(st * (2 * TL_IMAGE >> 4));
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            tc_mma_ts(tmem + 384 + 64 * i, tmem + 128 * (k6 % 3) + 8 * x, v + 128 * x, idesc,
                                      j > un.lo || x > 0);
                        tc_commit(pv_done(k6));
                        tc_commit(kv_empty(st));
                    }
                    __syncwarp();
                    k6 = k6 >= 4 ? k6 - 4 : k6 + 2;
                    use += k6 < 2;
                }
                if (lane == 0) bar_arrive(q_empty(n & 1));
            }
        }
        // nothing may be in flight when the tensor memory goes
        if (elect_one()) tc_commit(fin);
        __syncwarp();
        if (!bar_wait(fin, 0, WAIT_POLLS)) atomicOr(a.status, ST_TIMEOUT);
        __syncwarp();
    } else {
        // ---- softmax: of a query row (`row` of stream `i`) two threads own 64
        // columns of scores each (half `h`), so that four warps of each scheduler
        // hide one another's latencies. A wait that gave up is known to both warps
        // of a pair at their next meeting, where they leave together.
        const int i = warp / 8, h = warp / 4 % 2, row = tid % 128, pair = 4 * i + warp % 4;
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;   // lane 32 (warp % 4), in bits 16 up
        const uint32_t O = tmem + lanes + 384 + 64 * i + 32 * h;
        float *const mine = reinterpret_cast<float *>(sm + TL_HALVES_AT) + (2 * i + h) * 128 + row;
        float *const other = reinterpret_cast<float *>(sm + TL_HALVES_AT) + (2 * i + 1 - h) * 128 + row;
        int k6 = i, use = 0;                                 // the stream's next step k: k % 6, k / 6
        int last = 0, last_use = 0;                          // its last one
        for (int n = 0;; ++n) {
            wait(q_full(n & 1), n >> 1);
            if (pair_any(pair, lost)) break;
            const TilesUnit un = unit_sm[n & 1];
            if (un.end) break;
            const int r = 128 * i + row;
            const bool any_row = r - lane < un.rows;         // of this warp's 32
            const int p = min(un.p_lo + r / g.H, un.p_hi);
            const ChunkView::Row sees{p, p + 1 - view.window, view.sinks};
            float ref = -INFINITY, l = 0.0f;
            bool left = false;
            const WholeTiles is_whole = whole_tiles(view, un.p_lo, un.p_hi, un.early, un.jump);
            for (int j = un.lo; j < un.hi; ++j) {
                const int t0 = (j < un.early ? j : j + un.jump) * TL_TILE + 64 * h;
                const bool whole = is_whole(j);
                const uint32_t S = tmem + lanes + 128 * (k6 >= 3 ? k6 - 3 : k6);
                wait(s_ready(k6), use);
                tc_fence_after();
                if (any_row) {
                    float sum = 0.0f;
                    uint32_t w[32];
                    bool over = lost || j == un.lo;
                    // the exponentials are taken under the maximum so far, and again in
                    // the rare case that there is none, or it was too low
                    if (!over) {
                        if (whole) over = weigh_half<false, TL_POLY>(S + 64 * h, ref, sum, w, sees, t0);
                        else over = weigh_half<true, 0>(S + 64 * h, ref, sum, w, sees, t0);
                    }
                    if (pair_any(pair, over)) {
                        // O is this stream's once its last value product is done
                        if (j > un.lo && !lost) wait(pv_done(last), last_use);
                        tc_fence_after();
                        if (pair_any(pair, lost)) {
                            left = true;
                            break;
                        }
                        *mine = largest_half(S + 64 * h, ref, sees, t0);
                        pair_any(pair, false);
                        const float now = fmaxf(*mine, *other), f = now > -INFINITY ? ex2(ref - now) : 1.0f;
                        ref = now;
                        l *= f;
                        if (j > un.lo) scale_half(O, f);
                        weigh_half<true, 0>(S + 64 * h, ref, sum, w, sees, t0);
                        pair_any(pair, false);               // all scores have been read: P may replace them
                    }
                    l += sum;
                    tc_store16(S + 32 * h, w);
                    tc_store16(S + 32 * h + 16, w + 16);
                    tc_wait_st();
                } else if (lost) {
                    left = true;
                    break;
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(p_ready(k6));
                last = k6, last_use = use;
                k6 = k6 >= 4 ? k6 - 4 : k6 + 2;
                use += k6 < 2;
            }
            // (warps without rows meet nowhere in the loop)
            if (!left && !lost) wait(pv_done(last), last_use);
            *mine = l;
            if (pair_any(pair, left || lost)) break;
            l += *other;
            tc_fence_after();
            // this row's sums out, 32 channels each half
            uint32_t x[32];
            tc_load32(x, O);
            tc_wait_load(x);
            if (r < un.rows) {
                if (un.slot < 0) {
                    const float inv = a.out_unit / l;        // (every row sees itself)
                    uint4 *dst = reinterpret_cast<uint4 *>(
                        a.out + (((int64_t)(un.node0 + un.first + r / g.H) * g.n_kv + un.head) * g.H + r % g.H) * D + 32 * h);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t o[4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(x[8 * k + 2 * y]) * inv,
                                                                           __uint_as_float(x[8 * k + 2 * y + 1]) * inv);
                            o[y] = *reinterpret_cast<const uint32_t *>(&v);
                        }
                        dst[k] = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                } else {
                    const int64_t at = (int64_t)un.slot * TL_ROWS + r;
                    uint4 *dst = reinterpret_cast<uint4 *>(a.acc + at * 64 + 32 * h);
#pragma unroll
                    for (int k = 0; k < 8; ++k) dst[k] = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
                    if (h == 0) a.ml[at * 2] = ref, a.ml[at * 2 + 1] = l;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(q_empty(n & 1));
        }
    }
    __syncthreads();
    if (warp == 16)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// The pieces of a row tile, scaled to the largest of their maxima, added in
// order and divided by the sum of weights. A piece of which a row sees nothing
// has a maximum of -inf and weighs nothing; the one that holds the row's own
// token has a finite one. One CTA per 8 rows; a sequence whose row tiles are
// whole has nothing to join.
template <class Src>
__global__ void __launch_bounds__(128) k_chunk_join(Geo g, TilesArgs a, ChunkView view, const __grid_constant__ Src src) {
    extern __shared__ float wt[];                    // [8][splits]
    wait_prior_grid();
    const ChunkSeq *seqs = reinterpret_cast<const ChunkSeq *>(src.data());
    constexpr int PER = TL_ROWS / 8;
    const int part8 = blockIdx.x % PER * 8, group = blockIdx.x / PER, head = group % g.n_kv, item = group / g.n_kv;
    const ChunkSeq sq = seqs[find_seq<true>(seqs, a.n_seqs, item)];
    const int rt = item - sq.group0, splits = sq.splits;
    const RowTile t = row_tile(view, sq, g.H, rt);
    const int rows = min(8, t.n * g.H - part8);
    if (splits == 1 || rows <= 0) return;
    const int64_t unit = sq.unit0 + ((int64_t)(sq.rts - 1 - rt) * g.n_kv + head) * splits;
    auto slot = [&](int s, int r) { return (unit + s) * TL_ROWS + part8 + r; };
    for (int r = threadIdx.x / 32; r < rows; r += 4) {
        const int lane = threadIdx.x % 32;
        float M = -INFINITY, sum = 0.0f;
        for (int s = lane; s < splits; s += 32) M = fmaxf(M, a.ml[slot(s, r) * 2]);
        for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(FULL, M, o));
        for (int s = lane; s < splits; s += 32) {
            const float f = ex2(a.ml[slot(s, r) * 2] - M);
            sum += f * a.ml[slot(s, r) * 2 + 1];
            wt[r * splits + s] = f;
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
        const float inv = a.out_unit / sum;
        for (int s = lane; s < splits; s += 32) wt[r * splits + s] *= inv;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * 16; i += 128) {
        const int r = i / 16, c4 = i % 16, qr = part8 + r;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int s = 0; s < splits; ++s) {
            const float f = wt[r * splits + s];
            if (f == 0.0f) continue;                 // (a piece of no tiles has written no sums)
            const float4 v = reinterpret_cast<const float4 *>(a.acc)[slot(s, r) * 16 + c4];
            o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
        }
        __nv_bfloat162 *dst = reinterpret_cast<__nv_bfloat162 *>(
            a.out + (((int64_t)(sq.node0 + t.first + qr / g.H) * g.n_kv + head) * g.H + qr % g.H) * D + c4 * 4);
        dst[0] = __floats2bfloat162_rn(o.x, o.y);
        dst[1] = __floats2bfloat162_rn(o.z, o.w);
    }
}

}  // namespace ins
