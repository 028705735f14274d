// Attention of drafted trees over the compressed cache.
//
// Each of B sequences holds `context` tokens followed by `nodes` drafted ones
// (all already in the cache). Node i attends the whole context and the
// drafted tokens that its mask names (its ancestors and itself). With a
// cached row's key k = norm_k/2^9 * cent_k[code]/2^15 and its value likewise,
// the scores are s = <q/2^16, k>, the output sum exp(s - m) v / sum exp(s - m).
// This is the floating-point reading of the cache that the fixed-point scans
// read in integers; a tree of one node is a decode token's attention.
//
// The queries of a (sequence, KV head) are nodes x kv_groups rows that share
// every cached row, so both products are matrix products whose second operand
// is decoded from codes on the way: fp16 operands (a centroid, a query or a
// probability is rounded to 11 bits, which moves the bf16 result by less than
// its own rounding), fp32 sums, maxima and exponents.
//
// The products take the query as q/2^16 and the norms as norm/2^9 whatever
// the cache's formats are: 32-bit queries stay below 2^15 then and 16-bit
// norms up to 2^6, inside fp16's range with the weights' own factors. The
// powers of two between these and the formats (1 for the default ones) go to
// the scores and to the outputs in fp32 (TreeArgs::score_unit, out_unit);
// k_tree_many, whose exponentials have no room for another multiplication (2 %
// of its time), takes a score's down to its queries or up to its keys' norms.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "plan.cuh"

namespace ins {

constexpr int TREE_MAX_NODES = 256;          // drafted tokens of one sequence
constexpr float LOG2E = 1.4426950408889634f;
constexpr float Q_UNIT = LOG2E / 65536.0f;   // of a query, in log2 units
constexpr float NORM_UNIT = 1.0f / 512.0f;

// One sequence of a call. Its work units are [unit0, next sequence's unit0):
// (split of `chunk` tokens, row tile, KV head), the head innermost.
struct TreeSeq {
    int32_t seq, context, nodes, node0, splits, unit0, group0;
};

struct TreeArgs {
    const DevTables *tb;
    const uint8_t *pool;
    const int32_t *table;
    const int32_t *q;
    const uint64_t *mask;
    __nv_bfloat16 *out;
    float *acc, *ml;                         // partials: [unit][rows][64], [unit][rows][2]
    int32_t *status;
    int32_t n_seqs, words, chunk, row_tiles_rows;
    int32_t poll_limit, hold_cta, hold_tile; // tests: the tile whose copies are announced too large
    // what the products' fixed units leave to the formats: for the scores (k_tree_many: its two factors), the outputs
    float score_unit, q_scale, k_scale, out_unit;
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_init_fence() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Orders this thread's ordinary accesses to shared memory before later ones by
// copies and tensor cores (once a barrier has passed).
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Waits for the phase of `parity`, at most `limit` polls; false: it gave up
// (this thread did: a warp has to agree before it goes on).
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int limit) {
    for (int i = 0; i < limit; ++i) {
        uint32_t done;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                     : "=r"(done)
                     : "r"(bar), "r"(parity)
                     : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ void copy_bulk(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Byte `i` of w times 256 plus `lane4` (below 256): the address of a code
// byte's entry in a table of 256-byte entries, at this lane's copy.
__device__ __forceinline__ uint32_t entry_at(uint32_t w, int i, uint32_t lane4) {
    return __byte_perm(w, lane4, 0x5504 | (i << 4));
}
// A word of the constant tables (not volatile: loads may be batched).
__device__ __forceinline__ uint32_t load_shared(uint32_t at) {
    uint32_t x;
    asm("ld.shared.u32 %0, [%1];" : "=r"(x) : "r"(at));
    return x;
}
// c += a b, one 16x8 tile of 16-wide products
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 matrix of 16-bit elements, two of row lane / 4 a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// A 16-bit norm's value (int16 / 2^norm_frac): 2^23 + x is a float's bits, so
// no integer conversion (which runs at an eighth of the rate) is needed.
__device__ __forceinline__ float norm_value(uint32_t x16, float unit) {
    return fmaf(__uint_as_float(0x4b000000u | (x16 ^ 0x8000u)), unit, -8421376.0f * unit);
}

// Position p's page index and row in the page (a shift where pages hold a power
// of two rows, as they do by default: a division is some 20 instructions).
__device__ __forceinline__ int page_of(const Geo &g, int p) { return g.p_log2 >= 0 ? p >> g.p_log2 : p / g.P; }
__device__ __forceinline__ int row_in_page(const Geo &g, int p) {
    return g.p_log2 >= 0 ? p & (g.P - 1) : p % g.P;
}

// The sequence that unit (or, GROUP, row group) `i` belongs to.
template <bool GROUP>
__device__ __forceinline__ int find_seq(const TreeSeq *seqs, int n, int i) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if ((GROUP ? seqs[mid].group0 : seqs[mid].unit0) <= i) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// ---------------------------------------------------------------------------
// few rows: warps, codes decoded straight into mma fragments
// ---------------------------------------------------------------------------
//
// A CTA takes 16 MT rows and a run of tokens; its warps take tiles of 64
// tokens in turn, each with a running maximum, sum and accumulator of its own
// (joined at the end through shared memory) and a ring of bulk copies of its
// tiles' three planes, so no warp waits for another inside the loop.
//
// The products' inner orders are free: of a token's key a lane decodes 16
// adjacent channels (one run of its bits), of its value 8 adjacent channels,
// and the query fragments are laid out to match. A pair of key codes is one
// index into a table of half2 with a copy for each lane (32 banks: no
// conflicts), and so is a pair of value codes of two tokens.
// Norms stay factored out: the key's scales the score, the value's the
// probability.
//
// The running maximum moves only when a score exceeds it by more than 2^8
// (LAG, in the exponent's base): until then exp2 stays below 256 and times a
// norm (at most 2^6) below 2^14, inside fp16's range, so a rescale of the accumulators is
// rare and the maximum needs no exchange of lanes at every step.
//
// Up to 8 rows (HALF) the products are taken transposed, S^T = K Q^T and
// O^T += V^T P^T: tokens and channels are the 16 rows of a matrix instruction
// and queries its 8 columns, which halves the products and the accumulators;
// P^T changes from a result's layout to an operand's by two 8 x 8 transposes.
//
// Bound by instructions: of the 16 tokens' 2,048 codes a warp's step makes 32
// table addresses and 24 loads, and some 190 instructions in all (other code
// widths decode a code at a time: 3b/2b 641 us where 4b/2b takes 139). One token
// of 1,048,576 (8 KV heads of 4 query heads, 4b/2b) takes 139 us: 3.1 TB/s of
// the 436 MB of codes and norms. With the products the other way round,
// 4-byte value entries and 16 warps of 128 registers it took 198 us.

constexpr int FEW_TILE = 64;
constexpr float LAG = 8.0f;
// The running maximum of a row that has seen nothing: finite, so that a masked
// score's exponential is exp2(-inf) = 0 under it too, and below every score.
constexpr float NONE = -1e30f;

template <int KB, int VB>
struct FewLayout {
    static constexpr bool PAIRS = KB != 0;                       // else one code at a time, any width
    static constexpr int K_ENTRIES = PAIRS ? 1 << (2 * KB) : 0;
    static constexpr int V_ENTRIES = PAIRS && VB > 2 ? 1 << (2 * VB) : 0;
    // 4b/2b: a key entry's 32 lanes' copies fill 128 of its 256 bytes, so that
    // one byte permute makes an entry's address of a code byte; the other 128
    // hold, for a byte of two tokens' codes of two channels, both channels'
    // pairs: 8 bytes, 16 copies (a 64-bit load takes half a warp at a time)
    static constexpr bool WIDE = KB == 4 && VB == 2;
    static constexpr int KLUT = K_ENTRIES * (WIDE ? 256 : 128), VLUT = V_ENTRIES * 128, SINGLE = PAIRS ? 0 : 1024;
    static constexpr int NORMS_AT = KLUT + VLUT + SINGLE;        // [warps][64] (key, value) norms
    // ring slots a warp
    __host__ __device__ static constexpr int stages(int warps) { return warps > 16 ? 2 : 3; }
    __host__ __device__ static constexpr int stages_at(int warps) { return NORMS_AT + warps * 512; }
    __host__ __device__ static int stage_bytes(const Geo &g) { return FEW_TILE * (g.kbytes + g.vbytes + 4); }
    __host__ __device__ static int bars_at(const Geo &g, int warps) {
        return stages_at(warps) + warps * stages(warps) * stage_bytes(g);
    }
    // the end-of-loop join reuses the stages: [warps][rows][64] floats, [warps][rows][2]
    __host__ static size_t bytes(const Geo &g, int warps, int rows) {
        const size_t loop = (size_t)bars_at(g, warps) + warps * stages(warps) * 8;
        const size_t join = (size_t)stages_at(warps) + (size_t)warps * rows * (64 + 2) * 4;
        return std::max(loop, join);
    }
};

template <int KB, int VB, int MT, bool HALF, int NW, class Src>
__global__ void __launch_bounds__(NW * 32, 1) k_tree_few(Geo g, TreeArgs a, const __grid_constant__ Src src) {
    using L = FewLayout<KB, VB>;
    constexpr int R = 16 * MT;                       // rows of this CTA's tile
    constexpr int HR = HALF ? 1 : 2;                 // of a query fragment's two row halves, those that hold queries
    constexpr int STAGES = L::stages(NW);
    extern __shared__ __align__(128) uint8_t sm[];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, t4 = lane % 4, g8 = lane / 4;
    const uint32_t sm0 = smem_u32(sm);
    const int kbytes = KB ? KB * 8 : g.kbytes, vbytes = VB ? VB * 8 : g.vbytes;
    const int stage = FEW_TILE * (kbytes + vbytes + 4);
    const uint32_t ring = sm0 + L::stages_at(NW) + warp * STAGES * stage;
    const uint32_t bars = sm0 + L::bars_at(g, NW) + warp * STAGES * 8;

    // tables: constant, so filled before the wait for earlier launches
    const float cunit = exp2f((float)-g.centroid_frac);
    if (L::PAIRS) {
        float *cent = reinterpret_cast<float *>(sm + L::stages_at(NW));
        if (tid < (1 << KB)) cent[tid] = (float)a.tb->k_cent[tid] * cunit;
        if (tid >= 32 && tid < 32 + (1 << VB)) cent[tid] = (float)a.tb->v_cent[tid - 32] * cunit;
        __syncthreads();
        for (int e = warp; e < L::K_ENTRIES; e += NW)
            reinterpret_cast<uint32_t *>(sm)[e * (L::WIDE ? 64 : 32) + lane] =
                pack_half2(cent[e & ((1 << KB) - 1)], cent[e >> KB]);
        if (L::WIDE)
            for (int e = warp; e < 256; e += NW) {
                const int c = 2 * (lane / 16);                   // this half warp's channel of the two
                reinterpret_cast<uint32_t *>(sm)[e * 64 + 32 + lane % 16 * 2 + lane / 16] =
                    pack_half2(cent[32 + (e >> c & 3)], cent[32 + (e >> (4 + c) & 3)]);
            }
        for (int e = warp; e < L::V_ENTRIES; e += NW)
            reinterpret_cast<uint32_t *>(sm + L::KLUT)[e * 32 + lane] =
                pack_half2(cent[32 + (e & ((1 << VB) - 1))], cent[32 + (e >> VB)]);
    } else {
        __half *tab = reinterpret_cast<__half *>(sm);
        for (int i = tid; i < 512; i += NW * 32)
            tab[i] = __float2half_rn((float)(i < 256 ? a.tb->k_cent[i] : a.tb->v_cent[i - 256]) * cunit);
    }
    if (lane == 0)
        for (int i = 0; i < STAGES; ++i) bar_init(bars + i * 8, 1);
    bar_init_fence();
    fence_async();                                   // copies overwrite the centroids
    wait_prior_grid();
    __syncthreads();

    const TreeSeq *seqs = reinterpret_cast<const TreeSeq *>(src.data());
    const TreeSeq sq = seqs[find_seq<false>(seqs, a.n_seqs, blockIdx.x)];
    const int G = g.H, rows_all = sq.nodes * G, tiles = (rows_all + R - 1) / R;
    int unit = blockIdx.x - sq.unit0;
    const int head = unit % g.n_kv;
    unit /= g.n_kv;
    const int rt = unit % tiles, split = unit / tiles;
    const int row0 = rt * R, len = sq.context + sq.nodes;
    const int lo = split * a.chunk, hi = min(len, lo + a.chunk);
    const int n_tiles = (hi - lo + FEW_TILE - 1) / FEW_TILE;

    // query fragments: rows g8 and g8 + 8 of each 16; k pairs (2 t4, +1) and
    // (+8, +9) of step ks hold channels 16 t4 + 4 ks + {0, 1} and + {2, 3}
    uint32_t qf[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = row0 + m * 16 + half * 8 + g8;
            const bool ok = r < rows_all && half < HR;
            const int4 *p = reinterpret_cast<const int4 *>(
                a.q + (((int64_t)(sq.node0 + (ok ? r / G : 0)) * g.n_kv + head) * G + (ok ? r % G : 0)) * D + 16 * t4);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                const int4 v = ok ? p[ks] : make_int4(0, 0, 0, 0);
                const float u = Q_UNIT;
                qf[m][ks][half] = pack_half2((float)v.x * u, (float)v.y * u);
                qf[m][ks][half + 2] = pack_half2((float)v.z * u, (float)v.w * u);
            }
        }

    // copies of tile j of this CTA into the ring slot of this warp's n-th tile
    auto issue = [&](int n) {
        const int j = warp + n * NW;
        if (j >= n_tiles) return;
        const int p0 = lo + j * FEW_TILE, rows16 = (min(FEW_TILE, hi - p0) + 15) & ~15;
        const uint32_t bar = bars + (n % STAGES) * 8, dst = ring + (n % STAGES) * stage;
        const bool held = (int)blockIdx.x == a.hold_cta && j == a.hold_tile;
        if (lane == 0) bar_expect(bar, rows16 * (kbytes + vbytes + 4) + (held ? 16 : 0));
        __syncwarp();
        // one lane per run of rows inside a page; pages hold a multiple of 16 rows
        int at = 0;
        for (int k = 0; at < rows16; ++k) {
            const int p = p0 + at, in = row_in_page(g, p), n_rows = min(rows16 - at, g.P - in);
            if (lane == k) {
                const uint8_t *reg = a.pool + region_off(g, a.table[(int64_t)sq.seq * g.max_pages + page_of(g, p)], head);
                copy_bulk(dst + at * kbytes, reg + (int64_t)in * kbytes, n_rows * kbytes, bar);
                copy_bulk(dst + FEW_TILE * kbytes + at * vbytes, reg + vplane_off(g) + (int64_t)in * vbytes,
                          n_rows * vbytes, bar);
                copy_bulk(dst + FEW_TILE * (kbytes + vbytes) + at * 4, reg + nplane_off(g) + (int64_t)in * 4,
                          n_rows * 4, bar);
            }
            at += n_rows;
        }
    };

    float acc[MT][HALF ? 4 : 8][4], m_ref[MT][2], l[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int c = 0; c < (HALF ? 4 : 8); ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][c][i] = 0.0f;
        m_ref[m][0] = m_ref[m][1] = NONE;
        l[m][0] = l[m][1] = 0.0f;
    }
    // this warp's norms of a tile: 16 tokens' (key, value) in each 128 bytes
    uint8_t *norms = sm + L::NORMS_AT + warp * 512;
    const uint32_t lane4 = lane * 4, value8 = 128 + lane % 16 * 8;
    bool lost = false;
    int issued = 0;
    for (; issued < STAGES - 1; ++issued) issue(issued);
    int n = 0;
    for (int j = warp; j < n_tiles; j += NW, ++n) {
        __syncwarp();                                 // every lane has read the slot's previous tile
        issue(issued++);
        // the lanes poll one by one: the warp gives up as one, as what follows
        // takes all of its lanes
        if (__any_sync(FULL, !bar_wait(bars + (n % STAGES) * 8, (n / STAGES) & 1, a.poll_limit))) {
            lost = true;
            break;
        }
        const uint8_t *st = sm + (ring - sm0) + (n % STAGES) * stage;
        const uint8_t *sv = st + FEW_TILE * kbytes, *sn = sv + FEW_TILE * vbytes;
        // the tile's norms as floats, once
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int tok = lane + 32 * i;
            const uint32_t w = *reinterpret_cast<const uint32_t *>(sn + tok * 4);
            *reinterpret_cast<float2 *>(norms + tok * 8) =
                make_float2(norm_value(w & 0xffffu, NORM_UNIT) * a.score_unit, norm_value(w >> 16, NORM_UNIT));
        }
        __syncwarp();
        const int p0 = lo + j * FEW_TILE;
        auto step = [&](int s16, auto masked) {
            constexpr bool M = decltype(masked)::value;
            // keys: fragment column g8 of token group nt is token s16 + 8 nt + g8
            uint32_t kf[2][4][2];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const int tok = s16 + nt * 8 + g8;
                if constexpr (KB == 4) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(st + tok * 32 + t4 * 8);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        kf[nt][i / 2][i % 2] =
                            *reinterpret_cast<const uint32_t *>(sm + entry_at(i < 4 ? w.x : w.y, i & 3, lane4));
                } else if constexpr (KB == 3) {
                    const uint16_t *p = reinterpret_cast<const uint16_t *>(st + tok * 24 + t4 * 6);
                    const uint64_t w = (uint64_t)p[0] | (uint64_t)p[1] << 16 | (uint64_t)p[2] << 32;
                    const uint32_t lut = sm0 + lane * 4;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        kf[nt][i / 2][i % 2] = load_shared(lut + ((uint32_t)(w >> (6 * i)) & 63u) * 128u);
                } else {
                    const uint8_t *row = st + tok * kbytes;
                    const uint16_t *tab = reinterpret_cast<const uint16_t *>(sm);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        kf[nt][i / 2][i % 2] =
                            (uint32_t)tab[code_at_bytes(row, 16 * t4 + 2 * i, g.kb, kbytes)] |
                            (uint32_t)tab[code_at_bytes(row, 16 * t4 + 2 * i + 1, g.kb, kbytes)] << 16;
                }
            }
            [[maybe_unused]] uint32_t pf[MT][4], pt[2];
            if constexpr (HALF) {
                // tokens are the rows (g8, g8 + 8), queries the columns (2 t4, 2 t4 + 1)
                const float *nr = reinterpret_cast<const float *>(norms + s16 * 8 + g8 * 8);
                const float2 n0 = *reinterpret_cast<const float2 *>(nr), n1 = *reinterpret_cast<const float2 *>(nr + 16);
                float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {
                    const uint32_t k[4] = {kf[0][ks][0], kf[1][ks][0], kf[0][ks][1], kf[1][ks][1]};
                    mma16816(s, k, qf[0][ks][0], qf[0][ks][2]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] *= i < 2 ? n0.x : n1.x;
                if (M) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int node = min((row0 + 2 * t4 + (i & 1)) / G, sq.nodes - 1);
                        const uint64_t *mk = a.mask + (int64_t)(sq.node0 + node) * a.words;
                        const int p = p0 + s16 + (i / 2) * 8 + g8, d = p - sq.context;
                        if (!(p < hi && (d < 0 || ((mk[d >> 6] >> (d & 63)) & 1)))) s[i] = -INFINITY;
                    }
                }
                const float mx[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
                bool over = false;
#pragma unroll
                for (int q = 0; q < 2; ++q) over |= mx[q] > m_ref[0][q] + LAG;      // never for -inf
                if (__any_sync(FULL, over)) {
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        float now = fmaxf(m_ref[0][q], mx[q]);
#pragma unroll
                        for (int o = 4; o < 32; o *= 2) now = fmaxf(now, __shfl_xor_sync(FULL, now, o));
                        const float f = ex2(m_ref[0][q] - now);
                        m_ref[0][q] = now;
                        l[0][q] *= f;
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc[0][c][q] *= f, acc[0][c][2 + q] *= f;
                    }
                }
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = ex2(s[i] - m_ref[0][i & 1]);
                    l[0][i & 1] += e[i];
                }
                pt[0] = transpose8(pack_half2(e[0] * n0.y, e[1] * n0.y));
                pt[1] = transpose8(pack_half2(e[2] * n1.y, e[3] * n1.y));
            } else {
                // norms of the fragment's tokens: columns 2 t4, 2 t4 + 1 of both groups
                float kn[4], vn[4];
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    const float4 w = *reinterpret_cast<const float4 *>(norms + s16 * 8 + (nt * 8 + 2 * t4) * 8);
                    kn[2 * nt] = w.x, vn[2 * nt] = w.y, kn[2 * nt + 1] = w.z, vn[2 * nt + 1] = w.w;
                }
                float s[MT][2][4];
                float top = -INFINITY;                    // largest excess over the running maximum
#pragma unroll
                for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[m][nt][i] = 0.0f;
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) mma16816(s[m][nt], qf[m][ks], kf[nt][ks][0], kf[nt][ks][1]);
#pragma unroll
                        for (int i = 0; i < 2 * HR; ++i) s[m][nt][i] *= kn[2 * nt + (i & 1)];
                    }
                }
                if (M) {
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int half = 0; half < HR; ++half) {
                            const int node = min((row0 + m * 16 + half * 8 + g8) / G, sq.nodes - 1);
                            const uint64_t *mk = a.mask + (int64_t)(sq.node0 + node) * a.words;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int p = p0 + s16 + (i / 2) * 8 + 2 * t4 + (i & 1), d = p - sq.context;
                                const bool see = p < hi && (d < 0 || ((mk[d >> 6] >> (d & 63)) & 1));
                                if (!see) s[m][i / 2][half * 2 + (i & 1)] = -INFINITY;
                            }
                        }
                }
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int half = 0; half < HR; ++half) {
                        const float mx = fmaxf(fmaxf(s[m][0][half * 2], s[m][0][half * 2 + 1]),
                                               fmaxf(s[m][1][half * 2], s[m][1][half * 2 + 1]));
                        top = fmaxf(top, mx - m_ref[m][half]);
                    }
                if (__any_sync(FULL, top > LAG)) {
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int half = 0; half < HR; ++half) {
                            float mx = fmaxf(fmaxf(s[m][0][half * 2], s[m][0][half * 2 + 1]),
                                             fmaxf(s[m][1][half * 2], s[m][1][half * 2 + 1]));
                            mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 1));
                            mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, 2));
                            const float now = fmaxf(m_ref[m][half], mx);
                            const float f = ex2(m_ref[m][half] - now);
                            m_ref[m][half] = now;
                            l[m][half] *= f;
#pragma unroll
                            for (int c = 0; c < 8; ++c) {
                                acc[m][c][half * 2] *= f;
                                acc[m][c][half * 2 + 1] *= f;
                            }
                        }
                }
#pragma unroll
                for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int nt = 0; nt < 2; ++nt) {
                            if (half >= HR) {
                                pf[m][nt * 2 + half] = 0;
                                continue;
                            }
                            const float e0 = ex2(s[m][nt][half * 2] - m_ref[m][half]), e1 = ex2(s[m][nt][half * 2 + 1] - m_ref[m][half]);
                            l[m][half] += e0 + e1;
                            pf[m][nt * 2 + half] = pack_half2(e0 * vn[2 * nt], e1 * vn[2 * nt + 1]);
                        }
                }
            }
            // channel group c's two value registers: an operand's columns, or (HALF) every
            // second time half its rows
            [[maybe_unused]] uint32_t even[2] = {0u, 0u};
            auto add_values = [&](int c, const uint32_t (&b)[2]) {
                if constexpr (HALF) {
                    if (c & 1) {
                        const uint32_t v[4] = {even[0], b[0], even[1], b[1]};
                        mma16816(acc[0][c / 2], v, pt[0], pt[1]);
                    } else {
                        even[0] = b[0], even[1] = b[1];
                    }
                } else {
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma16816(acc[m][c], pf[m], b[0], b[1]);
                }
            };
            // values: fragment rows (tokens) 2 t4, +1, +8, +9; column g8 of channel group c is channel 8 g8 + c
            if constexpr (VB == 2) {
                // a byte of z: the codes of two channels of a token (low half)
                // and of the next one (high half), an entry of both channels' pairs
                uint32_t z[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t x[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int tok = s16 + 2 * t4 + k + i * 8;
                        x[k] = __byte_perm(*reinterpret_cast<const uint16_t *>(sv + tok * 16 + g8 * 2), 0, 0x4140);
                        x[k] = (x[k] | x[k] << 4) & 0x0f0f0f0fu;
                    }
                    z[i] = x[1] * 16 + x[0];
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint2 v0 = *reinterpret_cast<const uint2 *>(sm + entry_at(z[0], k, value8));
                    const uint2 v1 = *reinterpret_cast<const uint2 *>(sm + entry_at(z[1], k, value8));
                    add_values(2 * k, {v0.x, v1.x});
                    add_values(2 * k + 1, {v0.y, v1.y});
                }
            } else if constexpr (VB == 3) {
                uint32_t x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = s16 + 2 * t4 + (i & 1) + (i >> 1) * 8, at = tok * 24 + g8 * 3;
                    const uint32_t *p = reinterpret_cast<const uint32_t *>(sv + (at & ~3));
                    x[i] = __funnelshift_r(p[0], p[1], 8 * (at & 3));
                }
                const uint32_t lut = sm0 + L::KLUT + lane * 4;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t b[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t idx = ((x[2 * i] >> (3 * c)) & 7u) | (((x[2 * i + 1] >> (3 * c)) & 7u) << 3);
                        b[i] = load_shared(lut + idx * 128u);
                    }
                    add_values(c, b);
                }
            } else {
                const uint16_t *tab = reinterpret_cast<const uint16_t *>(sm) + 256;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t b[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint8_t *row = sv + (s16 + 2 * t4 + 8 * i) * vbytes;
                        b[i] = (uint32_t)tab[code_at_bytes(row, 8 * g8 + c, g.vb, vbytes)] |
                               (uint32_t)tab[code_at_bytes(row + vbytes, 8 * g8 + c, g.vb, vbytes)] << 16;
                    }
                    add_values(c, b);
                }
            }
        };
        // a tile inside the context is whole (hi - lo is a multiple of it) and needs no mask
        if (p0 + FEW_TILE <= sq.context) {
#pragma unroll 1
            for (int s16 = 0; s16 < FEW_TILE; s16 += 16) step(s16, std::false_type());
        } else {
#pragma unroll 1
            for (int s16 = 0; s16 < min(FEW_TILE, hi - p0); s16 += 16) step(s16, std::true_type());
        }
    }
    if (lost) {
        // report it, and let the copies in flight land before the CTA goes
        if (lane == 0) atomicOr(a.status, ST_TIMEOUT);
        for (int k = n; k < issued; ++k)
            if (warp + k * NW < n_tiles) bar_wait(bars + (k % STAGES) * 8, (k / STAGES) & 1, a.poll_limit);
    }

    // join the warps: each row's maximum, then the scaled sums
    __syncthreads();
    float *jacc = reinterpret_cast<float *>(sm + L::stages_at(NW)), *jml = jacc + NW * R * 64;
    if constexpr (HALF) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float sum = l[0][q];
#pragma unroll
            for (int o = 4; o < 32; o *= 2) sum += __shfl_xor_sync(FULL, sum, o);
            const int r = 2 * t4 + q;
            if (g8 == 0) jml[(warp * R + r) * 2] = m_ref[0][q] > NONE ? m_ref[0][q] : -INFINITY, jml[(warp * R + r) * 2 + 1] = sum;
#pragma unroll
            for (int c = 0; c < 4; ++c)              // rows g8, g8 + 8 are channels 8 g8 + 2 c, + 1
                *reinterpret_cast<float2 *>(jacc + (warp * R + r) * 64 + 8 * g8 + 2 * c) =
                    make_float2(acc[0][c][q], acc[0][c][2 + q]);
        }
    } else {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int half = 0; half < HR; ++half) {
                float sum = l[m][half];
                sum += __shfl_xor_sync(FULL, sum, 1);
                sum += __shfl_xor_sync(FULL, sum, 2);
                const int r = m * 16 + half * 8 + g8;
                if (t4 == 0) jml[(warp * R + r) * 2] = m_ref[m][half] > NONE ? m_ref[m][half] : -INFINITY, jml[(warp * R + r) * 2 + 1] = sum;
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    // columns 2 t4, 2 t4 + 1 are channels 16 t4 + c and 16 t4 + 8 + c
                    jacc[(warp * R + r) * 64 + 16 * t4 + c] = acc[m][c][half * 2];
                    jacc[(warp * R + r) * 64 + 16 * t4 + 8 + c] = acc[m][c][half * 2 + 1];
                }
            }
    }
    __syncthreads();
    constexpr int ROWS = HALF ? 8 : R;
    const int used = min(NW, n_tiles);
    for (int i = tid; i < ROWS * 16; i += NW * 32) {
        const int r = i / 16, c4 = i % 16;
        if (row0 + r >= rows_all) continue;
        float M = -INFINITY;
        for (int w = 0; w < used; ++w) M = fmaxf(M, jml[(w * R + r) * 2]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.0f;
        if (M > -INFINITY)
            for (int w = 0; w < used; ++w) {
                const float f = ex2(jml[(w * R + r) * 2] - M);
                const float4 v = reinterpret_cast<const float4 *>(jacc)[(w * R + r) * 16 + c4];
                o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
                sum += f * jml[(w * R + r) * 2 + 1];
            }
        if (sq.splits == 1) {
            const float inv = sum > 0.0f ? a.out_unit / sum : 0.0f;   // a row that sees nothing is zero
            const int node = (row0 + r) / G, qh = (row0 + r) % G;
            __nv_bfloat162 *dst = reinterpret_cast<__nv_bfloat162 *>(
                a.out + (((int64_t)(sq.node0 + node) * g.n_kv + head) * G + qh) * D + c4 * 4);
            dst[0] = __floats2bfloat162_rn(o.x * inv, o.y * inv);
            dst[1] = __floats2bfloat162_rn(o.z * inv, o.w * inv);
        } else {
            const int64_t at = (int64_t)blockIdx.x * a.row_tiles_rows + r;
            reinterpret_cast<float4 *>(a.acc)[at * 16 + c4] = o;
            if (c4 == 0) a.ml[at * 2] = M, a.ml[at * 2 + 1] = sum;
        }
    }
}

// ---------------------------------------------------------------------------
// many rows: tcgen05
// ---------------------------------------------------------------------------
//
// One CTA an SM. Its four decode warps turn 128 cached rows at a time into
// fp16 key and value tiles in shared memory (a thread a row, norms applied);
// one warp issues the products S = Q K^T and O += P V on the tensor cores, and
// two groups of four warps (a stream each) turn S into P, a thread a query
// row. S, P and O stay in tensor memory: 128 + 64 + 64 columns for each
// stream, all 512.
//
// The two streams keep the exponentials (the bound: 16 a clock and SM) busy
// while the other's products run. With more than 128 query rows they are two
// row tiles that share every decoded tile (ROWS); with fewer, one row tile
// whose KV tiles they take in turn, joined when the CTA is done with it.
//
// The work is the list of KV tiles of all (sequence, KV head, row group)
// items, cut into equal runs, one for each CTA; a CTA walks its run's
// segments. An item that lies in one run is written at once, the others'
// parts are joined by k_tree_join: at most two partial slots a CTA.
//
// 64 nodes on each of 16 sequences of 32,768 tokens (8 KV heads of 4 query
// heads: 256 rows an item, 275 GFLOP) take 416 us, 0.66 PFLOP/s: 239 us of it
// are the exponentials (XU pipe 66 % busy), the rest the waits of a stream
// whose next scores are not there yet. A third score buffer would fill them,
// but tensor memory has no columns left.

constexpr int MANY_TILE = 128, MANY_STAGES = 3;
constexpr int MANY_THREADS = 13 * 32;
constexpr int MANY_LUT = 65536, MANY_KV = MANY_TILE * 128;
constexpr int MANY_Q_AT = MANY_LUT, MANY_K_AT = MANY_Q_AT + 2 * MANY_KV, MANY_V_AT = MANY_K_AT + MANY_STAGES * MANY_KV;
// each decode warp's ring of packed rows: 32 rows of 52 bytes a slot (both widths)
constexpr int MANY_RING = 4, MANY_SLOT = 32 * 52;
constexpr int MANY_ML_AT = MANY_V_AT + MANY_STAGES * MANY_KV;
constexpr int MANY_RING_AT = MANY_ML_AT + 128 * 2 * 4;
constexpr int MANY_BARS_AT = MANY_RING_AT + 4 * MANY_RING * MANY_SLOT;
constexpr int MANY_SMEM = MANY_BARS_AT + 320;

// Tile t of the run list -> its CTA, for `tiles` tiles in `ctas` equal runs.
__host__ __device__ __forceinline__ int run_of(int64_t t, int64_t tiles, int ctas) {
    return (int)(((t + 1) * ctas - 1) / tiles);
}
__host__ __device__ __forceinline__ int64_t run_start(int c, int64_t tiles, int ctas) { return c * tiles / ctas; }

// One CTA's part of one item.
struct Segment {
    int seq, head, row0, lo, hi;             // KV tiles [lo, hi) of the item
    int slot;                                // partial slot, -1: the whole item
};

// The segment that starts at tile t (< end) of the run.
__device__ __forceinline__ Segment segment_at(const TreeSeq *seqs, int n_seqs, const Geo &g, int rows, int64_t t,
                                              int64_t end, int cta, int64_t *next) {
    const int b = find_seq<false>(seqs, n_seqs, (int)t);
    const TreeSeq &sq = seqs[b];
    const int tiles = (sq.context + sq.nodes + MANY_TILE - 1) / MANY_TILE;
    const int rts = (sq.nodes * g.H + rows - 1) / rows;
    const int local = (int)t - sq.unit0, item = local / tiles;
    Segment s;
    s.seq = b;
    s.head = item / rts;
    s.row0 = (item % rts) * rows;
    s.lo = local - item * tiles;
    s.hi = (int)min((int64_t)tiles, s.lo + (end - t));
    s.slot = s.lo ? 2 * cta : s.hi < tiles ? 2 * cta + 1 : -1;
    *next = t + (s.hi - s.lo);
    return s;
}

// True in one lane of the (whole) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p;
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

#define TC_R32(r)                                                                                                  \
    "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),     \
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),      \
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),     \
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
#define TC_IN16(r, o)                                                                                              \
    "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]),            \
        "r"(r[o + 7]), "r"(r[o + 8]), "r"(r[o + 9]), "r"(r[o + 10]), "r"(r[o + 11]), "r"(r[o + 12]),                \
        "r"(r[o + 13]), "r"(r[o + 14]), "r"(r[o + 15])

// 32 columns of this warp's 32 lanes (thread: its lane's)
__device__ __forceinline__ void tc_load32(uint32_t (&r)[32], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
                 "%27,%28,%29,%30,%31}, [%32];"
                 : TC_R32(r)
                 : "r"(at)
                 : "memory");
}
#define TC_IO32(r)                                                                                                 \
    "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),     \
        "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),      \
        "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),     \
        "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
// The loads before it are done; the registers pass through it, so that no use
// of theirs can be moved ahead of it.
__device__ __forceinline__ void tc_wait_load(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : TC_IO32(r)::"memory");
}
__device__ __forceinline__ void tc_load16(uint32_t (&r)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tc_wait_load(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::
                     "memory");
}
__device__ __forceinline__ void tc_store8(uint32_t at, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tc_store16(uint32_t at, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
                 TC_IN16(r, 0)
                 : "memory");
}

// A shared-memory operand in 8-row groups of 1,024 bytes, 128-byte rows with
// the 128-byte swizzle: 64 fp16 of the inner dimension a row.
__device__ __forceinline__ uint64_t tc_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
// fp16 x fp16 -> fp32, M = 128; B's rows are N (K-major) or K (MN-major)
__host__ __device__ constexpr uint32_t tc_idesc(int n, bool b_mn) {
    return 1u << 4 | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n / 8) << 17 | (uint32_t)(128 / 16) << 24;
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}

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

// One stream's softmax of a tile, a thread a row of 128 columns.
template <bool MASKED>
__device__ __forceinline__ void hide(uint32_t (&x)[32], const uint64_t *mk, int nodes, int d) {
    if (!MASKED) return;
    const uint32_t see = seen32(mk, nodes, d);
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] = (see >> j) & 1 ? x[j] : 0xff800000u;
}
__device__ __forceinline__ float largest(const uint32_t (&x)[32], float m) {
    float m1 = __uint_as_float(x[0]);
#pragma unroll
    for (int j = 1; j < 32; j += 2) {
        m = fmaxf(m, __uint_as_float(x[j]));
        if (j + 1 < 32) m1 = fmaxf(m1, __uint_as_float(x[j + 1]));
    }
    return fmaxf(m, m1);
}
__device__ __forceinline__ uint64_t pair64(uint32_t lo, uint32_t hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float2 split64(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}

// P = exp2(S - ref) in fp16, sum = its row sum in fp32; true if some row of
// the warp exceeds its ref by more than LAG (P and sum are then not valid).
// p_free() waits until the product that reads the last P is complete.
template <bool MASKED, typename F>
__device__ __forceinline__ bool weigh(uint32_t S, uint32_t P, float ref, float &sum, const uint64_t *mk, int nodes,
                                      int d, F &&p_free) {
    // P carries a factor of 2^7 (as sum does): with LAG it stays below 2^15, and
    // fp16 keeps weights down to 2^-31 of the maximum
    const float sub = (ref > -INFINITY ? -ref : 0.0f) + 7.0f;
    const uint64_t sub2 = pair64(__float_as_uint(sub), __float_as_uint(sub));
    uint32_t x[2][16];
    uint64_t acc[2] = {0, 0};
    float top = -INFINITY, top1 = -INFINITY;
    tc_load16(x[0], S);
    tc_wait_load(x[0]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        uint32_t(&y)[16] = x[c & 1];
        if (c < 7) tc_load16(x[(c + 1) & 1], S + 16 * (c + 1));
        if (MASKED) {
            const uint32_t see = seen32(mk, nodes, d + 16 * c);
#pragma unroll
            for (int j = 0; j < 16; ++j) y[j] = (see >> j) & 1 ? y[j] : 0xff800000u;
        }
        uint32_t p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            top = fmaxf(top, __uint_as_float(y[2 * j]));
            top1 = fmaxf(top1, __uint_as_float(y[2 * j + 1]));
            const float2 v = split64(add_pair(pair64(y[2 * j], y[2 * j + 1]), sub2));
            const float e0 = ex2(v.x), e1 = ex2(v.y);
            acc[j & 1] = add_pair(acc[j & 1], pair64(__float_as_uint(e0), __float_as_uint(e1)));
            p[j] = pack_half2(e0, e1);
        }
        if (c == 0 && !p_free()) {
            tc_wait_load(x[1]);
            return false;
        }
        tc_store8(P + 8 * c, p);
        if (c < 7) tc_wait_load(x[(c + 1) & 1]);
    }
    top = fmaxf(top, top1);
    const float2 v = split64(add_pair(acc[0], acc[1]));
    sum = v.x + v.y;
    return __any_sync(FULL, top > ref + LAG);
}

// Moves ref up to the row's maximum and scales the sums so far to it.
template <bool MASKED>
__device__ __noinline__ void raise(uint32_t S, uint32_t O, bool scale, float &ref, float &l, const uint64_t *mk,
                                   int nodes, int d) {
    float now = ref;
    uint32_t x[32];
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        tc_load32(x, S + 32 * c);
        tc_wait_load(x);
        hide<MASKED>(x, mk, nodes, d + 32 * c);
        now = largest(x, now);
    }
    const float f = now > -INFINITY ? ex2(ref - now) : 1.0f;
    ref = now;
    l *= f;
    if (scale) {
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
            tc_load32(x, O + 32 * c);
            tc_wait_load(x);
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = __float_as_uint(__uint_as_float(x[j]) * f);
            tc_store16(O + 32 * c, x);
            tc_store16(O + 32 * c + 16, x + 16);
        }
    }
    tc_wait_st();
}

// half2 x (hi + lo): a 16-bit norm needs two halves to be exact
__device__ __forceinline__ uint32_t scale_half2(uint32_t x, __half2 hi, __half2 lo) {
    const __half2 v = *reinterpret_cast<const __half2 *>(&x);
    const __half2 r = __hfma2(v, hi, __hmul2(v, lo));
    return *reinterpret_cast<const uint32_t *>(&r);
}

template <int KB, int VB, bool ROWS, class Src>
__global__ void __launch_bounds__(MANY_THREADS, 1) k_tree_many(Geo g, TreeArgs a, int64_t all_tiles,
                                                               const __grid_constant__ Src src) {
    constexpr int RU = ROWS ? 256 : 128;             // query rows of an item
    // the tiles' swizzle needs 1,024-byte alignment; an address that is a
    // constant keeps the products' operands in uniform registers
    extern __shared__ __align__(1024) uint8_t many_smem[];
    uint8_t *const sm = many_smem;
    const uint32_t sm0 = smem_u32(sm);
    const int tid = threadIdx.x, warp = __shfl_sync(FULL, tid / 32, 0), lane = tid % 32;
    // barriers: full[3] empty[3] s_ready[2] p_ready[2] q_ready seg_done o_free m_full m_empty fin, the 16 of the rings
    // and pv_done[2]; then the TMEM address
    const uint32_t bars = sm0 + MANY_BARS_AT;
    auto full = [&](int i) { return bars + 8 * i; };
    auto empty = [&](int i) { return bars + 24 + 8 * i; };
    auto s_ready = [&](int i) { return bars + 48 + 8 * i; };
    auto p_ready = [&](int i) { return bars + 64 + 8 * i; };
    const uint32_t q_ready = bars + 80, seg_done = bars + 88, o_free = bars + 96, m_full = bars + 104,
                   m_empty = bars + 112, fin = bars + 120;
    auto row_bar = [&](int w, int slot) { return bars + 128 + 8 * (w * MANY_RING + slot); };
    volatile uint32_t *tmem_at = reinterpret_cast<uint32_t *>(sm + MANY_BARS_AT + 272);
    auto pv_done = [&](int i) { return bars + 256 + 8 * i; };

    // the codes' tables, an entry of 256 bytes: 32 lanes' copies of a key pair, then of a value pair
    const float cunit = exp2f((float)-g.centroid_frac);
    {
        float *cent = reinterpret_cast<float *>(sm + MANY_K_AT);
        if (tid < (1 << KB)) cent[tid] = (float)a.tb->k_cent[tid] * cunit;
        if (tid >= 32 && tid < 32 + (1 << VB)) cent[tid] = (float)a.tb->v_cent[tid - 32] * cunit;
        __syncthreads();
        for (int e = warp; e < (1 << (2 * KB)); e += MANY_THREADS / 32)
            reinterpret_cast<uint32_t *>(sm)[e * 64 + lane] = pack_half2(cent[e & ((1 << KB) - 1)], cent[e >> KB]);
        for (int e = warp; e < (1 << (2 * VB)); e += MANY_THREADS / 32)
            reinterpret_cast<uint32_t *>(sm)[e * 64 + 32 + lane] =
                pack_half2(cent[32 + (e & ((1 << VB) - 1))], cent[32 + (e >> VB)]);
    }
    if (tid == 0) {
        for (int i = 0; i < MANY_STAGES; ++i) bar_init(full(i), 4), bar_init(empty(i), 1);
        for (int i = 0; i < 2; ++i) bar_init(s_ready(i), 1), bar_init(p_ready(i), 4), bar_init(pv_done(i), 1);
        bar_init(q_ready, 8), bar_init(seg_done, 1), bar_init(o_free, 8);
        bar_init(m_full, 4), bar_init(m_empty, 4), bar_init(fin, 1);
        for (int i = 0; i < 4 * MANY_RING; ++i) bar_init(row_bar(0, i), 1);
        bar_init_fence();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32((void *)tmem_at))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    wait_prior_grid();
    __syncthreads();
    tc_fence_after();
    // All 512 columns are this CTA's, so they start at address 0 (a constant, for
    // the same reason).
    constexpr uint32_t tmem = 0;
    if (*tmem_at != tmem || (sm0 & 1023)) {                  // never: reported, not worked around
        if (tid == 0) atomicOr(a.status, ST_INTERNAL);
        __syncthreads();
        if (warp == 12)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(*tmem_at) : "memory");
        return;
    }
    // of stream i: S at 256 i, P at 256 i + 128, O at 256 i + 192

    const TreeSeq *seqs = reinterpret_cast<const TreeSeq *>(src.data());
    const int cta = blockIdx.x;
    int64_t t = run_start(cta, all_tiles, gridDim.x);
    const int64_t end = run_start(cta + 1, all_tiles, gridDim.x);
    bool lost = false;                               // a wait gave up: the same for all lanes that wait together
    auto wait = [&](uint32_t bar, int phase) {
        if (!lost && !bar_wait(bar, (uint32_t)phase & 1u, a.poll_limit)) {
            lost = true;
            atomicOr(a.status, ST_TIMEOUT);
        }
        lost = __any_sync(FULL, lost);
    };

    if (warp >= 8 && warp < 12) {
        // ---- decode: thread `row` owns row `row` of each tile, a warp 32 of them
        const int row = tid - 256;
        const uint32_t lane4 = lane * 4;
        const uint32_t ring = sm0 + MANY_RING_AT + (warp - 8) * MANY_RING * MANY_SLOT;
        int kt = 0, kr = 0;                                      // tiles so far; the ring slot of the segment's first
        // of ring slot i, bit i: the parity that its next wait is for; whether copies into it are on their way
        uint32_t uses = 0, coming = 0;
        for (int seg = 0; t < end && !lost; ++seg) {
            int64_t next;
            const Segment s = segment_at(seqs, a.n_seqs, g, RU, t, end, cta, &next);
            const TreeSeq sq = seqs[s.seq];
            const int len = sq.context + sq.nodes, kt0 = kt;
            constexpr int KV4 = KB * 2, VV4 = VB * 2;            // 32-bit words of a row's codes
            const int32_t *pages = a.table + (int64_t)sq.seq * g.max_pages;
            // Bulk copies of this warp's 32 rows of tile s.lo + k, in the runs
            // that pages leave: two at most, as pages hold a multiple of 16
            // rows; lane 0 copies the first, lane 1 the second. A run's page is
            // looked up one tile ahead.
            int page = 0;
            auto look_up = [&](int k) {
                const int p0 = (s.lo + k) * MANY_TILE + (warp - 8) * 32;
                const int p = p0 + (lane ? g.P - row_in_page(g, p0) : 0);
                if (lane < 2 && s.lo + k < s.hi && p < min(len, p0 + 32)) page = pages[page_of(g, p)];
            };
            auto issue = [&](int k) {
                const int p0 = (s.lo + k) * MANY_TILE + (warp - 8) * 32;
                if (s.lo + k >= s.hi || p0 >= len) return;
                const int slot = (kr + k) % MANY_RING, rows16 = (min(32, len - p0) + 15) & ~15;
                const uint32_t bar = row_bar(warp - 8, slot), dst = ring + slot * MANY_SLOT;
                const bool held = cta == a.hold_cta && kt0 + k == a.hold_tile && warp == 8;
                if (lane == 0) bar_expect(bar, rows16 * (8 * KB + 8 * VB + 4) + (held ? 16 : 0));
                coming |= 1u << slot;
                __syncwarp();
                const int in0 = row_in_page(g, p0), first = min(rows16, g.P - in0);
                const int at = lane ? first : 0, n = lane ? rows16 - first : first, in = lane ? 0 : in0;
                if (lane < 2 && n) {
                    const uint8_t *reg = a.pool + region_off(g, page, s.head);
                    copy_bulk(dst + at * 8 * KB, reg + (int64_t)in * (8 * KB), n * 8 * KB, bar);
                    copy_bulk(dst + 32 * 8 * KB + at * 8 * VB, reg + vplane_off(g) + (int64_t)in * (8 * VB), n * 8 * VB,
                              bar);
                    copy_bulk(dst + 32 * 8 * (KB + VB) + at * 4, reg + nplane_off(g) + (int64_t)in * 4, n * 4, bar);
                }
                look_up(k + 1);
            };
            look_up(0);
            for (int k = 0; k < MANY_RING - 1; ++k) issue(k);
            for (int k = 0; k < s.hi - s.lo && !lost; ++k, ++kt) {
                uint32_t ck[KV4], cv[VV4], cn = 0;
                const bool live = (s.lo + k) * MANY_TILE + row < len;
                __syncwarp();                                    // the slot's last rows have been read
                issue(k + MANY_RING - 1);
                if ((s.lo + k) * MANY_TILE + (warp - 8) * 32 < len) {
                    const int slot = (kr + k) % MANY_RING;
                    wait(row_bar(warp - 8, slot), uses >> slot);
                    if (!lost) uses ^= 1u << slot, coming ^= 1u << slot;
                    const uint8_t *st = sm + (ring - sm0) + slot * MANY_SLOT;
                    const uint8_t *pk = st + lane * 8 * KB, *pv = st + 32 * 8 * KB + lane * 8 * VB;
#pragma unroll
                    for (int i = 0; i < KV4; i += 2)
                        *reinterpret_cast<uint2 *>(ck + i) = *reinterpret_cast<const uint2 *>(pk + 4 * i);
#pragma unroll
                    for (int i = 0; i < VV4; i += 2)
                        *reinterpret_cast<uint2 *>(cv + i) = *reinterpret_cast<const uint2 *>(pv + 4 * i);
                    cn = *reinterpret_cast<const uint32_t *>(st + 32 * 8 * (KB + VB) + lane * 4);
                } else {
#pragma unroll
                    for (int i = 0; i < KV4; ++i) ck[i] = 0;
#pragma unroll
                    for (int i = 0; i < VV4; ++i) cv[i] = 0;
                }
                cn = live ? cn : 0;                              // past the end: a zero norm makes a zero row
                const int st = kt % MANY_STAGES;
                if (kt >= MANY_STAGES) wait(empty(st), kt / MANY_STAGES - 1);
                const float kn = norm_value(cn & 0xffffu, NORM_UNIT) * a.k_scale, vn = norm_value(cn >> 16, NORM_UNIT);
                auto codes = [&](const uint32_t *w, int bits, int j) -> uint32_t {   // pair j's entry, this lane's copy
                    if (bits == 4) return entry_at(w[j / 4], j % 4, lane4);
                    if (bits == 2) return entry_at((j & 1 ? w[j / 8] >> 4 : w[j / 8]) & 0x0f0f0f0fu, j % 8 / 2, lane4);
                    const int at = 2 * bits * j, i = at / 32, sh = at % 32;
                    const uint32_t x = sh + 2 * bits <= 32 ? w[i] >> sh : __funnelshift_r(w[i], w[i + 1], sh);
                    return (x & ((1u << (2 * bits)) - 1u)) << 8 | lane4;
                };
                auto put = [&](int base, const uint32_t *w, int bits, int off, float nrm) {
                    const __half2 hi = __float2half2_rn(nrm);
                    const __half2 lo = __float2half2_rn(nrm - __low2float(hi));
#pragma unroll
                    for (int c = 0; c < 8; c += 4) {
                        uint32_t v[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            v[j] = *reinterpret_cast<const uint32_t *>(sm + off + codes(w, bits, 4 * c + j));
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) v[4 * k + j] = scale_half2(v[4 * k + j], hi, lo);
                            *reinterpret_cast<uint4 *>(sm + base + st * MANY_KV + row * 128 +
                                                       (((c + k) ^ (row & 7)) * 16)) =
                                make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                        }
                    }
                };
                put(MANY_K_AT, ck, KB, 0, kn);
                put(MANY_V_AT, cv, VB, 128, vn);
                fence_async();
                __syncwarp();
                if (lane == 0) bar_arrive(full(st));
            }
            kr = (kr + s.hi - s.lo) % MANY_RING;
            t = next;
        }
        // copies that a lost wait left in flight land before the CTA goes
        if (lost)
            for (int i = 0; i < MANY_RING; ++i)
                if (coming >> i & 1u) bar_wait(row_bar(warp - 8, i), uses >> i & 1u, a.poll_limit);
    } else if (warp == 12) {
        // ---- this warp issues every product. All lanes walk the same steps
        // (so that operands stay in uniform registers: with one lane inside a
        // branch each product cost some 60 clocks of register moves), and one
        // elected lane issues.
        constexpr uint32_t iqk = tc_idesc(128, false), ipv = tc_idesc(64, true);
        int st_qk = 0, st_pv = 0, np[2] = {0, 0};     // stages of the next score product and the next value product
        int use = 0;                                  // rounds of the stages so far
        const uint64_t q_desc = tc_desc(sm0 + MANY_Q_AT), k_desc = tc_desc(sm0 + MANY_K_AT),
                       v_desc = tc_desc(sm0 + MANY_V_AT);
        for (int seg = 0; t < end && !lost; ++seg) {
            int64_t next;
            const Segment s = segment_at(seqs, a.n_seqs, g, RU, t, end, cta, &next);
            const int tiles = __shfl_sync(FULL, s.hi - s.lo, 0), steps = ROWS ? 2 * tiles : tiles;
            auto scores = [&](int step) {
                const int i = step & 1;
                if (!ROWS || i == 0) wait(full(st_qk), use);
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t q = q_desc + (ROWS ? i * (MANY_KV >> 4) : 0), k = k_desc + st_qk * (MANY_KV >> 4);
#pragma unroll
                    for (int x = 0; x < 4; ++x) tc_mma_ss(tmem + 256 * i, q + 2 * x, k + 2 * x, iqk, x > 0);
                    tc_commit(s_ready(i));
                }
                __syncwarp();
                if (!ROWS || i == 1) {
                    st_qk = st_qk == MANY_STAGES - 1 ? 0 : st_qk + 1;
                    use += st_qk == 0;
                }
            };
            wait(q_ready, seg);
            if (seg) wait(o_free, seg - 1);
            for (int step = 0; step < min(2, steps) && !lost; ++step) scores(step);
            for (int step = 0; step < steps && !lost; ++step) {
                const int i = step & 1;
                wait(p_ready(i), i ? np[1]++ : np[0]++);
                if (lost) break;
                // the stream's next scores first: S is read, P waits for pv_done
                if (step + 2 < steps) scores(step + 2);
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t v = v_desc + st_pv * (MANY_KV >> 4);
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        tc_mma_ts(tmem + 256 * i + 192, tmem + 256 * i + 128 + 8 * x, v + 128 * x, ipv,
                                  step >= 2 || x > 0);
                    if (!ROWS || i == 1) tc_commit(empty(st_pv));
                    tc_commit(pv_done(i));
                }
                __syncwarp();
                if (!ROWS || i == 1) st_pv = st_pv == MANY_STAGES - 1 ? 0 : st_pv + 1;
            }
            if (elect_one()) tc_commit(seg_done);
            __syncwarp();
            t = next;
        }
        // nothing may be in flight when the tensor memory goes
        if (elect_one()) tc_commit(fin);
        __syncwarp();
        if (!bar_wait(fin, 0, WAIT_POLLS)) atomicOr(a.status, ST_TIMEOUT);
        __syncwarp();
    } else {
        // ---- softmax: thread `row` of stream `i` owns one query row
        const int i = warp / 4, row = tid - 128 * i;
        const uint32_t lanes = (uint32_t)(warp % 4) << 21;   // lane 32 (warp % 4), in bits 16 up
        const uint32_t S = tmem + lanes + 256 * i, P = S + 128, O = S + 192;
        int ns = 0, nv = 0;                                  // score and value products waited for
        for (int seg = 0; t < end && !lost; ++seg) {
            int64_t next;
            const Segment s = segment_at(seqs, a.n_seqs, g, RU, t, end, cta, &next);
            const TreeSeq sq = seqs[s.seq];
            const int rows_all = sq.nodes * g.H, qr = s.row0 + (ROWS ? 128 * i : 0) + row;
            const bool any_row = qr - lane < rows_all;       // of this warp's 32
            const int node = min(qr / g.H, sq.nodes - 1);
            const uint64_t *mk = a.mask + (int64_t)(sq.node0 + node) * a.words;
            const int tiles = s.hi - s.lo, steps = ROWS ? tiles : (tiles + 1 - i) / 2;
            // The queries, in log2 units: this stream's row tile, whose products
            // are done, or (!ROWS) half of the one tile, once both streams' are.
            if (!ROWS && seg) wait(seg_done, seg - 1);
            {
                const float u = Q_UNIT * a.q_scale;
#pragma unroll
                for (int x = 0; x < (ROWS ? 8 : 4); ++x) {
                    const int at = (ROWS ? 1024 * i + row + 128 * x : tid + 256 * x), r = at / 8, c = at % 8;
                    const int q = s.row0 + r;
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (q < rows_all) {
                        const int4 *p = reinterpret_cast<const int4 *>(
                            a.q + (((int64_t)(sq.node0 + q / g.H) * g.n_kv + s.head) * g.H + q % g.H) * D + 8 * c);
                        const int4 y = p[0], z = p[1];
                        w = make_uint4(pack_half2((float)y.x * u, (float)y.y * u), pack_half2((float)y.z * u, (float)y.w * u),
                                       pack_half2((float)z.x * u, (float)z.y * u), pack_half2((float)z.z * u, (float)z.w * u));
                    }
                    *reinterpret_cast<uint4 *>(sm + MANY_Q_AT + r * 128 + ((c ^ (r & 7)) * 16)) = w;
                }
                fence_async();
                __syncwarp();
                if (lane == 0) bar_arrive(q_ready);
            }
            float ref = -INFINITY, l = 0.0f;
            for (int n = 0; n < steps && !lost; ++n) {
                const int t0 = (s.lo + (ROWS ? n : 2 * n + i)) * MANY_TILE;
                wait(s_ready(i), ns++);
                if (lost) break;
                tc_fence_after();
                // P and O are this stream's again once its last value product is done
                bool have = n == 0;
                auto p_free = [&] {
                    if (!have) wait(pv_done(i), nv++);
                    have = true;
                    return !lost;
                };
                if (any_row) {
                    float sum = 0.0f;
                    auto step = [&](auto masked) {
                        constexpr bool M = decltype(masked)::value;
                        // the exponentials are taken under the maximum so far, and
                        // again in the rare case that it was too low
                        bool over = true;
                        if (n > 0) over = weigh<M>(S, P, ref, sum, mk, sq.nodes, t0 - sq.context, p_free);
                        if (over && !lost) {
                            raise<M>(S, O, n > 0, ref, l, mk, sq.nodes, t0 - sq.context);
                            weigh<M>(S, P, ref, sum, mk, sq.nodes, t0 - sq.context, p_free);
                        }
                    };
                    if (t0 + MANY_TILE <= sq.context) step(std::false_type());
                    else step(std::true_type());
                    l += sum;
                    tc_wait_st();
                } else {
                    p_free();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(p_ready(i));
            }
            if (steps) wait(pv_done(i), nv++);
            tc_fence_after();
            if (lost) break;
            // this row's sums out
            float *ml = reinterpret_cast<float *>(sm + MANY_ML_AT);
            float *hand = reinterpret_cast<float *>(sm + MANY_Q_AT + MANY_KV);   // !ROWS: the second query tile is free
            float f0 = 1.0f, f1 = 0.0f, m = ref;
            const bool mine = ROWS || i == 0;
            if (!ROWS && i == 1) ml[row * 2] = ref, ml[row * 2 + 1] = l;
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                uint32_t x[32];
                if (steps) {
                    tc_load32(x, O + 32 * c);
                    tc_wait_load(x);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = 0;
                }
                if (!ROWS) {
                    const int turn = 2 * seg + c;
                    if (i == 1) {
                        if (turn) wait(m_empty, turn - 1);
                        if (lost) break;
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<uint4 *>(hand + row * 32 + ((j / 4 ^ (row & 7)) * 4)) =
                                make_uint4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                        __syncwarp();
                        if (lane == 0) bar_arrive(m_full);
                        continue;
                    }
                    wait(m_full, turn);
                    if (lost) break;
                    if (c == 0) {
                        const float m1 = ml[row * 2], l1 = ml[row * 2 + 1];
                        m = fmaxf(ref, m1);
                        f0 = m > -INFINITY ? ex2(ref - m) : 0.0f;
                        f1 = m > -INFINITY ? ex2(m1 - m) : 0.0f;
                        l = l * f0 + l1 * f1;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 y = *reinterpret_cast<const float4 *>(hand + row * 32 + ((j / 4 ^ (row & 7)) * 4));
                        const float z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            // a stream without weight may hold anything
                            const float u0 = f0 > 0.0f ? f0 * __uint_as_float(x[j + k]) : 0.0f;
                            x[j + k] = __float_as_uint(f1 > 0.0f ? fmaf(f1, z[k], u0) : u0);
                        }
                    }
                    __syncwarp();
                    if (lane == 0) bar_arrive(m_empty);
                }
                if (!mine || qr >= rows_all) continue;
                if (s.slot < 0) {
                    const float inv = l > 0.0f ? a.out_unit / l : 0.0f;
                    uint4 *dst = reinterpret_cast<uint4 *>(
                        a.out + (((int64_t)(sq.node0 + qr / g.H) * g.n_kv + s.head) * g.H + qr % g.H) * D + 32 * c);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(x[8 * j + 2 * k]) * inv,
                                                                           __uint_as_float(x[8 * j + 2 * k + 1]) * inv);
                            w[k] = *reinterpret_cast<const uint32_t *>(&v);
                        }
                        dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
                    const int64_t at = (int64_t)s.slot * RU + (ROWS ? 128 * i : 0) + row;
                    uint4 *dst = reinterpret_cast<uint4 *>(a.acc + at * 64 + 32 * c);
#pragma unroll
                    for (int j = 0; j < 8; ++j) dst[j] = make_uint4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
                    if (c == 0) a.ml[at * 2] = m, a.ml[at * 2 + 1] = l;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(o_free);
            t = next;
        }
    }
    __syncthreads();
    if (warp == 12)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ---------------------------------------------------------------------------
// joining the splits of a row tile
// ---------------------------------------------------------------------------

// One CTA per 8 rows of a (sequence, row tile, KV head): the parts' sums,
// scaled to the largest of their maxima, added in order and divided by the sum
// of weights. Bound by the parts' bytes, at few items by how many CTAs read
// them (one CTA an item took 100 us where 8 items had 19 parts of 256 rows).
// Rows are `R` a tile. MANY: the parts are the runs (of `ctas` over
// `all_tiles`) that the item's KV tiles lie in, else the item's splits.
template <bool MANY, class Src>
__global__ void __launch_bounds__(128) k_tree_join(Geo g, TreeArgs a, int32_t R, int64_t all_tiles, int32_t ctas,
                                                   const __grid_constant__ Src src) {
    extern __shared__ float wt[];                    // [8][splits]
    wait_prior_grid();
    const TreeSeq *seqs = reinterpret_cast<const TreeSeq *>(src.data());
    const int per = R / 8, part8 = blockIdx.x % per * 8;
    const TreeSeq sq = seqs[find_seq<true>(seqs, a.n_seqs, blockIdx.x / per)];
    const int G = g.H, rows_all = sq.nodes * G, tiles = (rows_all + R - 1) / R;
    const int group = blockIdx.x / per - sq.group0;
    const int head = MANY ? group / tiles : group % g.n_kv, rt = MANY ? group % tiles : group / g.n_kv;
    const int row0 = rt * R + part8, rows = min(8, rows_all - row0);
    int run0 = 0, splits = sq.splits;
    if (MANY) {
        const int kv = (sq.context + sq.nodes + MANY_TILE - 1) / MANY_TILE;
        const int64_t first = sq.unit0 + (int64_t)group * kv;
        run0 = run_of(first, all_tiles, ctas);
        splits = run_of(first + kv - 1, all_tiles, ctas) - run0 + 1;
    }
    if (splits == 1 || rows <= 0) return;
    auto slot = [&](int split, int r) {
        if (MANY) return ((int64_t)2 * (run0 + split) + (split == 0)) * R + part8 + r;
        return ((int64_t)sq.unit0 + ((int64_t)split * tiles + rt) * g.n_kv + head) * R + part8 + r;
    };
    for (int r = threadIdx.x / 32; r < rows; r += 4) {
        const int lane = threadIdx.x % 32;
        float M = -INFINITY, sum = 0.0f;
        for (int s = lane; s < splits; s += 32) M = fmaxf(M, a.ml[slot(s, r) * 2]);
        for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(FULL, M, o));
        for (int s = lane; s < splits; s += 32) {
            const float f = M > -INFINITY ? ex2(a.ml[slot(s, r) * 2] - M) : 0.0f;
            sum += f * a.ml[slot(s, r) * 2 + 1];
            wt[r * splits + s] = f;
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
        const float inv = sum > 0.0f ? a.out_unit / sum : 0.0f;
        for (int s = lane; s < splits; s += 32) wt[r * splits + s] *= inv;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * 16; i += 128) {
        const int r = i / 16, c4 = i % 16;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int s = 0; s < splits; ++s) {
            const float f = wt[r * splits + s];
            const float4 v = reinterpret_cast<const float4 *>(a.acc)[slot(s, r) * 16 + c4];
            o.x += f * v.x, o.y += f * v.y, o.z += f * v.z, o.w += f * v.w;
        }
        const int node = (row0 + r) / G, qh = (row0 + r) % G;
        __nv_bfloat162 *dst = reinterpret_cast<__nv_bfloat162 *>(
            a.out + (((int64_t)(sq.node0 + node) * g.n_kv + head) * G + qh) * D + c4 * 4);
        dst[0] = __floats2bfloat162_rn(o.x, o.y);
        dst[1] = __floats2bfloat162_rn(o.z, o.w);
    }
}

namespace {

// Above MANY_FROM query rows of a KV head the tcgen05 kernel takes over; up to
// MANY_SURE rows only where each SM has more than MANY_TILES of its KV tiles
// to do, as its start costs more (fewer units of work, tensor memory, the
// join of 128-row slots) and its tiles less. Measured, 8 KV heads of 4 query
// heads, 4b/2b, k_tree_few against k_tree_many: 9 nodes (36 rows) of one
// sequence, 2,304 tokens (1 tile an SM) 22.0 : 21.7 us, 18,800 (8) 27.1 : 28.8,
// 65,536 (28) 53.0 : 51.2, 131,072 (55) 88.1 : 83.3, 16 sequences of 32,768
// (222) 365 : 280; 16 nodes (64 rows) 20.3 : 18.1, 27.1 : 29.6, 52.9 : 52.1,
// 88.5 : 84.4, 376 : 287; 3b/3b, 6 sequences to 9,001 tokens (about 20), 16
// nodes 45.4 : 37.0. Above
// 64 rows k_tree_few decodes each row three times and more.
constexpr int MANY_FROM = 32, MANY_SURE = 64, MANY_TILES = 12;
// Its keys (centroid times norm, below 2^4 times 2^6) can take a factor of up
// to 2^5 of the scores' before they leave fp16; beyond, k_tree_few.
constexpr int MANY_SHIFT = 5;
int score_shift(const Geo &g) { return 16 + 9 - g.qk_frac - g.norm_frac; }

// How a call is cut: rows a tile, tokens a split, and what that takes.
struct TreePlan {
    int rows = 16;
    bool many = false;                       // k_tree_many's runs, else k_tree_few's units
    int64_t chunk = FEW_TILE, units = 0, groups = 0;
    int ctas = 0;                            // many: runs
    int max_splits = 1;
    std::vector<TreeSeq> seqs;
    int64_t slots() const { return many ? 2 * (int64_t)ctas : units; }
    size_t acc_bytes() const {
        return max_splits > 1 ? (size_t)slots() * rows * (64 + 2) * sizeof(float) : 0;
    }
};

int make_plan(const CacheBase *c, int32_t B, const int32_t *seq, const int32_t *nodes, int sms, TreePlan &p) {
    const Geo &g = c->g;
    int64_t most = 0, all = 0, total = 0;
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
            p.seqs.push_back(TreeSeq{seq[b], (int32_t)(len - nodes[b]), nodes[b], (int32_t)all, 1, 0, 0});
        all += nodes[b];
        most = std::max<int64_t>(most, (int64_t)nodes[b] * g.H);
    }
    if (all > INT32_MAX / (g.n_kv * g.H)) return fail(INS_EBADLEN, "too many nodes in one call");
    if (p.seqs.empty()) return INS_OK;
    const bool paired = ((g.kb == 4 && g.vb == 2) || (g.kb == 3 && g.vb == 3)) && score_shift(g) <= MANY_SHIFT;
    int64_t kv_tiles = 0;
    for (const TreeSeq &s : p.seqs) kv_tiles += g.n_kv * ((s.context + s.nodes + MANY_TILE - 1) / MANY_TILE);
    if (paired && (most > MANY_SURE || (most > MANY_FROM && kv_tiles > (int64_t)MANY_TILES * sms))) {
        p.many = true;
        // 256-row tiles share each decoded row between both streams: above 128
        // rows 122 us, with 128-row tiles 154 (64 nodes, 131,072 tokens); with
        // 128 rows or fewer one stream would idle, 88 : 105 us (32 nodes)
        p.rows = most > 128 ? 256 : 128;
        for (TreeSeq &s : p.seqs) {
            const int64_t rts = ((int64_t)s.nodes * g.H + p.rows - 1) / p.rows;
            s.unit0 = (int32_t)p.units;
            s.group0 = (int32_t)p.groups;
            p.groups += rts * g.n_kv;
            p.units += rts * g.n_kv * ((s.context + s.nodes + MANY_TILE - 1) / MANY_TILE);
            if (p.units > INT32_MAX) return fail(INS_EBADLEN, "too much work in one call");
        }
        p.ctas = (int)std::min<int64_t>(sms, p.units);
        for (const TreeSeq &s : p.seqs) {
            const int64_t kv = (s.context + s.nodes + MANY_TILE - 1) / MANY_TILE;
            const int64_t items = ((int64_t)s.nodes * g.H + p.rows - 1) / p.rows * g.n_kv;
            for (int64_t i = 0; i < items; ++i) {
                const int64_t first = s.unit0 + i * kv;
                p.max_splits = std::max(p.max_splits, run_of(first + kv - 1, p.units, p.ctas) -
                                                          run_of(first, p.units, p.ctas) + 1);
            }
        }
        return INS_OK;
    }
    // Rows a tile: two 16-row fragments share each decoded token where there
    // are more than 16 rows. At 16 rows (4 nodes, 131,072 tokens) one fragment
    // takes 38.9 us, two 54.0; at 17 to 32 one fragment would decode twice.
    p.rows = most > 16 ? 32 : 16;
    auto units_at = [&](int64_t chunk) {
        int64_t u = 0;
        for (const TreeSeq &s : p.seqs) {
            const int64_t tiles = ((int64_t)s.nodes * g.H + p.rows - 1) / p.rows;
            u += tiles * g.n_kv * ((s.context + s.nodes + chunk - 1) / chunk);
        }
        return u;
    };
    for (const TreeSeq &s : p.seqs) total += ((int64_t)s.nodes * g.H + p.rows - 1) / p.rows * g.n_kv * (s.context + s.nodes);
    // One CTA an SM. Where one split per item leaves SMs idle, the smallest
    // chunk whose units still fit one wave; else a quarter of an SM's share of
    // all tokens, so that the last wave's unevenness stays small.
    const int64_t least = 4 * FEW_TILE;
    int64_t chunk;
    if (units_at(INT32_MAX) <= sms) {
        int64_t lo = 1, hi = 1 << 25;                // in units of `least`
        while (lo < hi) {
            const int64_t mid = (lo + hi) / 2;
            if (units_at(mid * least) <= sms) hi = mid;
            else lo = mid + 1;
        }
        chunk = lo * least;
    } else {
        chunk = std::max<int64_t>(least, (total / (4 * sms) + least - 1) / least * least);
    }
    chunk = std::min<int64_t>(chunk, INT32_MAX - least);
    p.chunk = chunk;
    for (TreeSeq &s : p.seqs) {
        const int64_t tiles = ((int64_t)s.nodes * g.H + p.rows - 1) / p.rows;
        s.splits = (int32_t)(((int64_t)s.context + s.nodes + chunk - 1) / chunk);
        s.unit0 = (int32_t)p.units;
        s.group0 = (int32_t)p.groups;
        p.units += tiles * g.n_kv * s.splits;
        p.groups += tiles * g.n_kv;
        p.max_splits = std::max(p.max_splits, (int)s.splits);
        if (p.units > INT32_MAX) return fail(INS_EBADLEN, "too much work in one call");
    }
    return INS_OK;
}

int device_sms(int dev, int *sms) {
    CK(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    return INS_OK;
}

template <int KB, int VB, int MT, bool HALF, int NW>
int launch_few(CacheBase *c, const TreePlan &p, const Plan &plan, const TreeArgs &a, cudaStream_t s) {
    const size_t smem = FewLayout<KB, VB>::bytes(c->g, NW, 16 * MT);
    return plan.run(c, s, [&](const auto &src) -> cudaError_t {
        auto fn = k_tree_few<KB, VB, MT, HALF, NW, std::decay_t<decltype(src)>>;
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        *c->launches += 1;
        return launch_after(fn, (unsigned)p.units, NW * 32u, smem, s, c->g, a, src);
    });
}

template <int KB, int VB>
int launch_few_rows(CacheBase *c, const TreePlan &p, bool half, const Plan &plan, const TreeArgs &a, cudaStream_t s) {
    // Warps: five a scheduler where 96 registers hold their state (1 token of
    // 1M rows: 20 warps 139 us, 23 warps of 80 registers 143; 3b/3b 200, 211),
    // three where 32 rows take 168 (8 nodes of 1M: 12 warps 302 us, 14 spill:
    // 468). 8-bit rows make a stage 8.4 KB: 8 warps of them fit.
    constexpr int N1 = KB ? 20 : 8, N2 = KB ? 12 : 8;
    if (p.rows == 32) return launch_few<KB, VB, 2, false, N2>(c, p, plan, a, s);
    if (half) return launch_few<KB, VB, 1, true, N1>(c, p, plan, a, s);
    return launch_few<KB, VB, 1, false, N1>(c, p, plan, a, s);
}

template <int KB, int VB, bool ROWS>
int launch_many(CacheBase *c, const TreePlan &p, const Plan &plan, const TreeArgs &a, cudaStream_t s) {
    return plan.run(c, s, [&](const auto &src) -> cudaError_t {
        auto fn = k_tree_many<KB, VB, ROWS, std::decay_t<decltype(src)>>;
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, MANY_SMEM);
        if (e != cudaSuccess) return e;
        *c->launches += 1;
        return launch_after(fn, (unsigned)p.ctas, (unsigned)MANY_THREADS, (size_t)MANY_SMEM, s, c->g, a,
                            (int64_t)p.units, src);
    });
}

int tree_body(CacheBase *c, int32_t B, const int32_t *seq, const int32_t *nodes, const uint64_t *mask, int32_t words,
              const int32_t *q, void *out, void *workspace, int64_t workspace_bytes, int64_t *need, cudaStream_t s) {
    int sms = 0;
    if (int rc = device_sms(c->device, &sms)) return rc;
    TreePlan p;
    if (int rc = make_plan(c, B, seq, nodes, sms, p)) return rc;
    if (need) {
        *need = (int64_t)p.acc_bytes();
        return INS_OK;
    }
    if (p.seqs.empty()) return INS_OK;
    // centroids are fp16 in real units, times a norm in k_tree_many
    if (c->g.qk_frac < 0 || c->g.qk_frac > 31 || c->cent_max > 16.0 || (c->cent_max > 0.0 && c->cent_max < 1.0 / 256))
        return fail(INS_EINVAL, "tree scan: qk_frac in [0, 31] and a largest centroid in [2^-8, 2^4] are supported");
    for (const TreeSeq &t : p.seqs)
        if (t.nodes > 64 * words) return fail(INS_EINVAL, "the mask's words are too few for a tree's nodes");
    if (!mask || !q || !out) return fail(INS_EINVAL, "tree scan: NULL buffer");
    if (((uintptr_t)mask & 7u) || ((uintptr_t)q & 15u) || ((uintptr_t)out & 15u))
        return fail(INS_EINVAL, "tree scan: mask 8-byte, q and out 16-byte aligned");
    if ((int64_t)p.acc_bytes() > workspace_bytes || (p.acc_bytes() && (!workspace || ((uintptr_t)workspace & 15u))))
        return fail(INS_EINVAL, "tree scan: a 16-byte aligned workspace of " + std::to_string(p.acc_bytes()) +
                                    " bytes is needed");
    TreeArgs a{};
    a.tb = c->d_tables;
    a.pool = c->d_pool;
    a.table = c->d_page_table;
    a.q = q;
    a.mask = mask;
    a.out = static_cast<__nv_bfloat16 *>(out);
    a.acc = static_cast<float *>(workspace);
    a.ml = a.acc + (size_t)p.slots() * p.rows * 64;
    a.status = c->d_status;
    a.n_seqs = (int32_t)p.seqs.size();
    a.words = words;
    a.chunk = (int32_t)p.chunk;
    a.row_tiles_rows = p.rows;
    a.poll_limit = std::min(c->wait.poll_limit, WAIT_POLLS);
    a.hold_cta = c->wait.item;
    a.hold_tile = c->wait.chunk;
    a.score_unit = std::ldexp(1.0f, score_shift(c->g));
    a.q_scale = std::min(a.score_unit, 1.0f);
    a.k_scale = std::max(a.score_unit, 1.0f);
    a.out_unit = std::ldexp(1.0f, 9 - c->g.norm_frac);
    Plan plan;
    plan.add(p.seqs);
    // up to 8 rows the products are taken transposed: one node of 1,048,576
    // tokens 139 us, by the 16-row variant 185
    bool half = true;
    for (const TreeSeq &t : p.seqs) half &= t.nodes * c->g.H <= 8;
    const int kb = c->g.kb, vb = c->g.vb;
    const bool wide = p.rows == 256;
    const int rc = p.many && kb == 4    ? (wide ? launch_many<4, 2, true>(c, p, plan, a, s)
                                                : launch_many<4, 2, false>(c, p, plan, a, s))
                   : p.many             ? (wide ? launch_many<3, 3, true>(c, p, plan, a, s)
                                                : launch_many<3, 3, false>(c, p, plan, a, s))
                   : kb == 4 && vb == 2 ? launch_few_rows<4, 2>(c, p, half, plan, a, s)
                   : kb == 3 && vb == 3 ? launch_few_rows<3, 3>(c, p, half, plan, a, s)
                                        : launch_few_rows<0, 0>(c, p, half, plan, a, s);
    if (rc) return rc;
    if (p.max_splits == 1) return INS_OK;
    const size_t smem = (size_t)8 * p.max_splits * sizeof(float);
    return plan.run(c, s, [&](const auto &src) -> cudaError_t {
        using S = std::decay_t<decltype(src)>;
        auto fn = p.many ? k_tree_join<true, S> : k_tree_join<false, S>;
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        *c->launches += 1;
        return launch_after(fn, (unsigned)(p.groups * (p.rows / 8)), 128u, smem, s, c->g, a, (int32_t)p.rows, (int64_t)p.units,
                            (int32_t)p.ctas, src);
    });
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
