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
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "plan.cuh"

namespace ins {

constexpr int TREE_MAX_NODES = 256;          // drafted tokens of one sequence
constexpr float LOG2E = 1.4426950408889634f;

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
// Waits for the phase of `parity`, at most 2^22 polls (about a second);
// false: it gave up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < (1 << 22); ++i) {
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
// c += a b, one 16x8 tile of 16-wide products
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// A 16-bit norm's value (int16 / 2^norm_frac): 2^23 + x is a float's bits, so
// no integer conversion (which runs at an eighth of the rate) is needed.
__device__ __forceinline__ float norm_value(uint32_t x16, float unit) {
    return fmaf(__uint_as_float(0x4b000000u | (x16 ^ 0x8000u)), unit, -8421376.0f * unit);
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
// conflicts); 2-bit values are picked from two registers by byte permutes.
// Norms stay factored out: the key's scales the score, the value's the
// probability.
//
// The running maximum moves only when a score exceeds it by more than 2^8
// (LAG, in the exponent's base): until then exp2 stays below 256 and times a
// norm below 2^14, inside fp16's range, so a rescale of the accumulators is
// rare and the maximum needs no exchange of lanes at every step.

constexpr int FEW_TILE = 64, FEW_STAGES = 3;
constexpr float LAG = 8.0f;

template <int KB, int VB>
struct FewLayout {
    static constexpr bool PAIRS = KB != 0;                       // else one code at a time, any width
    static constexpr int K_ENTRIES = PAIRS ? 1 << (2 * KB) : 0;
    static constexpr int V_ENTRIES = PAIRS && VB > 2 ? 1 << (2 * VB) : 0;
    static constexpr int KLUT = K_ENTRIES * 128, VLUT = V_ENTRIES * 128, SINGLE = PAIRS ? 0 : 1024;
    static constexpr int STAGES_AT = KLUT + VLUT + SINGLE;
    __host__ __device__ static int stage_bytes(const Geo &g) { return FEW_TILE * (g.kbytes + g.vbytes + 4); }
    __host__ __device__ static int bars_at(const Geo &g, int warps) {
        return STAGES_AT + warps * FEW_STAGES * stage_bytes(g);
    }
    // the end-of-loop join reuses the stages: [warps][rows][64] floats, [warps][rows][2]
    __host__ static size_t bytes(const Geo &g, int warps, int rows) {
        const size_t loop = (size_t)bars_at(g, warps) + warps * FEW_STAGES * 8;
        const size_t join = (size_t)STAGES_AT + (size_t)warps * rows * (64 + 2) * 4;
        return std::max(loop, join);
    }
};

template <int KB, int VB, int MT, bool HALF, int NW, class Src>
__global__ void __launch_bounds__(NW * 32, 1) k_tree_few(Geo g, TreeArgs a, const __grid_constant__ Src src) {
    using L = FewLayout<KB, VB>;
    constexpr int R = 16 * MT;                       // rows of this CTA's tile
    constexpr int HR = HALF ? 1 : 2;                 // of a fragment's two row halves, those that hold queries
    extern __shared__ __align__(128) uint8_t sm[];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, t4 = lane % 4, g8 = lane / 4;
    const uint32_t sm0 = smem_u32(sm);
    const int kbytes = KB ? KB * 8 : g.kbytes, vbytes = VB ? VB * 8 : g.vbytes;
    const int stage = FEW_TILE * (kbytes + vbytes + 4);
    const uint32_t ring = sm0 + L::STAGES_AT + warp * FEW_STAGES * stage;
    const uint32_t bars = sm0 + L::bars_at(g, NW) + warp * FEW_STAGES * 8;

    // tables: constant, so filled before the wait for earlier launches
    const float cunit = exp2f((float)-g.centroid_frac);
    if (L::PAIRS) {
        for (int i = tid; i < L::K_ENTRIES * 32; i += NW * 32) {
            const int e = i / 32;
            reinterpret_cast<uint32_t *>(sm)[i] = pack_half2((float)a.tb->k_cent[e & ((1 << KB) - 1)] * cunit,
                                                             (float)a.tb->k_cent[e >> KB] * cunit);
        }
        for (int i = tid; i < L::V_ENTRIES * 32; i += NW * 32) {
            const int e = i / 32;
            reinterpret_cast<uint32_t *>(sm + L::KLUT)[i] = pack_half2(
                (float)a.tb->v_cent[e & ((1 << VB) - 1)] * cunit, (float)a.tb->v_cent[e >> VB] * cunit);
        }
    } else {
        __half *tab = reinterpret_cast<__half *>(sm);
        for (int i = tid; i < 512; i += NW * 32)
            tab[i] = __float2half_rn((float)(i < 256 ? a.tb->k_cent[i] : a.tb->v_cent[i - 256]) * cunit);
    }
    uint32_t v_lo = 0, v_hi = 0;                     // the four 2-bit value centroids' low and high bytes
    if (VB == 2)
        for (int i = 0; i < 4; ++i) {
            const uint32_t h = __half_as_ushort(__float2half_rn((float)a.tb->v_cent[i] * cunit));
            v_lo |= (h & 255u) << (8 * i);
            v_hi |= (h >> 8) << (8 * i);
        }
    if (lane == 0)
        for (int i = 0; i < FEW_STAGES; ++i) bar_init(bars + i * 8, 1);
    bar_init_fence();
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
                const float u = LOG2E * exp2f((float)-g.qk_frac);
                qf[m][ks][half] = pack_half2((float)v.x * u, (float)v.y * u);
                qf[m][ks][half + 2] = pack_half2((float)v.z * u, (float)v.w * u);
            }
        }

    // copies of tile j of this CTA into the ring slot of this warp's n-th tile
    auto issue = [&](int n) {
        const int j = warp + n * NW;
        if (j >= n_tiles) return;
        const int p0 = lo + j * FEW_TILE, rows16 = (min(FEW_TILE, hi - p0) + 15) & ~15;
        const uint32_t bar = bars + (n % FEW_STAGES) * 8, dst = ring + (n % FEW_STAGES) * stage;
        if (lane == 0) bar_expect(bar, rows16 * (kbytes + vbytes + 4));
        __syncwarp();
        // one lane per run of rows inside a page; pages hold a multiple of 16 rows
        int at = 0;
        for (int k = 0; at < rows16; ++k) {
            const int p = p0 + at, in = p % g.P, n_rows = min(rows16 - at, g.P - in);
            if (lane == k) {
                const uint8_t *reg = a.pool + region_off(g, a.table[(int64_t)sq.seq * g.max_pages + p / g.P], head);
                copy_bulk(dst + at * kbytes, reg + (int64_t)in * kbytes, n_rows * kbytes, bar);
                copy_bulk(dst + FEW_TILE * kbytes + at * vbytes, reg + vplane_off(g) + (int64_t)in * vbytes,
                          n_rows * vbytes, bar);
                copy_bulk(dst + FEW_TILE * (kbytes + vbytes) + at * 4, reg + nplane_off(g) + (int64_t)in * 4,
                          n_rows * 4, bar);
            }
            at += n_rows;
        }
    };

    float acc[MT][8][4], m_ref[MT][2], l[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int c = 0; c < 8; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][c][i] = 0.0f;
        m_ref[m][0] = m_ref[m][1] = -INFINITY;
        l[m][0] = l[m][1] = 0.0f;
    }
    const float nunit = exp2f((float)-g.norm_frac);
    bool lost = false;
    int issued = 0;
    for (; issued < FEW_STAGES - 1; ++issued) issue(issued);
    int n = 0;
    for (int j = warp; j < n_tiles; j += NW, ++n) {
        __syncwarp();                                 // every lane has read the slot's previous tile
        issue(issued++);
        if (!bar_wait(bars + (n % FEW_STAGES) * 8, (n / FEW_STAGES) & 1)) {
            lost = true;
            break;
        }
        const uint8_t *st = sm + (ring - sm0) + (n % FEW_STAGES) * stage;
        const uint8_t *sv = st + FEW_TILE * kbytes, *sn = sv + FEW_TILE * vbytes;
        const int p0 = lo + j * FEW_TILE, live = min(FEW_TILE, hi - p0);
        const bool masked = p0 + FEW_TILE > sq.context;
#pragma unroll 1
        for (int s16 = 0; s16 < live; s16 += 16) {
            // keys: fragment column g8 of token group nt is token s16 + 8 nt + g8
            uint32_t kf[2][4][2];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const int tok = s16 + nt * 8 + g8;
                if constexpr (KB == 4) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(st + tok * 32 + t4 * 8);
                    const uint32_t lut = sm0 + lane * 4;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t word = i < 4 ? w.x : w.y;
                        const int s = 8 * (i & 3);
                        const uint32_t off = (s < 7 ? word << (7 - s) : word >> (s - 7)) & 0x7f80u;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(kf[nt][i / 2][i % 2]) : "r"(lut + off));
                    }
                } else if constexpr (KB == 3) {
                    const uint16_t *p = reinterpret_cast<const uint16_t *>(st + tok * 24 + t4 * 6);
                    const uint64_t w = (uint64_t)p[0] | (uint64_t)p[1] << 16 | (uint64_t)p[2] << 32;
                    const uint32_t lut = sm0 + lane * 4;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        asm volatile("ld.shared.u32 %0, [%1];"
                                     : "=r"(kf[nt][i / 2][i % 2])
                                     : "r"(lut + ((uint32_t)(w >> (6 * i)) & 63u) * 128u));
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
            // norms of the fragment's tokens: columns 2 t4, 2 t4 + 1 of both groups
            float kn[4], vn[4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const uint2 w = *reinterpret_cast<const uint2 *>(sn + (s16 + nt * 8 + 2 * t4) * 4);
                kn[2 * nt] = norm_value(w.x & 0xffffu, nunit);
                vn[2 * nt] = norm_value(w.x >> 16, nunit);
                kn[2 * nt + 1] = norm_value(w.y & 0xffffu, nunit);
                vn[2 * nt + 1] = norm_value(w.y >> 16, nunit);
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
            if (masked) {
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
                    top = fmaxf(top, mx > -INFINITY ? mx - m_ref[m][half] : -INFINITY);
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
                        const float f = now > -INFINITY ? ex2(m_ref[m][half] - now) : 1.0f;
                        m_ref[m][half] = now;
                        l[m][half] *= f;
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            acc[m][c][half * 2] *= f;
                            acc[m][c][half * 2 + 1] *= f;
                        }
                    }
            }
            uint32_t pf[MT][4];
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
                        // a row that has seen nothing yet keeps -inf - 0, not -inf - (-inf)
                        const float ref = m_ref[m][half] > -INFINITY ? m_ref[m][half] : 0.0f;
                        const float e0 = ex2(s[m][nt][half * 2] - ref), e1 = ex2(s[m][nt][half * 2 + 1] - ref);
                        l[m][half] += e0 + e1;
                        pf[m][nt * 2 + half] = pack_half2(e0 * vn[2 * nt], e1 * vn[2 * nt + 1]);
                    }
            }
            // values: fragment rows (tokens) 2 t4, +1, +8, +9; column g8 of channel group c is channel 8 g8 + c
            if constexpr (VB == 2) {
                uint32_t e[4], o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int tok = s16 + 2 * t4 + (i & 1) + (i >> 1) * 8;
                    uint32_t x = *reinterpret_cast<const uint16_t *>(sv + tok * 16 + g8 * 2);
                    x = (x | x << 8) & 0x00ff00ffu;
                    x = (x | x << 4) & 0x0f0f0f0fu;       // a byte: the codes of channels 2i, 2i + 1
                    e[i] = x & 0x03030303u;
                    o[i] = (x >> 2) & 0x03030303u;
                }
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t b[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t pair = __byte_perm(c & 1 ? o[2 * i] : e[2 * i], c & 1 ? o[2 * i + 1] : e[2 * i + 1],
                                                          (c >> 1) | ((4 + (c >> 1)) << 4));
                        b[i] = __byte_perm(v_lo, v_hi, pair * 0x11u + 0x4040u);
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma16816(acc[m][c], pf[m], b[0], b[1]);
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
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(b[i]) : "r"(lut + idx * 128u));
                    }
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma16816(acc[m][c], pf[m], b[0], b[1]);
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
#pragma unroll
                    for (int m = 0; m < MT; ++m) mma16816(acc[m][c], pf[m], b[0], b[1]);
                }
            }
        }
    }
    if (lost) {
        // report it, and let the copies in flight land before the CTA goes
        if (lane == 0) atomicOr(a.status, ST_TIMEOUT);
        for (int k = n; k < issued; ++k)
            if (warp + k * NW < n_tiles) bar_wait(bars + (k % FEW_STAGES) * 8, (k / FEW_STAGES) & 1);
    }

    // join the warps: each row's maximum, then the scaled sums
    __syncthreads();
    float *jacc = reinterpret_cast<float *>(sm + L::STAGES_AT), *jml = jacc + NW * R * 64;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int half = 0; half < HR; ++half) {
            float sum = l[m][half];
            sum += __shfl_xor_sync(FULL, sum, 1);
            sum += __shfl_xor_sync(FULL, sum, 2);
            const int r = m * 16 + half * 8 + g8;
            if (t4 == 0) jml[(warp * R + r) * 2] = m_ref[m][half], jml[(warp * R + r) * 2 + 1] = sum;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                // columns 2 t4, 2 t4 + 1 are channels 16 t4 + c and 16 t4 + 8 + c
                jacc[(warp * R + r) * 64 + 16 * t4 + c] = acc[m][c][half * 2];
                jacc[(warp * R + r) * 64 + 16 * t4 + 8 + c] = acc[m][c][half * 2 + 1];
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
            const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;   // a row that sees nothing is zero
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
// joining the splits of a row tile
// ---------------------------------------------------------------------------

// One CTA per (sequence, row tile, KV head): the splits' partial sums, scaled
// to the largest of their maxima, added in order and divided by the sum of
// weights. Rows are `R` a tile.
template <class Src>
__global__ void __launch_bounds__(256) k_tree_join(Geo g, TreeArgs a, int32_t R, const __grid_constant__ Src src) {
    extern __shared__ float wt[];                    // [rows][splits]
    wait_prior_grid();
    const TreeSeq *seqs = reinterpret_cast<const TreeSeq *>(src.data());
    const TreeSeq sq = seqs[find_seq<true>(seqs, a.n_seqs, blockIdx.x)];
    if (sq.splits == 1) return;
    const int G = g.H, rows_all = sq.nodes * G, tiles = (rows_all + R - 1) / R;
    const int group = blockIdx.x - sq.group0, head = group % g.n_kv, rt = group / g.n_kv;
    const int row0 = rt * R, rows = min(R, rows_all - row0);
    auto slot = [&](int split, int r) {
        return ((int64_t)sq.unit0 + ((int64_t)split * tiles + rt) * g.n_kv + head) * R + r;
    };
    for (int r = threadIdx.x / 32; r < rows; r += 8) {
        const int lane = threadIdx.x % 32;
        float M = -INFINITY, sum = 0.0f;
        for (int s = lane; s < sq.splits; s += 32) M = fmaxf(M, a.ml[slot(s, r) * 2]);
        for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(FULL, M, o));
        for (int s = lane; s < sq.splits; s += 32) {
            const float f = M > -INFINITY ? ex2(a.ml[slot(s, r) * 2] - M) : 0.0f;
            sum += f * a.ml[slot(s, r) * 2 + 1];
            wt[r * sq.splits + s] = f;
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        for (int s = lane; s < sq.splits; s += 32) wt[r * sq.splits + s] *= inv;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * 16; i += 256) {
        const int r = i / 16, c4 = i % 16;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < sq.splits; ++s) {
            const float f = wt[r * sq.splits + s];
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

// How a call is cut: rows a tile, tokens a split, and what that takes.
struct TreePlan {
    int rows = 16, warps = 16;
    int64_t chunk = FEW_TILE, units = 0, groups = 0;
    int max_splits = 1;
    std::vector<TreeSeq> seqs;
    size_t acc_bytes() const {
        return max_splits > 1 ? (size_t)units * rows * (64 + 2) * sizeof(float) : 0;
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
    // rows a tile: two 16-row fragments share each decoded token where there are more than 16 rows
    p.rows = most > 16 ? 32 : 16;
    p.warps = p.rows == 16 ? 16 : 12;
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
    // 8-bit rows make a stage 8.4 KB: 8 warps of them fit
    constexpr int N1 = KB ? 16 : 8, N2 = KB ? 12 : 8;
    if (p.rows == 32) return launch_few<KB, VB, 2, false, N2>(c, p, plan, a, s);
    if (half) return launch_few<KB, VB, 1, true, N1>(c, p, plan, a, s);
    return launch_few<KB, VB, 1, false, N1>(c, p, plan, a, s);
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
    a.ml = a.acc + (size_t)p.units * p.rows * 64;
    a.status = c->d_status;
    a.n_seqs = (int32_t)p.seqs.size();
    a.words = words;
    a.chunk = (int32_t)p.chunk;
    a.row_tiles_rows = p.rows;
    Plan plan;
    plan.add(p.seqs);
    bool half = true;
    for (const TreeSeq &t : p.seqs) half &= t.nodes * c->g.H <= 8;
    const int kb = c->g.kb, vb = c->g.vb;
    const int rc = kb == 4 && vb == 2   ? launch_few_rows<4, 2>(c, p, half, plan, a, s)
                   : kb == 3 && vb == 3 ? launch_few_rows<3, 3>(c, p, half, plan, a, s)
                                        : launch_few_rows<0, 0>(c, p, half, plan, a, s);
    if (rc) return rc;
    if (p.max_splits == 1) return INS_OK;
    const size_t smem = (size_t)p.rows * p.max_splits * sizeof(float);
    return plan.run(c, s, [&](const auto &src) -> cudaError_t {
        auto fn = k_tree_join<std::decay_t<decltype(src)>>;
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        *c->launches += 1;
        return launch_after(fn, (unsigned)p.groups, 256u, smem, s, c->g, a, (int32_t)p.rows, src);
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
