// Cached rows read back as keys and values in floating point.
//
// A cached row holds y = R x of a key or value x, R a product of rounds
// H diag(signs) / 8 (H the 64 x 64 Hadamard matrix of signs, R orthogonal):
// codes and a norm, y ~ norm * centroid[code]. Read back is y itself, or x =
// diag(signs) H / 8 applied round after round, last round first. Sums are fp32,
// the result is rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "plan.cuh"

namespace ins {

// Rows [t0, t0 + n) of `seq`, at row `row` of the outputs; the span's tiles of
// 32 rows are tiles [tile, next span's tile).
struct DenseSpan {
    int32_t seq, t0, n, tile;
    int64_t row;
};

constexpr int DENSE_WARPS = 8, DENSE_THREADS = DENSE_WARPS * 32;

// Two floats at once (one instruction for both).
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b) {
    float2 r;
    asm("{ .reg .b64 x, y, m; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 m, {%6, %6}; "
        "fma.rn.f32x2 x, y, m, x; mov.b64 {%0, %1}, x; }"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(-1.0f));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float s) {
    float2 r;
    asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %4}; mul.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(s));
    return r;
}

// The butterfly's stages of distances FROM to 32 channels over a vector (v[i]:
// channels 2 i and 2 i + 1).
template <int FROM>
__device__ __forceinline__ void butterfly(float2 (&v)[32]) {
    if constexpr (FROM == 1) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = make_float2(v[i].x + v[i].y, v[i].x - v[i].y);
    }
#pragma unroll
    for (int h = FROM > 1 ? FROM / 2 : 1; h < 32; h *= 2)
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (!(i & h)) {
                const float2 x = v[i], y = v[i + h];
                v[i] = add2(x, y), v[i + h] = sub2(x, y);
            }
}

// Tables in shared memory that decode several codes at a time, and take the
// butterfly's first stages with them (TURN): of a width of 4 bits a byte's two
// channels, of 3 bits six bits' two, of 2 bits a byte's four. A copy for each
// lane that reads at the same time (16 of 8 bytes, 8 of 16), so that no two
// meet in a bank. At 4b/2b both tables' entries alternate, 256 bytes apart, so
// that one byte permute makes an address of a byte of codes. Other widths: a
// table of single centroids.
template <int BITS, int STRIDE>
struct DenseTable {
    static constexpr int ENTRIES = BITS == 4 ? 256 : BITS == 3 ? 64 : BITS == 2 ? 256 : 256;
    static constexpr int BYTES = BITS == 0 ? 1024 : ENTRIES * STRIDE;
    static constexpr int STAGES = BITS == 2 ? 2 : BITS ? 1 : 0;      // of the butterfly, if TURN
    static __device__ __forceinline__ void fill(uint8_t *sm, const int64_t *cent, int count, bool turn) {
        if constexpr (BITS == 0) {
            for (int i = threadIdx.x; i < count; i += DENSE_THREADS) reinterpret_cast<float *>(sm)[i] = (float)cent[i];
        } else {
            // one thread an entry's copy
            constexpr int W = BITS == 2 ? 4 : 2, COPIES = 32 / W;
            for (int i = threadIdx.x; i < ENTRIES * COPIES; i += DENSE_THREADS) {
                const int e = i / COPIES;
                float c[W];
#pragma unroll
                for (int k = 0; k < W; ++k) c[k] = (float)cent[e >> (BITS * k) & ((1 << BITS) - 1)];
                if (turn) {
#pragma unroll
                    for (int h = 1; h < W; h *= 2)
#pragma unroll
                        for (int k = 0; k < W; ++k)
                            if (!(k & h)) {
                                const float x = c[k], y = c[k + h];
                                c[k] = x + y, c[k + h] = x - y;
                            }
                }
                float *to = reinterpret_cast<float *>(sm + e * STRIDE) + i % COPIES * W;
#pragma unroll
                for (int k = 0; k < W; ++k) to[k] = c[k];
            }
        }
    }
};

// A row's codes, as 8-byte words from global memory.
template <int BITS>
struct DenseCodes {
    static constexpr int WORDS = BITS ? BITS : 8;
    uint2 w[WORDS];
    __device__ __forceinline__ void load(const uint8_t *row, int bits) {
        if constexpr (BITS == 4 || BITS == 2) {
#pragma unroll
            for (int i = 0; i < BITS / 2; ++i) {
                const uint4 x = __ldg(reinterpret_cast<const uint4 *>(row) + i);
                w[2 * i] = make_uint2(x.x, x.y), w[2 * i + 1] = make_uint2(x.z, x.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; ++i)
                if (BITS || i < bits) w[i] = __ldg(reinterpret_cast<const uint2 *>(row) + i);
        }
    }
    __device__ __forceinline__ uint32_t word(int i) const { return i & 1 ? w[i / 2].y : w[i / 2].x; }
    // `bits` bits from bit `at` on (both constants once unrolled)
    __device__ __forceinline__ uint32_t field(int at, int bits) const {
        const int i = at / 32, sh = at % 32;
        const uint32_t x = sh + bits <= 32 ? word(i) >> sh : __funnelshift_r(word(i), word(i + 1), sh);
        return x & ((1u << bits) - 1u);
    }
    template <int B>
    __device__ __forceinline__ void singles(const uint8_t *sm, float2 (&v)[32]) const {
        if constexpr (B <= WORDS) {
            const float *cent = reinterpret_cast<const float *>(sm);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = make_float2(cent[field(2 * i * B, B)], cent[field((2 * i + 1) * B, B)]);
        }
    }
    // byte `i` times 256, plus what is below 256
    __device__ __forceinline__ uint32_t entry(int i, uint32_t plus) const {
        return __byte_perm(word(i / 4), plus, 0x5504 | i % 4 << 4);
    }
    __device__ __forceinline__ void decode(const uint8_t *sm, int bits, int lane, float2 (&v)[32]) const {
        if constexpr (BITS == 2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float4 x = *reinterpret_cast<const float4 *>(sm + entry(i, 128 + lane % 8 * 16));
                v[2 * i] = make_float2(x.x, x.y), v[2 * i + 1] = make_float2(x.z, x.w);
            }
        } else if constexpr (BITS == 4) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = *reinterpret_cast<const float2 *>(sm + entry(i, lane % 16 * 8));
        } else if constexpr (BITS != 0) {
            const uint8_t *mine = sm + lane % 16 * 8;
#pragma unroll
            for (int i = 0; i < 32; ++i)
                v[i] = *reinterpret_cast<const float2 *>(mine + field(2 * BITS * i, 2 * BITS) * 128);
        } else {
            switch (bits) {
                case 1: singles<1>(sm, v); break;
                case 2: singles<2>(sm, v); break;
                case 3: singles<3>(sm, v); break;
                case 4: singles<4>(sm, v); break;
                case 5: singles<5>(sm, v); break;
                case 6: singles<6>(sm, v); break;
                case 7: singles<7>(sm, v); break;
                default: singles<8>(sm, v); break;
            }
        }
    }
};

__device__ __forceinline__ uint32_t dense_pair(float2 x, __half *) {
    const __half2 h = __floats2half2_rn(x.x, x.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t dense_pair(float2 x, __nv_bfloat16 *) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x.x, x.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

template <int KB, int VB>
struct DenseLayout {
    static constexpr bool BOTH = KB == 4 && VB == 2;
    static constexpr int STRIDE = BOTH ? 256 : 128;
    static constexpr int K_BYTES = DenseTable<KB, STRIDE>::BYTES;
    // (at 4b/2b the values' entries begin at byte 128 of the keys', which their addresses add)
    static constexpr int V_AT = BOTH ? 128 : K_BYTES;
    static constexpr int SIGNS_AT = K_BYTES + (BOTH ? 0 : DenseTable<VB, STRIDE>::BYTES);
    static constexpr int STAGE_AT = SIGNS_AT + 256;
};

// A warp takes 32 rows of a KV head, a thread a row, in turn with the next
// task's codes already on their way. A thread holds its whole vector, so the
// butterfly needs no exchange (four threads a vector, with exchanges and single
// codes, took 115 us where this takes 67); the finished vectors go through shared
// memory (rows padded by 16 bytes) so that eight lanes write each 128 bytes.
//
// 52 bytes read and 256 or 512 written a row and head: 131,072 rows of 8 heads
// (4b/2b) in bf16 take 69 us, 4.7 TB/s, in fp32 124 to 128, 4.7 TB/s. Bound by L1 (81 %
// busy, most of it shared memory: table entries, the vectors' stage) and by its
// latency, which 15 warps an SM do not cover; 1,054 instructions a warp's 32 rows
// fill half of the issue slots.
template <int KB, int VB, typename T, class Src>
__global__ void __launch_bounds__(DENSE_THREADS, sizeof(T) == 4 ? 1 : 2)
    k_dense(Geo g, const DevTables *__restrict__ tb, const uint8_t *__restrict__ pool,
            const int32_t *__restrict__ table, T *__restrict__ k, T *__restrict__ v, int32_t n_spans, int64_t tasks,
            int32_t rounds, float unit, const __grid_constant__ Src src) {
    using L = DenseLayout<KB, VB>;
    using KT = DenseTable<KB, L::STRIDE>;
    using VT = DenseTable<VB, L::STRIDE>;
    constexpr int LINE = D * (int)sizeof(T) + 16;
    extern __shared__ __align__(128) uint8_t sm[];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
    uint8_t *const stage = sm + L::STAGE_AT + warp * 32 * LINE;
    KT::fill(sm, tb->k_cent, 1 << g.kb, rounds > 0);
    VT::fill(sm + L::V_AT, tb->v_cent, 1 << g.vb, rounds > 0);
    // the last signs, as the sign bits of a vector's words of type T
    uint32_t *const signs = reinterpret_cast<uint32_t *>(sm + L::SIGNS_AT);
    if (tid < 64) {
        const uint64_t m = rounds > 0 ? tb->sign_mask[0] : 0;
        if (sizeof(T) == 4) signs[tid] = (uint32_t)(m >> tid & 1) << 31;
        else if (tid < 32) signs[tid] = (uint32_t)(m >> (2 * tid) & 1) << 15 | (uint32_t)(m >> (2 * tid + 1) & 1) << 31;
    }
    wait_prior_grid();
    __syncthreads();
    const DenseSpan *spans = reinterpret_cast<const DenseSpan *>(src.data());
    // a task's rows: `n` of them, the first at row `row` of the outputs
    struct Task {
        int64_t row;
        int32_t n, head;
    };
    DenseCodes<KB> kc;
    DenseCodes<VB> vc;
    uint32_t norms = 0;
    auto load = [&](int64_t task) {
        Task t{0, 0, 0};
        if (task >= tasks) return t;
        const int tile = (int)(task / g.n_kv);
        t.head = (int)(task - (int64_t)tile * g.n_kv);
        int lo = 0, hi = n_spans - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (spans[mid].tile <= tile) lo = mid;
            else hi = mid - 1;
        }
        const DenseSpan sp = spans[lo];
        const int r0 = (tile - sp.tile) * 32;
        t.n = min(32, sp.n - r0);
        t.row = sp.row + r0;
        const int p = sp.t0 + r0 + min(lane, t.n - 1);
        const int page = g.p_log2 >= 0 ? p >> g.p_log2 : p / g.P, in = p - page * g.P;
        const uint8_t *region = pool + region_off(g, table[(int64_t)sp.seq * g.max_pages + page], t.head);
        kc.load(region + (int64_t)in * g.kbytes, g.kb);
        vc.load(region + vplane_off(g) + (int64_t)in * g.vbytes, g.vb);
        norms = __ldg(reinterpret_cast<const uint32_t *>(region + nplane_off(g)) + in);
        return t;
    };
    const int64_t stride = (int64_t)gridDim.x * DENSE_WARPS;
    int64_t task = (int64_t)blockIdx.x * DENSE_WARPS + warp;
    Task t = load(task);
    while (task < tasks) {
        const float ks = (float)(int16_t)(norms & 0xffffu) * unit, vs = (float)(int16_t)(norms >> 16) * unit;
        const Task now = t;
        auto finish = [&](float2 (&z)[32], auto stages, float scale, T *dst) {
            constexpr int DONE = decltype(stages)::value;
            for (int rd = rounds - 1; rd >= 0; --rd) {
                if (rd == rounds - 1) butterfly<1 << DONE>(z);
                else butterfly<1>(z);
                if (rd == 0) break;                              // the last signs go on after the rounding
                const uint64_t m = tb->sign_mask[rd];
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    z[i] = make_float2(m >> (2 * i) & 1 ? -z[i].x : z[i].x, m >> (2 * i + 1) & 1 ? -z[i].y : z[i].y);
            }
            __syncwarp();                                        // the stage's last vectors have been read
            uint32_t *to = reinterpret_cast<uint32_t *>(stage + lane * LINE);
            const uint4 *sign = reinterpret_cast<const uint4 *>(signs);
            if constexpr (sizeof(T) == 2) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = dense_pair(mul2(z[4 * c + j], scale), dst);
                    const uint4 s = sign[c];
                    reinterpret_cast<uint4 *>(to)[c] = make_uint4(w[0] ^ s.x, w[1] ^ s.y, w[2] ^ s.z, w[3] ^ s.w);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float2 a = mul2(z[2 * c], scale), b = mul2(z[2 * c + 1], scale);
                    const uint4 s = sign[c];
                    reinterpret_cast<uint4 *>(to)[c] =
                        make_uint4(__float_as_uint(a.x) ^ s.x, __float_as_uint(a.y) ^ s.y, __float_as_uint(b.x) ^ s.z,
                                   __float_as_uint(b.y) ^ s.w);
                }
            }
            __syncwarp();
            constexpr int CHUNKS = D * (int)sizeof(T) / 16, ROWS = 32 / CHUNKS;   // of 16 bytes a row; rows at a time
            T *out = dst + (now.row * g.n_kv + now.head) * D;
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += ROWS) {
                const int r = r0 + lane / CHUNKS, c = lane % CHUNKS;
                if (r < now.n)
                    __stcs(reinterpret_cast<uint4 *>(out + (int64_t)r * g.n_kv * D) + c,
                           *reinterpret_cast<const uint4 *>(stage + r * LINE + c * 16));
            }
        };
        float2 x[32];
        kc.decode(sm, g.kb, lane, x);
        finish(x, std::integral_constant<int, KT::STAGES>(), ks, k);
        vc.decode(L::BOTH ? sm : sm + L::V_AT, g.vb, lane, x);
        task += stride;
        t = load(task);
        finish(x, std::integral_constant<int, VT::STAGES>(), vs, v);
    }
}

namespace {

template <typename T>
int launch_dense(CacheBase *c, const Plan &plan, int32_t n_spans, int64_t tiles, void *k, void *v, bool rotated,
                 cudaStream_t s) {
    const Geo &g = c->g;
    int sms = 148;
    CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, c->device));
    // a round of the rotation multiplies by 2^-rot_shift (or rot_inv / 2^15), and H H = 64
    const int rounds = rotated ? 0 : g.rounds;
    const double back = (g.rot_shift >= 0 ? std::ldexp(1.0, g.rot_shift) : 32768.0 / g.rot_inv) / 64.0;
    const float unit = (float)(std::pow(back, rounds) * std::ldexp(1.0, -g.norm_frac - g.centroid_frac));
    return plan.run(c, s, [&](const auto &src) -> cudaError_t {
        using S = std::decay_t<decltype(src)>;
        auto fn = g.kb == 4 && g.vb == 2   ? k_dense<4, 2, T, S>
                  : g.kb == 3 && g.vb == 3 ? k_dense<3, 3, T, S>
                                           : k_dense<0, 0, T, S>;
        const size_t tables = g.kb == 4 && g.vb == 2   ? DenseLayout<4, 2>::STAGE_AT
                              : g.kb == 3 && g.vb == 3 ? DenseLayout<3, 3>::STAGE_AT
                                                       : DenseLayout<0, 0>::STAGE_AT;
        const size_t smem = tables + DENSE_THREADS * (D * sizeof(T) + 16);
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        const int64_t tasks = tiles * g.n_kv, ctas = (tasks + DENSE_WARPS - 1) / DENSE_WARPS;
        const unsigned grid = (unsigned)std::min<int64_t>(ctas, (int64_t)sms * (sizeof(T) == 4 ? 1 : 2));
        *c->launches += 1;
        return launch_after(fn, grid, (unsigned)DENSE_THREADS, smem, s, g, (const DevTables *)c->d_tables,
                            (const uint8_t *)c->d_pool, (const int32_t *)c->d_page_table, (T *)k, (T *)v, n_spans,
                            tasks, (int32_t)rounds, unit, src);
    });
}

int dense_body(CacheBase *c, int32_t B, const int32_t *seq, const int64_t *t0, const int64_t *n, void *k, void *v,
               int32_t dtype, bool rotated, cudaStream_t s) {
    std::vector<DenseSpan> spans;
    spans.reserve((size_t)B);
    int64_t tiles = 0, total = 0;
    for (int32_t b = 0; b < B; ++b) {
        if (seq[b] < 0 || seq[b] >= c->cfg.max_seqs)
            return fail(INS_EINVAL, "sequence id " + std::to_string(seq[b]) + " out of range");
        const int64_t len = c->h_seq_lens[seq[b]];
        if (t0[b] < 0 || n[b] < 0 || t0[b] > len || n[b] > len - t0[b])
            return fail(INS_EBADLEN, "rows outside sequence " + std::to_string(seq[b]) + "'s " + std::to_string(len) +
                                         " cached tokens");
        if (n[b] == 0) continue;
        spans.push_back(DenseSpan{seq[b], (int32_t)t0[b], (int32_t)n[b], (int32_t)tiles, total});
        tiles += (n[b] + 31) / 32;
        total += n[b];
        if (tiles > INT32_MAX) return fail(INS_EBADLEN, "too many rows in one call");
    }
    if (spans.empty()) return INS_OK;
    if (!k || !v) return fail(INS_EINVAL, "dense: NULL buffer");
    Plan plan;
    plan.add(spans);
    const int32_t m = (int32_t)spans.size();
    if (dtype == INS_F32) return launch_dense<float>(c, plan, m, tiles, k, v, rotated, s);
    if (dtype == INS_F16) return launch_dense<__half>(c, plan, m, tiles, k, v, rotated, s);
    return launch_dense<__nv_bfloat16>(c, plan, m, tiles, k, v, rotated, s);
}

}  // namespace
}  // namespace ins

using namespace ins;

extern "C" int ins_cache_dense(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int64_t *t0,
                               const int64_t *n, void *k, void *v, int32_t dtype, int32_t rotated, void *stream) {
    if (!cache) return fail(INS_EINVAL, "cache is NULL");
    if (B < 0 || (B > 0 && (!seq_ids || !t0 || !n))) return fail(INS_EINVAL, "dense arguments");
    if (dtype != INS_F32 && dtype != INS_F16 && dtype != INS_BF16)
        return fail(INS_EINVAL, "dense: k and v are INS_F32, INS_F16 or INS_BF16");
    if (((uintptr_t)k & 15u) || ((uintptr_t)v & 15u)) return fail(INS_EINVAL, "dense: k and v 16-byte aligned");
    if (B == 0) return INS_OK;
    CacheBase *c = cache_base(cache);
    return guarded([&] {
        DeviceGuard dg(c->device);
        return dense_body(c, B, seq_ids, t0, n, k, v, dtype, rotated != 0, (cudaStream_t)stream);
    });
}
