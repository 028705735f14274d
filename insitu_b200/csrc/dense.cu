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
// DENSE_TILE rows are tiles [tile, next span's tile).
struct DenseSpan {
    int32_t seq, t0, n, tile;
    int64_t row;
};

constexpr int DENSE_TILE = 32, DENSE_THREADS = 256;

template <typename T>
__device__ __forceinline__ void store8(T *dst, const float (&x)[8]);
template <>
__device__ __forceinline__ void store8(float *dst, const float (&x)[8]) {
    reinterpret_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8(__half *dst, const float (&x)[8]) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(h);
}
template <>
__device__ __forceinline__ void store8(__nv_bfloat16 *dst, const float (&x)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(h);
}

// The centroids of 8 codes of `bits` bits from byte `at` of a row on.
template <int BITS>
__device__ __forceinline__ void centroids8(const uint8_t *at, int bits_any, const float *cent, float (&y)[8]) {
    const int bits = BITS ? BITS : bits_any;
    uint64_t w = 0;
    if constexpr (BITS == 4) w = *reinterpret_cast<const uint32_t *>(at);
    else if constexpr (BITS == 2) w = *reinterpret_cast<const uint16_t *>(at);
    else
        for (int i = 0; i < bits; ++i) w |= (uint64_t)at[i] << (8 * i);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = cent[(uint32_t)(w >> (i * bits)) & ((1u << bits) - 1u)];
}

// Four threads a vector; thread t holds channels 8 t + i and 32 + 8 t + i (a
// store of 16 bytes is then a contiguous run of the four). Stages 1, 2, 4 and
// 32 of the butterfly stay in a thread, 8 and 16 exchange with threads t ^ 1
// and t ^ 2.
__device__ __forceinline__ void hadamard(float (&a)[8], float (&b)[8], int t) {
#pragma unroll
    for (int h = 1; h < 8; h *= 2)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (!(i & h)) {
                const float x = a[i], y = a[i + h], u = b[i], v = b[i + h];
                a[i] = x + y, a[i + h] = x - y, b[i] = u + v, b[i + h] = u - v;
            }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = a[i], y = b[i];
        a[i] = x + y, b[i] = x - y;
    }
#pragma unroll
    for (int h = 1; h < 4; h *= 2) {
        const float s = t & h ? -1.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = fmaf(s, a[i], __shfl_xor_sync(FULL, a[i], h));
            b[i] = fmaf(s, b[i], __shfl_xor_sync(FULL, b[i], h));
        }
    }
}

// One CTA per 32 rows of a span, all KV heads. Bound by the bytes: 52 read and
// 256 or 512 written a row and head.
template <int KB, int VB, typename T, class Src>
__global__ void __launch_bounds__(DENSE_THREADS) k_dense(Geo g, const DevTables *__restrict__ tb,
                                                         const uint8_t *__restrict__ pool,
                                                         const int32_t *__restrict__ table, T *__restrict__ k,
                                                         T *__restrict__ v, int32_t n_spans, int32_t rounds,
                                                         float unit, const __grid_constant__ Src src) {
    __shared__ float cent[2][256];
    __shared__ int64_t at[DENSE_TILE];
    __shared__ int32_t in_page[DENSE_TILE];
    const int tid = threadIdx.x, t = tid % 4;
    for (int i = tid; i < (1 << g.kb); i += DENSE_THREADS) cent[0][i] = (float)tb->k_cent[i];
    for (int i = tid; i < (1 << g.vb); i += DENSE_THREADS) cent[1][i] = (float)tb->v_cent[i];
    wait_prior_grid();
    const DenseSpan *spans = reinterpret_cast<const DenseSpan *>(src.data());
    int lo = 0, hi = n_spans - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (spans[mid].tile <= (int)blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    const DenseSpan sp = spans[lo];
    const int r0 = (blockIdx.x - sp.tile) * DENSE_TILE, n = min(DENSE_TILE, sp.n - r0);
    if (tid < n) {
        const int p = sp.t0 + r0 + tid;
        at[tid] = (int64_t)table[(int64_t)sp.seq * g.max_pages + p / g.P] * g.page_bytes;
        in_page[tid] = p % g.P;
    }
    __syncthreads();
    const int all = n * g.n_kv;
    // whole warps go around, as the butterfly exchanges lanes
    for (int i = tid / 4; i / 8 * 8 < all; i += DENSE_THREADS / 4) {
        const bool live = i < all;
        const int r = live ? i / g.n_kv : 0, head = live ? i % g.n_kv : 0;
        const uint8_t *region = pool + at[r] + head * g.head_bytes;
        const uint32_t norms = *reinterpret_cast<const uint32_t *>(region + nplane_off(g) + (int64_t)in_page[r] * 4);
        const int64_t to = ((sp.row + r0 + r) * g.n_kv + head) * D + 8 * t;
        auto vector = [&](auto width, const uint8_t *row, int bits, const float *c, int16_t norm, T *dst) {
            constexpr int BITS = decltype(width)::value;
            float a[8], b[8];
            centroids8<BITS>(row + t * bits, bits, c, a);
            centroids8<BITS>(row + (4 + t) * bits, bits, c, b);
            const float scale = (float)norm * unit;
            for (int rd = rounds - 1; rd >= 0; --rd) {
                hadamard(a, b, t);
                const uint64_t m = tb->sign_mask[rd];
                const uint32_t ma = (uint32_t)(m >> (8 * t)), mb = (uint32_t)(m >> (32 + 8 * t));
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    a[j] = __uint_as_float(__float_as_uint(a[j]) ^ (ma >> j << 31));
                    b[j] = __uint_as_float(__float_as_uint(b[j]) ^ (mb >> j << 31));
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] *= scale, b[j] *= scale;
            if (!live) return;
            store8(dst + to, a);
            store8(dst + to + 32, b);
        };
        vector(std::integral_constant<int, KB>(), region + (int64_t)in_page[r] * g.kbytes, g.kb, cent[0],
               (int16_t)(norms & 0xffffu), k);
        vector(std::integral_constant<int, VB>(), region + vplane_off(g) + (int64_t)in_page[r] * g.vbytes, g.vb,
               cent[1], (int16_t)(norms >> 16), v);
    }
}

namespace {

template <typename T>
int launch_dense(CacheBase *c, const Plan &plan, int32_t n_spans, int64_t tiles, void *k, void *v, bool rotated,
                 cudaStream_t s) {
    const Geo &g = c->g;
    // a round of the rotation multiplies by 2^-rot_shift (or rot_inv / 2^15), and H H = 64
    const int rounds = rotated ? 0 : g.rounds;
    const double back = (g.rot_shift >= 0 ? std::ldexp(1.0, g.rot_shift) : 32768.0 / g.rot_inv) / 64.0;
    const float unit = (float)(std::pow(back, rounds) * std::ldexp(1.0, -g.norm_frac - g.centroid_frac));
    return plan.run(c, s, [&](const auto &src) -> cudaError_t {
        using S = std::decay_t<decltype(src)>;
        auto fn = g.kb == 4 && g.vb == 2   ? k_dense<4, 2, T, S>
                  : g.kb == 3 && g.vb == 3 ? k_dense<3, 3, T, S>
                                           : k_dense<0, 0, T, S>;
        *c->launches += 1;
        return launch_after(fn, (unsigned)tiles, (unsigned)DENSE_THREADS, 0, s, g, (const DevTables *)c->d_tables,
                            (const uint8_t *)c->d_pool, (const int32_t *)c->d_page_table, (T *)k, (T *)v, n_spans,
                            (int32_t)rounds, unit, src);
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
        tiles += (n[b] + DENSE_TILE - 1) / DENSE_TILE;
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
