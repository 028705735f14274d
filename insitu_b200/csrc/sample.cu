// Sampling one token per row of logits: temperature, top-k, top-p, min-p, and
// the draw itself from given uniform random numbers.
//
// With z_i = x_i / t and w_i = exp(z_i - max z), a row keeps the k largest x
// (ties: the lowest indexes), of those the shortest leading run, in falling
// order of x, whose mass reaches top_p of theirs, of those the ones with
// w_i >= min_p; the token is the kept i with the largest z_i - log(-log u_i),
// which is distributed as the kept w_i normalised.
//
// No sort: both cuts are order statistics (by count, by mass), found by
// histograms that narrow a range of values. The row's logits are read from
// memory once, into the shared memory of a thread-block cluster (each CTA a
// contiguous slice of the vocabulary), and the CTAs exchange histograms through
// distributed shared memory. The cuts run over the few tokens within 6 nats
// of the maximum, which one pass lists, where those decide them (they hold the
// k-th largest, the mass), else over the whole slice. The histograms' last
// levels work on the values' bits, and on the indexes where equal values are
// split, so the order is exact.
//
// Masses are summed as integers (64-bit totals), so that a result does not
// depend on the order of the atomics. Those that decide a cut are w_i rounded
// to 2^-31, 2^-32 a token at most against a largest w of 1: a cut by top_p is
// that of the definition with masses moved by up to vocab * 2^-32 of the total
// (6e-5 at 262,144 tokens, where all but one lie just below 2^-32, 22.2 nats
// under the maximum, and count as nothing). The log-probability's mass is
// summed to 2^-40.
//
// Bound: one read of the logits (and of the random numbers, where a row is
// not filtered); at a few rows the passes' latency. Histograms over the whole
// slice alone, with exact divisions, took 322 us for 256 rows of 128,000
// (186 instructions a logit).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>

#include "cache.h"

namespace ins {
namespace cg = cooperative_groups;

constexpr int SMP_THREADS = 512, SMP_WARPS = SMP_THREADS / 32, SMP_BINS = 256;
constexpr int SMP_MAX_VOCAB = 1 << 18;
constexpr int SMP_WINDOWS = 4;               // first-level windows of 8 nats each, the last one open
constexpr int SMP_LIST = 2048;               // tokens a CTA can list
// Nats below the maximum that are listed: as few tokens as still decide the cuts
// of rows with a few likely tokens. 256 x 128,000, with 4, 6, 8 and 12 nats, us:
// top-k of 50 96, 99, 144, 159; and top-p of 0.9 151, 148, 234, 266; top-k of
// 1,000 210, 157, 204, 245; top-p 0.9 at temperature 0.5 141, 115, 111, 125. One
// row of 32,000, top-k of 50: 20.0, 15.6, 14.9, 14.6. Rows that the list does
// not decide pass over their slices whatever it is: top-p 0.9 of wide rows 515
// to 534, N(0, 1) logits 460; those of k = 50 160.
constexpr float SMP_NEAR = 6.0f;

struct SampleArgs {
    const void *logits;
    int64_t stride;
    const float *uniform;
    int64_t u_stride;
    const float *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int64_t *tokens;
    float *logprobs;
    int32_t vocab, slice;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// Unsigned integers in the order of the floats.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// What a CTA publishes to its cluster; two copies, used in turn, so that one
// cluster barrier a step is enough.
struct SampleShared {
    uint32_t cnt[2][SMP_BINS], lo[2][SMP_BINS], hi[2][SMP_BINS];
    unsigned long long sum[2], sum2[2];
    float val[2];
    int32_t idx[2];
    // this CTA only
    unsigned long long wsum[SMP_WARPS], wsum2[SMP_WARPS];
    float wval[SMP_WARPS];
    int32_t widx[SMP_WARPS];
    uint32_t scan_c[SMP_BINS / 32];
    unsigned long long scan_m[SMP_BINS / 32];
    int32_t hit_bin;
    uint32_t hit_cnt, hit_before_c;
    unsigned long long hit_mass, hit_before_m;
    uint32_t key_lo, key_hi;
    int32_t listed;
    float list_x[SMP_LIST];
    int32_t list_i[SMP_LIST];
};

// The largest of a 16-byte vector's elements (NaN ignored).
__device__ __forceinline__ float vec_max(const uint4 &v, const float *) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
__device__ __forceinline__ float vec_max(const uint4 &v, const __half *) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&v);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float vec_max(const uint4 &v, const __nv_bfloat16 *) {
    const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
}

// A slice in shared memory: `head` single elements, `body` 16-byte vectors,
// single elements again, at the alignment within 16 bytes that the row has in
// global memory.
template <typename T>
struct Slice {
    static constexpr int V = 16 / sizeof(T);
    T *at;
    const uint4 *vec;                        // the body, 16-byte aligned also where it is empty
    int n, head, body;

    // Copies n elements from global memory; returns this thread's largest.
    __device__ __forceinline__ float stage(uint8_t *smem, const T *src, int count) {
        const int shift = (int)(((uintptr_t)src & 15u) / sizeof(T));
        at = reinterpret_cast<T *>(smem) + shift;
        n = count;
        head = min(n, (V - shift) % V);
        body = (n - head) / V;
        float top = -INFINITY;
        const uint4 *vs = reinterpret_cast<const uint4 *>(((uintptr_t)src + 15u) & ~(uintptr_t)15u);
        uint4 *vd = reinterpret_cast<uint4 *>(smem + (shift ? 16 : 0));
        vec = vd;
        int i = threadIdx.x;
        for (; i + 7 * SMP_THREADS < body; i += 8 * SMP_THREADS) {
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = __ldcs(vs + i + k * SMP_THREADS);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                vd[i + k * SMP_THREADS] = v[k];
                top = fmaxf(top, vec_max(v[k], at));
            }
        }
#pragma unroll 4
        for (; i < body; i += SMP_THREADS) {
            const uint4 v = __ldcs(vs + i);
            vd[i] = v;
            top = fmaxf(top, vec_max(v, at));
        }
        for (int k = threadIdx.x; k < n - body * V; k += SMP_THREADS) {
            const int e = k < head ? k : k + body * V;
            at[e] = src[e];
            top = fmaxf(top, to_f32(at[e]));
        }
        __syncthreads();
        return top;
    }
    // f(x, i) for each element whose value is at least `from` (never a NaN, and
    // -0 as 0).
    template <typename F>
    __device__ __forceinline__ void above(float from, F &&f) const {
        for (int i = threadIdx.x; i < body; i += SMP_THREADS) {
            const uint4 v = vec[i];
            if (!(vec_max(v, at) >= from)) continue;
            const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float x = to_f32(e[k]);
                if (x >= from) f(x + 0.0f, head + i * V + k);
            }
        }
        for (int k = threadIdx.x; k < n - body * V; k += SMP_THREADS) {
            const int e = k < head ? k : k + body * V;
            const float x = to_f32(at[e]);
            if (x >= from) f(x + 0.0f, e);
        }
    }
};

// A row's tokens as the cuts see them: the CTA's slice, or its list.
template <typename T>
struct Row {
    SampleShared &sm;
    cg::cluster_group cl;
    Slice<T> slice;                          // this CTA's logits, in shared memory
    int n, first, parity, C;                 // n: tokens listed
    float xmax, inv_t, bins;                 // 1 / t; first-level bins a unit of x
    // kept so far: value key above thr_key, or equal to it at an index up to thr_idx
    uint32_t thr_key;
    int32_t thr_idx;
    bool list;

    // f(x, key, index) for each kept token that is not below `from`
    template <typename F>
    __device__ __forceinline__ void each(float from, F &&f) const {
        auto token = [&](float x, int i) {
            const uint32_t key = order_key(x);
            if (key > thr_key || (key == thr_key && i <= thr_idx)) f(x, key, i);
        };
        if (list) {
            for (int i = threadIdx.x; i < n; i += SMP_THREADS)
                if (sm.list_x[i] >= from) token(sm.list_x[i], sm.list_i[i]);
        } else {
            slice.above(fmaxf(from, -3.4028235e38f), [&](float x, int i) { token(x, first + i); });
        }
    }
    // z and w: 2^-23 of z from the two roundings, 2^-22 of w from the exponential
    __device__ __forceinline__ float z_of(float x) const { return x == xmax ? 0.0f : (x - xmax) * inv_t; }
    __device__ __forceinline__ float w_of(float z) const {
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(z * 1.4426950408889634f));
        return w;
    }
    // w in units of 2^-31
    __device__ __forceinline__ uint32_t mass_of(float x) const {
        return __float2uint_rn(w_of(z_of(x)) * 2147483648.0f);
    }
    // First-level bin: the distance below the maximum in 1/32 of t. Rounding
    // is monotone, so the bins are ranges of values.
    __device__ __forceinline__ int bin_of(float x) const {
        const float d = x == xmax ? 0.0f : xmax - x;
        return min(__float2int_rz(d * bins), SMP_WINDOWS * SMP_BINS - 1);
    }

    // Two sums of the cluster, for every thread.
    __device__ void cluster_sum(unsigned long long &v, unsigned long long &u) {
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o), u += __shfl_xor_sync(FULL, u, o);
        if (threadIdx.x % 32 == 0) sm.wsum[threadIdx.x / 32] = v, sm.wsum2[threadIdx.x / 32] = u;
        __syncthreads();
        if (threadIdx.x < 32) {
            v = threadIdx.x < SMP_WARPS ? sm.wsum[threadIdx.x] : 0;
            u = threadIdx.x < SMP_WARPS ? sm.wsum2[threadIdx.x] : 0;
            for (int o = SMP_WARPS / 2; o; o >>= 1) v += __shfl_xor_sync(FULL, v, o), u += __shfl_xor_sync(FULL, u, o);
            if (threadIdx.x == 0) sm.sum[parity] = v, sm.sum2[parity] = u;
        }
        cl.sync();
        v = u = 0;
        for (int r = 0; r < C; ++r)
            v += *cl.map_shared_rank(&sm.sum[parity], r), u += *cl.map_shared_rank(&sm.sum2[parity], r);
        parity ^= 1;
    }
    // The largest value of the cluster and the lowest index that has it.
    __device__ void cluster_best(float &v, int &i) {
        auto better = [](float a, int ai, float b, int bi) { return a > b || (a == b && ai < bi); };
        for (int o = 16; o; o >>= 1) {
            const float ov = __shfl_xor_sync(FULL, v, o);
            const int oi = __shfl_xor_sync(FULL, i, o);
            if (better(ov, oi, v, i)) v = ov, i = oi;
        }
        if (threadIdx.x % 32 == 0) sm.wval[threadIdx.x / 32] = v, sm.widx[threadIdx.x / 32] = i;
        __syncthreads();
        if (threadIdx.x < 32) {
            v = threadIdx.x < SMP_WARPS ? sm.wval[threadIdx.x] : -INFINITY;
            i = threadIdx.x < SMP_WARPS ? sm.widx[threadIdx.x] : INT_MAX;
            for (int o = SMP_WARPS / 2; o; o >>= 1) {
                const float ov = __shfl_xor_sync(FULL, v, o);
                const int oi = __shfl_xor_sync(FULL, i, o);
                if (better(ov, oi, v, i)) v = ov, i = oi;
            }
            if (threadIdx.x == 0) sm.val[parity] = v, sm.idx[parity] = i;
        }
        cl.sync();
        v = -INFINITY, i = INT_MAX;
        for (int r = 0; r < C; ++r) {
            const float ov = *cl.map_shared_rank(&sm.val[parity], r);
            const int oi = *cl.map_shared_rank(&sm.idx[parity], r);
            if (better(ov, oi, v, i)) v = ov, i = oi;
        }
        parity ^= 1;
    }

    __device__ void clear() {
        __syncthreads();
        for (int b = threadIdx.x; b < SMP_BINS; b += SMP_THREADS)
            sm.cnt[parity][b] = sm.lo[parity][b] = sm.hi[parity][b] = 0;
        __syncthreads();
    }
    __device__ __forceinline__ void count(int b, uint32_t mass) {
        atomicAdd(&sm.cnt[parity][b], 1u);
        if (mass) {
            atomicAdd(&sm.lo[parity][b], mass & 0xffffu);
            atomicAdd(&sm.hi[parity][b], mass >> 16);
        }
    }
    // Adds the cluster's histograms up and finds the first bin at which the
    // running count reaches need_c (BY_MASS: the running mass need_m).
    // Returns it (SMP_BINS: none) with the bin's own count and the totals
    // before it (all of them where there is none).
    template <bool BY_MASS>
    __device__ int crossing(uint32_t need_c, unsigned long long need_m, uint32_t &before_c,
                            unsigned long long &before_m, uint32_t &in_c) {
        cl.sync();
        uint32_t c = 0, ic = 0;
        unsigned long long m = 0, im = 0;
        const int b = threadIdx.x, lane = b % 32;
        if (b < SMP_BINS) {
            for (int r = 0; r < C; ++r) {
                c += cl.map_shared_rank(&sm.cnt[parity][0], r)[b];
                if (BY_MASS)
                    m += cl.map_shared_rank(&sm.lo[parity][0], r)[b] +
                         ((unsigned long long)cl.map_shared_rank(&sm.hi[parity][0], r)[b] << 16);
            }
            ic = c, im = m;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t pc = __shfl_up_sync(FULL, ic, o);
                const unsigned long long pm = __shfl_up_sync(FULL, im, o);
                if (lane >= o) ic += pc, im += pm;
            }
            if (lane == 31) sm.scan_c[b / 32] = ic, sm.scan_m[b / 32] = im;
        }
        if (b == 0) sm.hit_bin = SMP_BINS;
        __syncthreads();
        if (b < SMP_BINS) {
            for (int w = 0; w < b / 32; ++w) ic += sm.scan_c[w], im += sm.scan_m[w];
            const bool before = BY_MASS ? im - m < need_m : ic - c < need_c;
            const bool after = BY_MASS ? im >= need_m : ic >= need_c;
            if (before && after) sm.hit_bin = b, sm.hit_cnt = c, sm.hit_before_c = ic - c, sm.hit_before_m = im - m;
            if (b == SMP_BINS - 1 && !after) sm.hit_before_c = ic, sm.hit_before_m = im, sm.hit_cnt = 0;
        }
        __syncthreads();
        before_c = sm.hit_before_c;
        before_m = sm.hit_before_m;
        in_c = sm.hit_cnt;
        parity ^= 1;
        return sm.hit_bin;
    }

    // The smallest (LOW) or largest key whose value lies in first-level bin
    // `bin`, by a 32-way search of one warp over all keys of non-masked values.
    template <bool LOW>
    __device__ uint32_t bin_edge(int bin) const {
        uint32_t a = order_key(-INFINITY) + 1, b = order_key(xmax);   // the answer lies in [a, b]
        const int lane = threadIdx.x % 32;
        while (a < b) {
            const uint32_t step = (b - a) / 32 + 1;
            // bins fall as keys rise: LOW wants the first key at or below `bin`
            // (as a bin number), the other the last one at or above it
            const uint64_t at = LOW ? (uint64_t)a + (uint64_t)step * (lane + 1) - 1 : (uint64_t)a + (uint64_t)step * lane;
            const bool in = at <= b;
            const int v = bin_of(key_value(in ? (uint32_t)at : b));
            if (LOW) {
                const unsigned ok = __ballot_sync(FULL, !in || v <= bin);
                const int l = __ffs(ok) - 1;             // lane 31's `at` is b or beyond: always ok
                const uint64_t hi = (uint64_t)a + (uint64_t)step * (l + 1) - 1;
                const uint64_t lo = (uint64_t)a + (uint64_t)step * l;
                b = (uint32_t)(hi < b ? hi : b);
                a = (uint32_t)lo;
            } else {
                const unsigned ok = __ballot_sync(FULL, in && v >= bin);
                const int l = 31 - __clz(ok);            // lane 0's `at` is a: always ok
                const uint64_t hi = (uint64_t)a + (uint64_t)step * (l + 1) - 1;
                a = (uint32_t)((uint64_t)a + (uint64_t)step * l);
                b = (uint32_t)(hi < b ? hi : b);
            }
        }
        return a;
    }

    // Narrows the kept set to its first need_c tokens (BY_MASS: the shortest
    // run whose mass reaches need_m), in falling order of value, ties by index.
    template <bool BY_MASS>
    __device__ void cut(uint32_t need_c, unsigned long long need_m) {
        uint32_t before_c, in_c;
        unsigned long long before_m;
        int bin = SMP_BINS, win = 0;
        for (; win < SMP_WINDOWS; ++win) {
            clear();
            // (the margin covers the bins' roundings; below an infinite maximum
            // every distance is infinite, so only the last window holds more)
            const float edge = xmax < INFINITY ? xmax - (win + 1) * SMP_BINS * 1.0001f / bins - 1e-6f * fabsf(xmax)
                                               : xmax;
            const float from = win + 1 < SMP_WINDOWS ? edge : -INFINITY;
            each(from, [&](float x, uint32_t, int) {
                const int b = bin_of(x) - win * SMP_BINS;
                if (b >= 0 && b < SMP_BINS) count(b, BY_MASS ? mass_of(x) : 0u);
            });
            bin = crossing<BY_MASS>(need_c, need_m, before_c, before_m, in_c);
            need_c -= before_c;
            need_m -= before_m;
            if (bin < SMP_BINS) break;
        }
        if (bin == SMP_BINS) return;                    // fewer tokens than asked for: all stay
        if (threadIdx.x < 32) {
            const uint32_t e = bin_edge<true>(win * SMP_BINS + bin);
            if (threadIdx.x == 0) sm.key_lo = e;
        } else if (threadIdx.x < 64) {
            const uint32_t e = bin_edge<false>(win * SMP_BINS + bin);
            if (threadIdx.x == 32) sm.key_hi = e;
        }
        __syncthreads();
        uint32_t a = max(sm.key_lo, thr_key), b = sm.key_hi;
        // the run ends inside [a, b], in_c tokens of which need_c (need_m) are wanted
        auto whole = [&] { return BY_MASS ? in_c == 1 : in_c == need_c; };
        while (a < b && !whole()) {
            const int sh = max(0, 32 - __clz(b - a) - 8);
            clear();
            each(key_value(a), [&](float x, uint32_t key, int) {
                if (key >= a && key <= b) count((int)((b - key) >> sh), BY_MASS ? mass_of(x) : 0u);
            });
            const int c = crossing<BY_MASS>(need_c, need_m, before_c, before_m, in_c);
            need_c -= before_c;
            need_m -= before_m;
            b -= (uint32_t)c << sh;
            a = max(a, b - min(b, (1u << sh) - 1u));
        }
        int ties = INT_MAX;
        if (!whole()) {
            // a == b: equal values, of which the first `need` indexes stay
            uint32_t need = need_c;
            if (BY_MASS) {
                const uint32_t q = max(1u, mass_of(key_value(a)));
                need = (uint32_t)min((unsigned long long)in_c, (need_m + q - 1) / q);
            }
            int ia = 0, ib = SMP_MAX_VOCAB - 1;
            while (need != in_c && ia < ib) {
                const int sh = max(0, 32 - __clz(ib - ia) - 8);
                clear();
                each(key_value(a), [&](float, uint32_t key, int i) {
                    if (key == a && i >= ia && i <= ib) count((i - ia) >> sh, 0u);
                });
                const int c = crossing<false>(need, 0, before_c, before_m, in_c);
                need -= before_c;
                ia += c << sh;
                ib = min(ib, ia + (1 << sh) - 1);
            }
            ties = ib;
        }
        // an earlier cut may have split the same ties
        thr_idx = a == thr_key ? min(thr_idx, ties) : ties;
        thr_key = a;
    }
};

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS) k_sample(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ SampleShared sm;
    wait_prior_grid();
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int64_t row = blockIdx.x / C;
    const int first = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - first);
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const int k = a.top_k ? a.top_k[row] : 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f, floor_w = a.min_p ? a.min_p[row] : 0.0f;
    if (threadIdx.x == 0) sm.listed = 0;
    Slice<T> slice;
    float best = slice.stage(dyn, reinterpret_cast<const T *>(a.logits) + row * a.stride + first, n);
    Row<T> R{sm, cl, slice, 0, first, 0, C, 0.0f, 1.0f, 32.0f, 0u, INT_MAX, false};
    int at = INT_MAX;
    R.cluster_best(best, at);
    best += 0.0f;
    const bool none = !(best > -INFINITY);
    if (none || !(t > 0.0f)) {
        // nothing to choose from, or the largest logit at its lowest index
        float v = -INFINITY;
        if (!none) slice.above(best, [&](float x, int i) { v = x, at = min(at, first + i); });
        R.cluster_best(v, at);
        if (rank == 0 && threadIdx.x == 0) {
            a.tokens[row] = none ? -1 : at;
            if (a.logprobs) a.logprobs[row] = none ? -INFINITY : 0.0f;
        }
        cl.sync();
        return;
    }
    R.xmax = best;
    R.inv_t = __fdiv_rn(1.0f, t);
    R.bins = __fdiv_rn(32.0f, t);
    const bool by_count = k > 0 && k < a.vocab, by_mass = p < 1.0f;
    unsigned long long total = 0;            // mass of all tokens, where top_p cuts them
    if (by_count || by_mass || floor_w > 0.0f) {
        // List the tokens near the maximum. What top_p takes its share of (all
        // tokens: w below 2^-32, 22.2 nats away, counts as 0) is summed in the
        // same pass.
        const bool sum_all = by_mass && !by_count;
        float near = SMP_NEAR;
        if (!by_count && !by_mass) near = -logf(floor_w) + 0.01f;        // min_p alone cuts there
        const float list_from = best - near * t;
        const float from = sum_all ? fminf(list_from, best - 22.2f * t) : list_from;
        unsigned long long mass = 0, listed = 0;
        slice.above(fmaxf(from, -3.4028235e38f), [&](float x, int i) {
            const uint32_t m = by_mass ? R.mass_of(x) : 0u;
            mass += m;
            if (x < list_from) return;
            const int to = atomicAdd(&sm.listed, 1);
            if (to < SMP_LIST) sm.list_x[to] = x, sm.list_i[to] = first + i;
        });
        __syncthreads();
        // tokens listed in the low half, CTAs whose list ran over in the high one
        const int mine = sm.listed;
        if (threadIdx.x == 0) listed = (unsigned long long)mine + ((unsigned long long)(mine > SMP_LIST) << 32);
        total = mass;
        R.cluster_sum(total, listed);
        bool enough = listed >> 32 == 0;
        if (by_count) enough &= listed >= (unsigned long long)k;
        if (enough && sum_all) {
            unsigned long long in = 0, unused = 0;
            for (int i = threadIdx.x; i < mine; i += SMP_THREADS) in += R.mass_of(sm.list_x[i]);
            R.cluster_sum(in, unused);
            enough = (double)in >= ceil((double)p * (double)total);
        }
        if (enough) R.list = true, R.n = mine;
    }
    if (by_count) R.template cut<false>((uint32_t)k, 0);
    if (by_mass) {
        if (by_count) {
            unsigned long long unused = 0;
            total = 0;
            R.each(-INFINITY, [&](float x, uint32_t, int) { total += R.mass_of(x); });
            R.cluster_sum(total, unused);
        }
        const double want = ceil((double)p * (double)total);
        R.template cut<true>(0, want > 1.0 ? (unsigned long long)want : 1ull);
    }
    unsigned long long mass = 0, unused = 0;
    float key = -INFINITY, z_key = 0.0f, reach = INFINITY;
    int token = INT_MAX;
    const float *u = a.uniform + row * a.u_stride;
    // adds the token's mass by add(w), unless min_p drops it
    auto draw = [&](float x, float un, int i, auto &&add) {
        const float z = R.z_of(x), w = R.w_of(z);
        if (!(w >= floor_w)) return;
        add(w);
        // z - log(-log u) beats `key` only where -log u < w exp(-key), and
        // 1 - u <= -log u: most tokens need no logarithm (the margin covers
        // the roundings)
        if (1.0f - un > w * reach) return;
        float r = z - logf(-logf(un));
        r = r == r ? r : -INFINITY;                        // a random number outside [0, 1]
        if (r > key || token == INT_MAX || (r == key && i < token)) {
            key = r, token = i, z_key = z;
            reach = 1.001f * expf(-key);                   // infinite for -inf: no bound
        }
    };
    // in units of 2^-40 (2^18 tokens of mass 1 make 2^58); integers where the order is the list's
    auto units = [](float w) { return __float2ull_rn(w * 0x1p40f); };
    if (R.list || R.thr_key) {
        R.each(R.thr_key ? key_value(R.thr_key) : -INFINITY,
               [&](float x, uint32_t, int i) { draw(x, __ldcs(u + i), i, [&](float w) { mass += units(w); }); });
    } else {
        u += first;
        float sum = 0.0f, lost = 0.0f;
        for (int i = threadIdx.x; i < n; i += 8 * SMP_THREADS) {
            float un[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) un[k] = i + k * SMP_THREADS < n ? __ldcs(u + i + k * SMP_THREADS) : 0.0f;
            float eight = 0.0f;              // the tokens' sum, within 2^-21 of itself
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int e = i + k * SMP_THREADS;
                const float x = e < n ? to_f32(slice.at[e]) : -INFINITY;
                if (x > -INFINITY) draw(x + 0.0f, un[k], first + e, [&](float w) { eight += w; });
            }
            // compensated: the thread's sum (in a fixed order) is rounded as one addition is
            const float y = eight - lost, next = sum + y;
            lost = next - sum - y;
            sum = next;
        }
        mass = units(sum);
    }
    const int mine = token;
    R.cluster_best(key, token);
    R.cluster_sum(mass, unused);
    const bool empty = token == INT_MAX;     // a min_p above 1, or a NaN, keeps no token
    if (empty ? rank == 0 && threadIdx.x == 0 : mine == token) {
        a.tokens[row] = empty ? -1 : token;
        if (a.logprobs) a.logprobs[row] = empty ? -INFINITY : (float)((double)z_key - log((double)mass * 0x1p-40));
    }
    cl.sync();
}

namespace {

template <typename T>
int launch_sample(SampleArgs a, int32_t rows, cudaStream_t s) {
    int dev = 0, sms = 148;
    CK(cudaGetDevice(&dev));
    CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // A cluster of up to 8 CTAs a row: as many as a vocabulary slice of 2,048
    // tokens each leaves, until the rows alone give every SM two CTAs and the
    // slice fits.
    int C = 1;
    auto bytes = [&](int c) {
        const int slice = (a.vocab + c - 1) / c;
        return (size_t)slice * sizeof(T) + 32;
    };
    while (C < 8 && (bytes(C) > 72 * 1024 || ((int64_t)rows * C < 2 * sms && a.vocab / C > 2048))) C *= 2;
    a.slice = (a.vocab + C - 1) / C;
    const size_t smem = bytes(C);
    CK(cudaFuncSetAttribute(k_sample<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * C));
    cfg.blockDim = dim3(SMP_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)C;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    CK(cudaLaunchKernelEx(&cfg, k_sample<T>, a));
    return INS_OK;
}

}  // namespace
}  // namespace ins

using namespace ins;

extern "C" int ins_sample(int32_t rows, int32_t vocab, const void *logits, int32_t dtype, int64_t stride,
                          const float *uniform, int64_t uniform_stride, const float *temperature,
                          const int32_t *top_k, const float *top_p, const float *min_p, int64_t *tokens,
                          float *logprobs, void *stream) {
    return guarded([&]() -> int {
        if (rows < 0 || vocab < 1 || vocab > SMP_MAX_VOCAB || rows > INT_MAX / 8)
            return fail(INS_EINVAL, "sample: rows >= 0, vocab in [1, 262144]");
        if (dtype != INS_F32 && dtype != INS_F16 && dtype != INS_BF16)
            return fail(INS_EINVAL, "sample: logits are INS_F32, INS_F16 or INS_BF16");
        if (rows == 0) return INS_OK;
        if (!logits || !uniform || !tokens) return fail(INS_EINVAL, "sample: NULL buffer");
        if (stride < 0 || uniform_stride < 0) return fail(INS_EINVAL, "sample: a negative row stride");
        if ((uintptr_t)logits % (dtype == INS_F32 ? 4 : 2) || (uintptr_t)uniform % 4)
            return fail(INS_EINVAL, "sample: a buffer is not aligned to its elements");
        const SampleArgs a{logits, stride, uniform, uniform_stride, temperature, top_p, min_p,
                           top_k,  tokens, logprobs, vocab, 0};
        cudaStream_t s = (cudaStream_t)stream;
        if (dtype == INS_F32) return launch_sample<float>(a, rows, s);
        if (dtype == INS_F16) return launch_sample<__half>(a, rows, s);
        return launch_sample<__nv_bfloat16>(a, rows, s);
    });
}
