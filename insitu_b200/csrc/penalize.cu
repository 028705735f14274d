// Penalties of the tokens so far, a bias and a mask of allowed tokens on rows
// of logits: what comes before the draw (sample.cu).
//
// Of a row's tokens so far, `prompt` were asked and the others said. With c
// how often token i has been said and x its logit,
//   y = (asked or said) ? (x > 0 ? x / r : x r) : x
//   y = y - frequency c - presence [c > 0] + bias
// and -inf where the mask does not allow i.
//
// One pass: a CTA owns a slice of a row's vocabulary, counts the row's tokens
// that fall into it in shared memory (a bit says which tokens have a count at
// all), then changes and writes its logits, which it has read meanwhile. 256 rows
// of 128,000 in bf16 with a mask take 30 us without tokens, 4.6 TB/s of reads and
// writes; with 2,048 tokens a row 47 to 49, of 8,000 70 (12 us of a chain of loads
// and atomics, then 3 us for each 1,000 tokens a row: each slice reads all of them).
// With 2,048 the issue slots are busy to 67 %, DRAM to 22 %.
// 256 threads a CTA take 50 us, 1,024 77. Tried: a cluster that counts a row's
// tokens once in distributed shared memory (79 us), equal tokens of a warp merged
// before they are added (60), a kernel that lists each sequence's tokens once
// (67; where 24 rows share a sequence of 9,000 tokens 77 us, this way 30), the
// next tokens loaded while the last are added (a CTA an SM: 80), logits loaded
// after the count so that three CTAs fit an SM (47, and 29). All rows' first
// slices come first: common tokens fall into them, and such a CTA as the last one
// holds the call up (33 -> 30 us at those 24 rows a sequence).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "cache.h"

namespace ins {

constexpr int PEN_THREADS = 512, PEN_BYTES = 32768;      // logits of a slice, at most
constexpr int PEN_MAX_VOCAB = 1 << 18, PEN_MAX_HISTORY = 1 << 30;
constexpr int PEN_LIST = 4096;               // tokens with a count that a slice can list
constexpr uint32_t PEN_ASKED = 1u << 31;     // in a count: the token is in the prompt

struct PenaltyArgs {
    const void *logits;
    void *out;
    int64_t stride, out_stride;
    const int64_t *tokens, *drafted;
    int64_t tokens_stride, drafted_stride;
    const int32_t *lengths, *prompts, *of;
    const float *repetition, *presence, *frequency;
    const float *bias;
    const uint32_t *mask;
    int64_t bias_stride, mask_stride;
    int32_t rows, vocab, slice_log2;         // a CTA: 2^slice_log2 tokens of a row
    int32_t history, histories, n_drafted;
};

// Eight logits as 16-byte vectors: two of floats, one of halves.
template <typename T>
struct Eight {
    static constexpr int N = sizeof(T) / 2;
    uint4 v[N];
    __device__ __forceinline__ T *at() { return reinterpret_cast<T *>(v); }
};

__device__ __forceinline__ float pen_f32(float x) { return x; }
__device__ __forceinline__ float pen_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float pen_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void pen_set(float &to, float x) { to = x; }
__device__ __forceinline__ void pen_set(__half &to, float x) { to = __float2half_rn(x); }
__device__ __forceinline__ void pen_set(__nv_bfloat16 &to, float x) { to = __float2bfloat16_rn(x); }

// -inf in the elements whose bit is 0.
__device__ __forceinline__ void forbid(Eight<float> &e, uint32_t bits) {
    uint32_t *w = reinterpret_cast<uint32_t *>(e.v);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = bits >> i & 1u ? w[i] : 0xff800000u;
}
template <typename T>
__device__ __forceinline__ void forbid(Eight<T> &e, uint32_t bits) {
    constexpr uint32_t none = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    uint32_t *w = reinterpret_cast<uint32_t *>(e.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t keep = (bits >> (2 * i) & 1u) * 0xffffu | (bits >> (2 * i + 1) & 1u) * 0xffff0000u;
        w[i] = (w[i] & keep) | (none & ~keep);
    }
}

// Eight elements from an address of any alignment (to its element): the
// 16-byte vectors around them, shifted together. `off`: the address modulo 16,
// the same for the whole row.
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T *from, uint32_t off) {
    Eight<T> e;
    const uint4 *p = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(from) - off);
    uint4 x = __ldcs(p);
#pragma unroll
    for (int i = 0; i < Eight<T>::N; ++i) {
        if (off == 0) {
            e.v[i] = x;
            if (i + 1 < Eight<T>::N) x = __ldcs(p + i + 1);
            continue;
        }
        const uint4 y = __ldcs(p + i + 1);
        uint32_t a, b, c, d, f;                      // the words that hold the 16 bytes
        switch (off / 4) {
            case 0: a = x.x, b = x.y, c = x.z, d = x.w, f = y.x; break;
            case 1: a = x.y, b = x.z, c = x.w, d = y.x, f = y.y; break;
            case 2: a = x.z, b = x.w, c = y.x, d = y.y, f = y.z; break;
            default: a = x.w, b = y.x, c = y.y, d = y.z, f = y.w; break;
        }
        const uint32_t sh = off % 4 * 8;
        e.v[i] = make_uint4(__funnelshift_r(a, b, sh), __funnelshift_r(b, c, sh), __funnelshift_r(c, d, sh),
                            __funnelshift_r(d, f, sh));
        x = y;
    }
    return e;
}

// A thread changes GROUPS groups of eight logits, the groups where its result's
// rows are aligned to 16 bytes, and single ones at a slice's ends. It loads them
// before the tokens are counted, so that their latency passes meanwhile.
template <typename T>
__global__ void __launch_bounds__(PEN_THREADS) k_penalize(const PenaltyArgs a) {
    // [slice] counts, then values; a bit each; up to PEN_LIST tokens that have one
    extern __shared__ __align__(16) uint32_t counts[];
    __shared__ int listed;
    constexpr int GROUPS = PEN_BYTES / (8 * (int)sizeof(T)) / PEN_THREADS;
    wait_prior_grid();
    const int64_t row = blockIdx.x % a.rows;
    const int slice = 1 << a.slice_log2, first = (int)(blockIdx.x / a.rows) << a.slice_log2;
    const int n = min(slice, a.vocab - first);
    const int tid = threadIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.stride + first;
    T *y = static_cast<T *>(a.out) + row * a.out_stride + first;
    const int head = min(n, (int)((16 - ((uintptr_t)y & 15)) & 15) / (int)sizeof(T));
    const int body = (n - head) / 8;
    const uint32_t off = (uint32_t)((uintptr_t)(x + head) & 15);
    const uint32_t *mask = a.mask ? a.mask + row * a.mask_stride + first / 32 : nullptr;
    // bits i to i + 7 of a row of words
    auto eight_bits = [&](const uint32_t *w, int i) -> uint32_t {
        if (head == 0) return reinterpret_cast<const uint8_t *>(w)[i / 8];      // i is a multiple of 8
        const uint32_t lo = w[i / 32], hi = w[(i + 7) / 32];
        return __funnelshift_r(lo, hi, i % 32) & 0xffu;
    };
    Eight<T> e[GROUPS];
    uint32_t allowed[GROUPS];
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        const int i = head + 8 * (tid + k * PEN_THREADS);
        allowed[k] = 0xffu;
        if (tid + k * PEN_THREADS < body) {
            e[k] = load_eight(x + i, off);
            if (mask) allowed[k] = eight_bits(mask, i);
        }
    }

    const float r = a.repetition ? a.repetition[row] : 1.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f, frequency = a.frequency ? a.frequency[row] : 0.0f;
    const bool counted = r != 1.0f || presence != 0.0f || frequency != 0.0f;
    uint32_t *any = counts + slice;
    uint16_t *list = reinterpret_cast<uint16_t *>(any + slice / 32);
    if (counted) {
        if (tid == 0) listed = 0;
        for (int i = tid; i < (slice + slice / 32) / 4; i += PEN_THREADS)
            reinterpret_cast<uint4 *>(counts)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        // A warp adds up to 8 tokens a lane: all counts first, then the tokens
        // that had none before join the list.
        auto add = [&](const int64_t (&id)[8], int i, int step, int prompt) {
            uint32_t fresh = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (id[k] >= first && id[k] < first + n) {       // else another slice's, or no token at all
                    uint32_t *count = &counts[(int)id[k] - first];
                    const uint32_t old = i + k * step < prompt ? atomicOr(count, PEN_ASKED) : atomicAdd(count, 1u);
                    fresh |= (old == 0) << k;
                }
            if (!__any_sync(FULL, fresh)) return;
            int total = __popc(fresh), at = total;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int before = __shfl_up_sync(FULL, at, o);
                if (tid % 32 >= o) at += before;
            }
            int base = 0;
            if (tid % 32 == 31) base = atomicAdd(&listed, at);
            at += __shfl_sync(FULL, base, 31) - total;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (fresh >> k & 1u) {
                    if (at < PEN_LIST) list[at] = (uint16_t)((int)id[k] - first);
                    ++at;
                }
        };
        const int64_t h = a.of ? a.of[row] : row;
        if (a.tokens && h >= 0 && h < a.histories) {
            const int len = a.lengths ? max(0, min(a.lengths[h], a.history)) : a.history;
            const int prompt = a.prompts ? a.prompts[h] : 0;
            const int64_t *t = a.tokens + h * a.tokens_stride;
            for (int i = tid; i - tid < len; i += 8 * PEN_THREADS) {
                int64_t id[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) id[k] = i + k * PEN_THREADS < len ? t[i + k * PEN_THREADS] : -1;
                add(id, i, PEN_THREADS, prompt);
            }
        }
        for (int i = tid; i - tid < a.n_drafted; i += PEN_THREADS) {
            int64_t id[8] = {-1, -1, -1, -1, -1, -1, -1, -1};
            if (i < a.n_drafted) id[0] = a.drafted[row * a.drafted_stride + i];
            add(id, 0, 0, 0);
        }
        __syncthreads();
        // each such token's value takes its count's place, before any result is written
        auto value = [&](int i, float v) {
            const uint32_t said = counts[i] & ~PEN_ASKED;
            v = v > 0.0f ? __fdiv_rn(v, r) : v * r;
            if (said) v = v - frequency * (float)said - presence;
            counts[i] = __float_as_uint(v);
            atomicOr(&any[i / 32], 1u << (i % 32));
        };
        if (listed <= PEN_LIST) {
            for (int j = tid; j < listed; j += 4 * PEN_THREADS) {
                int i[4];
                float v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) i[k] = j + k * PEN_THREADS < listed ? list[j + k * PEN_THREADS] : -1;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = i[k] >= 0 ? pen_f32(x[i[k]]) : 0.0f;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i[k] >= 0) value(i[k], v[k]);
            }
        } else {
            for (int i = tid; i < n; i += PEN_THREADS)
                if (counts[i]) value(i, pen_f32(x[i]));
        }
        __syncthreads();
    }
    const float *bias = a.bias ? a.bias + row * a.bias_stride + first : nullptr;
    // element i, whose logit is v and whose bit of `any` is `has`
    auto change = [&](float v, int i, bool has) {
        if (has) v = __uint_as_float(counts[i]);
        return bias ? v + bias[i] : v;
    };
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
        if (tid + k * PEN_THREADS >= body) break;
        const int i = head + 8 * (tid + k * PEN_THREADS);
        const uint32_t has = counted ? eight_bits(any, i) : 0u;
        if (bias || has) {
#pragma unroll
            for (int j = 0; j < 8; ++j) pen_set(e[k].at()[j], change(pen_f32(e[k].at()[j]), i + j, has >> j & 1u));
        }
        if (allowed[k] != 0xffu) forbid(e[k], allowed[k]);
#pragma unroll
        for (int j = 0; j < Eight<T>::N; ++j) __stcs(reinterpret_cast<uint4 *>(y + i) + j, e[k].v[j]);
    }
    if (tid < n - 8 * body) {                                    // at most 7 of the head, 7 of the tail
        const int i = tid < head ? tid : tid + 8 * body;
        float v = change(pen_f32(x[i]), i, counted && (any[i / 32] >> (i % 32) & 1u));
        if (mask && !(mask[i / 32] >> (i % 32) & 1u)) v = -INFINITY;
        pen_set(y[i], v);
    }
}

namespace {

template <typename T>
int launch_penalize(PenaltyArgs a, int32_t rows, cudaStream_t s) {
    int dev = 0, sms = 148;
    CK(cudaGetDevice(&dev));
    CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // Slices of up to 32 KB of logits, smaller ones where they leave SMs idle.
    const int64_t least = 4 * (int64_t)sms;
    a.slice_log2 = sizeof(T) == 4 ? 13 : 14;
    while (a.slice_log2 > 11 && (int64_t)rows * ((a.vocab - 1 >> a.slice_log2) + 1) < least) --a.slice_log2;
    const int64_t slices = (a.vocab - 1 >> a.slice_log2) + 1;
    if (rows * slices > INT32_MAX) return fail(INS_EBADLEN, "penalties: too many rows in one call");
    const size_t slice = (size_t)1 << a.slice_log2;
    const size_t smem = (slice + slice / 32) * sizeof(uint32_t) + PEN_LIST * sizeof(uint16_t);
    CK(cudaFuncSetAttribute(k_penalize<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    CK(launch_after(k_penalize<T>, (unsigned)(rows * slices), (unsigned)PEN_THREADS, smem, s, a));
    return INS_OK;
}

}  // namespace
}  // namespace ins

using namespace ins;

extern "C" int ins_penalize(int32_t rows, int32_t vocab, const void *logits, int32_t dtype, int64_t stride, void *out,
                            int64_t out_stride, const ins_penalties *p, void *stream) {
    return guarded([&]() -> int {
        if (rows < 0 || vocab < 1 || vocab > PEN_MAX_VOCAB) return fail(INS_EINVAL, "penalties: rows >= 0, vocab in [1, 262144]");
        if (dtype != INS_F32 && dtype != INS_F16 && dtype != INS_BF16)
            return fail(INS_EINVAL, "penalties: logits are INS_F32, INS_F16 or INS_BF16");
        if (rows == 0) return INS_OK;
        if (!logits || !out || !p) return fail(INS_EINVAL, "penalties: NULL argument");
        if (stride < 0 || (out_stride < vocab && rows > 1))
            return fail(INS_EINVAL, "penalties: a negative row stride, or rows of the result that overlap");
        const int size = dtype == INS_F32 ? 4 : 2;
        bool aligned = (uintptr_t)logits % size == 0 && (uintptr_t)out % size == 0;
        for (const void *of_8 : {p->tokens, p->drafted}) aligned &= (uintptr_t)of_8 % 8 == 0;
        for (const void *of_4 : {(const void *)p->lengths, (const void *)p->prompts, (const void *)p->of,
                                 (const void *)p->repetition, (const void *)p->presence, (const void *)p->frequency,
                                 (const void *)p->bias, (const void *)p->mask})
            aligned &= (uintptr_t)of_4 % 4 == 0;
        if (!aligned) return fail(INS_EINVAL, "penalties: a buffer is not aligned to its elements");
        if (p->history < 0 || p->histories < 0 || p->n_drafted < 0 || p->tokens_stride < 0 || p->drafted_stride < 0 ||
            p->bias_stride < 0 || p->mask_stride < 0)
            return fail(INS_EINVAL, "penalties: a negative size or stride");
        if (p->history > PEN_MAX_HISTORY || p->n_drafted > PEN_MAX_HISTORY)
            return fail(INS_EBADLEN, "penalties: more than 2^30 tokens a row");
        if ((int64_t)p->history + p->n_drafted >= PEN_ASKED)
            return fail(INS_EBADLEN, "penalties: a row's tokens and drafted ones are 2^31, which a count does not hold");
        if (p->tokens && !p->of && p->histories != rows)
            return fail(INS_EINVAL, "penalties: " + std::to_string(p->histories) + " rows of tokens for " +
                                        std::to_string(rows) + " rows of logits");
        const PenaltyArgs a{logits, out, stride, out_stride, p->tokens, p->drafted, p->tokens_stride,
                            p->drafted_stride, p->lengths, p->prompts, p->of, p->repetition, p->presence,
                            p->frequency, p->bias, reinterpret_cast<const uint32_t *>(p->mask), p->bias_stride,
                            p->mask_stride, rows, vocab, 0, p->history, p->histories, p->drafted ? p->n_drafted : 0};
        cudaStream_t s = (cudaStream_t)stream;
        if (dtype == INS_F32) return launch_penalize<float>(a, rows, s);
        if (dtype == INS_F16) return launch_penalize<__half>(a, rows, s);
        return launch_penalize<__nv_bfloat16>(a, rows, s);
    });
}
