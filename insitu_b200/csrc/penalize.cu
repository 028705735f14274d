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
// all), then reads, changes and writes its logits. Bound by the logits' bytes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "cache.h"

namespace ins {

constexpr int PEN_THREADS = 256;
constexpr int PEN_MAX_VOCAB = 1 << 18;
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
    int32_t vocab, slice, history, histories, n_drafted;
};

__device__ __forceinline__ float pen_f32(float x) { return x; }
__device__ __forceinline__ float pen_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float pen_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T pen_to(float x);
template <>
__device__ __forceinline__ float pen_to(float x) { return x; }
template <>
__device__ __forceinline__ __half pen_to(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 pen_to(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__global__ void __launch_bounds__(PEN_THREADS) k_penalize(const PenaltyArgs a) {
    extern __shared__ __align__(16) uint32_t counts[];          // [slice] counts, then a bit each
    wait_prior_grid();
    const int slices = (a.vocab + a.slice - 1) / a.slice;
    const int64_t row = blockIdx.x / slices;
    const int first = (int)(blockIdx.x % slices) * a.slice, n = min(a.slice, a.vocab - first);
    const int tid = threadIdx.x;
    const float r = a.repetition ? a.repetition[row] : 1.0f;
    const float presence = a.presence ? a.presence[row] : 0.0f, frequency = a.frequency ? a.frequency[row] : 0.0f;
    const bool counted = r != 1.0f || presence != 0.0f || frequency != 0.0f;
    uint32_t *any = counts + a.slice;
    if (counted) {
        for (int i = tid; i < a.slice + a.slice / 32; i += PEN_THREADS) counts[i] = 0;
        __syncthreads();
        auto add = [&](int64_t token, bool asked) {
            const int64_t at = token - first;
            if (at < 0 || at >= n) return;                       // another slice's, or no token at all
            if (asked) atomicOr(&counts[at], PEN_ASKED);
            else atomicAdd(&counts[at], 1u);
            atomicOr(&any[at / 32], 1u << (at % 32));
        };
        const int64_t h = a.of ? a.of[row] : row;
        if (a.tokens && h >= 0 && h < a.histories) {
            const int len = a.lengths ? max(0, min(a.lengths[h], a.history)) : a.history;
            const int prompt = a.prompts ? a.prompts[h] : 0;
            const int64_t *t = a.tokens + h * a.tokens_stride;
            for (int i = tid; i < len; i += PEN_THREADS) add(t[i], i < prompt);
        }
        for (int i = tid; i < a.n_drafted; i += PEN_THREADS) add(a.drafted[row * a.drafted_stride + i], false);
        __syncthreads();
    }
    const T *x = static_cast<const T *>(a.logits) + row * a.stride;
    T *y = static_cast<T *>(a.out) + row * a.out_stride;
    const float *bias = a.bias ? a.bias + row * a.bias_stride : nullptr;
    const uint32_t *mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    auto change = [&](float v, int i) {
        if (counted && (any[(i - first) / 32] >> ((i - first) % 32) & 1u)) {
            const uint32_t c = counts[i - first], said = c & ~PEN_ASKED;
            v = v > 0.0f ? __fdiv_rn(v, r) : v * r;
            if (said) v = v - frequency * (float)said - presence;
        }
        if (bias) v += bias[i];
        if (mask && !(mask[i / 32] >> (i % 32) & 1u)) v = -INFINITY;
        return v;
    };
    for (int i = first + tid; i < first + n; i += PEN_THREADS) y[i] = pen_to<T>(change(pen_f32(x[i]), i));
}

namespace {

template <typename T>
int launch_penalize(PenaltyArgs a, int32_t rows, cudaStream_t s) {
    int dev = 0, sms = 148;
    CK(cudaGetDevice(&dev));
    CK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    int slices = (a.vocab + 16383) / 16384;
    while ((int64_t)rows * slices < 4 * sms && a.vocab / slices > 4096) slices *= 2;
    a.slice = ((a.vocab + slices - 1) / slices + 31) / 32 * 32;
    slices = (a.vocab + a.slice - 1) / a.slice;
    if ((int64_t)rows * slices > INT32_MAX) return fail(INS_EBADLEN, "penalties: too many rows in one call");
    const size_t smem = ((size_t)a.slice + a.slice / 32) * sizeof(uint32_t);
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
        if ((uintptr_t)logits % size || (uintptr_t)out % size || (uintptr_t)p->tokens % 8 || (uintptr_t)p->drafted % 8)
            return fail(INS_EINVAL, "penalties: a buffer is not aligned to its elements");
        if (p->history < 0 || p->histories < 0 || p->n_drafted < 0 || p->tokens_stride < 0 || p->drafted_stride < 0 ||
            p->bias_stride < 0 || p->mask_stride < 0)
            return fail(INS_EINVAL, "penalties: a negative size or stride");
        if (p->tokens && !p->of && p->histories != rows)
            return fail(INS_EINVAL, "penalties: " + std::to_string(p->histories) + " rows of tokens for " +
                                        std::to_string(rows) + " rows of logits");
        const PenaltyArgs a{logits, out, stride, out_stride, p->tokens, p->drafted, p->tokens_stride,
                            p->drafted_stride, p->lengths, p->prompts, p->of, p->repetition, p->presence,
                            p->frequency, p->bias, reinterpret_cast<const uint32_t *>(p->mask), p->bias_stride,
                            p->mask_stride, vocab, 0, p->history, p->histories, p->drafted ? p->n_drafted : 0};
        cudaStream_t s = (cudaStream_t)stream;
        if (dtype == INS_F32) return launch_penalize<float>(a, rows, s);
        if (dtype == INS_F16) return launch_penalize<__half>(a, rows, s);
        return launch_penalize<__nv_bfloat16>(a, rows, s);
    });
}
