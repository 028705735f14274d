// The thin PyTorch extension over the C ABI: the per-step calls of the decode
// path (ingress, scan, and both in one call) registered as torch operators.
//
// Nothing here computes. Each operator checks its tensors, takes torch's
// current CUDA stream, calls the C ABI of libinsitu_b200.so and raises on a
// non-zero status; device memory comes from torch's allocator. The cache
// handle crosses as an int64 (the ins_cache pointer the Python mirror holds).
// The Python mirror (insitu_b200.engine.PagedCache) routes its ingress and
// scan through these operators, which keeps the per-call host work in C++.

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <utility>
#include <vector>

#include "../../include/insitu_b200.h"

namespace {

ins_cache *handle(int64_t h) {
    TORCH_CHECK(h != 0, "insitu: the cache handle is closed");
    return reinterpret_cast<ins_cache *>(static_cast<intptr_t>(h));
}

void check(int rc) {
    if (rc == INS_OK) return;
    const std::string msg = std::string("[status ") + std::to_string(rc) + "] " + ins_last_error();
    switch (rc) {
        case INS_EBADLEN:
        case INS_EINVAL:
            TORCH_CHECK_VALUE(false, msg);
        case INS_ERANGE:
        case INS_ETIMEOUT:
        default:
            TORCH_CHECK(false, msg);
    }
}

void check_i32(const at::Tensor &t, const char *name, int64_t tail0, int64_t tail1) {
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.is_contiguous(), "insitu: ", name,
                " must be a contiguous int32 CUDA tensor");
    TORCH_CHECK(t.dim() == 3 && t.size(1) == tail0 && t.size(2) == tail1, "insitu: ", name, " must be (n, ",
                tail0, ", ", tail1, "), got ", t.sizes());
}

std::vector<int32_t> ids32(at::IntArrayRef ids) {
    std::vector<int32_t> v(ids.size());
    for (size_t i = 0; i < ids.size(); ++i) {
        TORCH_CHECK(ids[i] >= INT32_MIN && ids[i] <= INT32_MAX, "insitu: sequence id out of range");
        v[i] = static_cast<int32_t>(ids[i]);
    }
    return v;
}

// ins_ingress: rotate, quantise, pack and append one token per row of k, v
// ((n, n_kv, 64) int32); q ((n, n_kv*groups, 64) int32) is rotated into the
// returned tensor, or omitted.
c10::optional<at::Tensor> ingress(int64_t h, at::IntArrayRef seq_ids, const at::Tensor &k,
                                  const at::Tensor &v, const c10::optional<at::Tensor> &q,
                                  int64_t n_kv, int64_t q_heads, bool prerotated) {
    check_i32(k, "k", n_kv, 64);
    check_i32(v, "v", n_kv, 64);
    const int64_t n = k.size(0);
    TORCH_CHECK(v.size(0) == n && (int64_t)seq_ids.size() == n, "insitu: k, v and seq_ids disagree on n");
    c10::cuda::CUDAGuard guard(k.device());
    c10::optional<at::Tensor> q_rot;
    if (q.has_value()) {
        check_i32(*q, "q", q_heads, 64);
        TORCH_CHECK(q->size(0) == n, "insitu: q carries a different token count");
        q_rot = at::empty_like(*q);
    }
    const std::vector<int32_t> ids = ids32(seq_ids);
    check(ins_ingress(handle(h), (int32_t)n, ids.data(), q.has_value() ? q->data_ptr<int32_t>() : nullptr,
                      k.data_ptr<int32_t>(), v.data_ptr<int32_t>(),
                      q_rot.has_value() ? q_rot->data_ptr<int32_t>() : nullptr,
                      prerotated ? INS_INGRESS_PREROTATED : 0u, at::cuda::getCurrentCUDAStream().stream()));
    return q_rot;
}

// ins_scan: one decode step of attention for B sequences; returns out
// ((B, q_heads, 64) int64) and, when asked, stats ((B, n_kv, 6) int64).
std::tuple<at::Tensor, c10::optional<at::Tensor>> scan(int64_t h, at::IntArrayRef seq_ids,
                                                       c10::optional<at::IntArrayRef> lengths,
                                                       const at::Tensor &q_rot, int64_t n_kv, int64_t mode,
                                                       bool with_stats) {
    TORCH_CHECK(q_rot.dim() == 3, "insitu: q_rot must be (B, q_heads, 64)");
    check_i32(q_rot, "q_rot", q_rot.size(1), 64);
    const int64_t B = q_rot.size(0);
    TORCH_CHECK((int64_t)seq_ids.size() == B, "insitu: seq_ids and q_rot disagree on B");
    c10::cuda::CUDAGuard guard(q_rot.device());
    at::Tensor out = at::empty({B, q_rot.size(1), 64}, q_rot.options().dtype(at::kLong));
    c10::optional<at::Tensor> st;
    if (with_stats) st = at::empty({B, n_kv, 6}, q_rot.options().dtype(at::kLong));
    const std::vector<int32_t> ids = ids32(seq_ids);
    const int64_t *lens = nullptr;
    if (lengths.has_value()) {
        TORCH_CHECK((int64_t)lengths->size() == B, "insitu: lengths and q_rot disagree on B");
        lens = lengths->data();
    }
    check(ins_scan(handle(h), (int32_t)B, ids.data(), lens, q_rot.data_ptr<int32_t>(), out.data_ptr<int64_t>(),
                   st.has_value() ? reinterpret_cast<ins_stats *>(st->data_ptr<int64_t>()) : nullptr,
                   static_cast<ins_softmax>(mode), at::cuda::getCurrentCUDAStream().stream()));
    return {out, st};
}

// One decode token per sequence: the ingress of q, k, v, then the scan of
// every sequence with the new token included (kernel.py:253-355 below the
// seam), in one operator call.
std::tuple<at::Tensor, c10::optional<at::Tensor>> step(int64_t h, at::IntArrayRef seq_ids, const at::Tensor &q,
                                                       const at::Tensor &k, const at::Tensor &v, int64_t n_kv,
                                                       int64_t mode, bool with_stats) {
    TORCH_CHECK(q.dim() == 3, "insitu: q must be (B, q_heads, 64)");
    c10::optional<at::Tensor> q_rot = ingress(h, seq_ids, k, v, q, n_kv, q.size(1), false);
    return scan(h, seq_ids, c10::nullopt, *q_rot, n_kv, mode, with_stats);
}

// ins_project: y = fp16(x) @ w16^T (+ bias) with fp32 products and sums;
// w16 (out, in) fp16, x (n, in) fp32, bias (out) fp32 or none -> y (n, out) fp32.
at::Tensor project(const at::Tensor &w16, const at::Tensor &x, const c10::optional<at::Tensor> &bias) {
    TORCH_CHECK(w16.is_cuda() && w16.scalar_type() == at::kHalf && w16.dim() == 2 && w16.is_contiguous(),
                "insitu: w16 must be a contiguous (out, in) float16 CUDA tensor");
    TORCH_CHECK(x.is_cuda() && x.scalar_type() == at::kFloat && x.dim() == 2 && x.is_contiguous() &&
                    x.size(1) == w16.size(1),
                "insitu: x must be a contiguous (n, in) float32 CUDA tensor");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty({x.size(0), w16.size(0)}, x.options());
    const float *b = nullptr;
    if (bias.has_value()) {
        TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->numel() == w16.size(0),
                    "insitu: bias must be a contiguous float32 tensor of out elements");
        b = bias->data_ptr<float>();
    }
    check(ins_project((int32_t)x.size(0), (int32_t)x.size(1), (int32_t)w16.size(0),
                      reinterpret_cast<const uint16_t *>(w16.data_ptr<at::Half>()), x.data_ptr<float>(), b,
                      y.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()));
    return y;
}

// Tells the allocator that the current stream reads `t`, a tensor that an
// object keeps between calls: once dropped, its memory is not reused before.
void used_here(const at::Tensor &t) {
    c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), at::cuda::getCurrentCUDAStream());
}

int32_t n_ids(at::IntArrayRef ids) {
    TORCH_CHECK(ids.size() <= INT32_MAX, "insitu: too many sequences");
    return static_cast<int32_t>(ids.size());
}

// ins_cache_fork, ins_cache_compact, ins_cache_truncate: the page operations
// of a decode step. `anchor` is a tensor on the cache's device, which selects
// the device and its current stream.
void fork(int64_t h, const at::Tensor &anchor, at::IntArrayRef src, at::IntArrayRef dst,
          c10::optional<at::IntArrayRef> lengths) {
    c10::cuda::CUDAGuard guard(anchor.device());
    TORCH_CHECK_VALUE(src.size() == dst.size() && (!lengths || lengths->size() == src.size()),
                      "insitu: src, dst and lengths disagree on their number");
    const std::vector<int32_t> s = ids32(src), d = ids32(dst);
    check(ins_cache_fork(handle(h), n_ids(src), s.data(), d.data(), lengths ? lengths->data() : nullptr,
                         at::cuda::getCurrentCUDAStream().stream()));
}

void compact(int64_t h, const at::Tensor &anchor, at::IntArrayRef seq_ids, at::IntArrayRef base,
             at::IntArrayRef counts, const at::Tensor &keep) {
    c10::cuda::CUDAGuard guard(anchor.device());
    TORCH_CHECK_VALUE(base.size() == seq_ids.size() && counts.size() == seq_ids.size(),
                      "insitu: seq_ids, base and keep disagree on their number");
    TORCH_CHECK_VALUE(keep.device().is_cpu() && keep.scalar_type() == at::kLong && keep.is_contiguous(),
                      "insitu: keep must be a contiguous int64 host tensor");
    int64_t total = 0;
    for (const int64_t n : counts) {
        TORCH_CHECK_VALUE(n >= 0 && n <= keep.numel(), "insitu: a count outside keep");
        total += n;
    }
    TORCH_CHECK_VALUE(total == keep.numel(), "insitu: the counts do not add up to keep's length");
    const std::vector<int32_t> s = ids32(seq_ids);
    check(ins_cache_compact(handle(h), n_ids(seq_ids), s.data(), base.data(), counts.data(),
                            keep.data_ptr<int64_t>(), at::cuda::getCurrentCUDAStream().stream()));
}

void truncate(int64_t h, const at::Tensor &anchor, at::IntArrayRef seq_ids, at::IntArrayRef lengths) {
    c10::cuda::CUDAGuard guard(anchor.device());
    TORCH_CHECK_VALUE(lengths.size() == seq_ids.size(), "insitu: seq_ids and lengths disagree on their number");
    const std::vector<int32_t> s = ids32(seq_ids);
    check(ins_cache_truncate(handle(h), n_ids(seq_ids), s.data(), lengths.data(),
                             at::cuda::getCurrentCUDAStream().stream()));
}

// How many rows [t0, t0 + n) of the sequences are, all of which have to be
// cached: known before a result of that size is allocated.
int64_t cached_rows(int64_t h, const std::vector<int32_t> &seq, at::IntArrayRef t0, at::IntArrayRef n) {
    int64_t total = 0;
    for (size_t i = 0; i < seq.size(); ++i) {
        const int64_t len = ins_cache_length(handle(h), seq[i]);
        TORCH_CHECK_VALUE(len >= 0, "[status ", INS_EINVAL, "] sequence id ", seq[i], " out of range");
        TORCH_CHECK_VALUE(t0[i] >= 0 && n[i] >= 0 && t0[i] <= len && n[i] <= len - t0[i], "[status ", INS_EBADLEN,
                          "] rows outside sequence ", seq[i], "'s ", len, " cached tokens");
        total += n[i];
    }
    return total;
}

// ins_cache_rows into a new (sum n, n_kv, row_bytes) uint8 tensor.
at::Tensor rows(int64_t h, const at::Tensor &anchor, at::IntArrayRef seq_ids, at::IntArrayRef t0, at::IntArrayRef n,
                int64_t n_kv, int64_t row_bytes) {
    c10::cuda::CUDAGuard guard(anchor.device());
    TORCH_CHECK_VALUE(t0.size() == seq_ids.size() && n.size() == seq_ids.size(),
                      "insitu: seq_ids, t0 and n disagree on their number");
    const std::vector<int32_t> s = ids32(seq_ids);
    at::Tensor out = at::empty({cached_rows(h, s, t0, n), n_kv, row_bytes}, anchor.options().dtype(at::kByte));
    check(ins_cache_rows(handle(h), n_ids(seq_ids), s.data(), t0.data(), n.data(), out.data_ptr<uint8_t>(),
                         at::cuda::getCurrentCUDAStream().stream()));
    return out;
}

void put_rows(int64_t h, at::IntArrayRef seq_ids, at::IntArrayRef n, const at::Tensor &rows) {
    TORCH_CHECK_VALUE(rows.is_cuda() && rows.scalar_type() == at::kByte && rows.is_contiguous(),
                      "insitu: rows must be a contiguous uint8 CUDA tensor");
    TORCH_CHECK_VALUE(n.size() == seq_ids.size(), "insitu: seq_ids and n disagree on their number");
    int64_t total = 0;
    for (const int64_t k : n) {
        TORCH_CHECK_VALUE(k >= 0 && k <= INT32_MAX, "insitu: a row count out of range");
        total += k;
    }
    TORCH_CHECK_VALUE(rows.dim() == 3 && rows.size(0) == total, "insitu: rows must hold ", total, " rows, got ",
                      rows.sizes());
    c10::cuda::CUDAGuard guard(rows.device());
    const std::vector<int32_t> s = ids32(seq_ids);
    check(ins_cache_put_rows(handle(h), n_ids(seq_ids), s.data(), n.data(), rows.data_ptr<uint8_t>(),
                             at::cuda::getCurrentCUDAStream().stream()));
}

// ins_tree_scan: attention of each sequence's last nodes[i] cached tokens as
// a drafted tree; q (sum nodes, q_heads, 64) int32 -> the same shape in bf16.
at::Tensor tree_scan(int64_t h, at::IntArrayRef seq_ids, at::IntArrayRef nodes, const at::Tensor &mask,
                     const at::Tensor &q, int64_t q_heads) {
    check_i32(q, "q", q_heads, 64);
    TORCH_CHECK_VALUE(nodes.size() == seq_ids.size(), "insitu: seq_ids and the trees disagree on their number");
    int64_t total = 0;
    for (const int64_t n : nodes) {
        TORCH_CHECK_VALUE(n >= 0 && n <= INT32_MAX, "insitu: a node count out of range");
        total += n;
    }
    TORCH_CHECK_VALUE(q.size(0) == total, "insitu: q must hold ", total, " nodes, got ", q.size(0));
    TORCH_CHECK_VALUE(mask.device() == q.device() && mask.scalar_type() == at::kLong && mask.is_contiguous() &&
                          mask.dim() == 2 && mask.size(0) == total,
                      "insitu: mask must be a contiguous int64 (nodes, words) tensor on q's device");
    c10::cuda::CUDAGuard guard(q.device());
    used_here(mask);
    const std::vector<int32_t> s = ids32(seq_ids), n = ids32(nodes);
    // (what refuses the size refuses the scan too, which says why by its status)
    const int64_t bytes = std::max<int64_t>(0, ins_tree_workspace(handle(h), n_ids(seq_ids), s.data(), n.data()));
    at::Tensor out = at::empty(q.sizes(), q.options().dtype(at::kBFloat16));
    at::Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));
    check(ins_tree_scan(handle(h), n_ids(seq_ids), s.data(), n.data(),
                        reinterpret_cast<const uint64_t *>(mask.data_ptr<int64_t>()), (int32_t)mask.size(1),
                        q.data_ptr<int32_t>(), out.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes,
                        at::cuda::getCurrentCUDAStream().stream()));
    return out;
}

// ins_chunk_scan: attention of each sequence's last counts[i] cached tokens,
// causal, under a window and sinks (window 0: none); q (sum counts, q_heads,
// 64) int32 -> the same shape in bf16.
at::Tensor chunk_scan(int64_t h, at::IntArrayRef seq_ids, at::IntArrayRef counts, int64_t window, int64_t sinks,
                      const at::Tensor &q, int64_t q_heads) {
    check_i32(q, "q", q_heads, 64);
    TORCH_CHECK_VALUE(counts.size() == seq_ids.size(), "insitu: seq_ids and counts disagree on their number");
    int64_t total = 0;
    for (const int64_t n : counts) {
        TORCH_CHECK_VALUE(n >= 0 && n <= INT32_MAX, "insitu: a token count out of range");
        total += n;
    }
    TORCH_CHECK_VALUE(q.size(0) == total, "insitu: q must hold ", total, " tokens, got ", q.size(0));
    TORCH_CHECK_VALUE(window >= 0 && window <= INT32_MAX && sinks >= 0 && sinks <= INT32_MAX,
                      "insitu: a window or a number of sinks out of range");
    c10::cuda::CUDAGuard guard(q.device());
    const std::vector<int32_t> s = ids32(seq_ids), n = ids32(counts);
    // (what refuses the size refuses the scan too, which says why by its status)
    const int64_t bytes = std::max<int64_t>(
        0, ins_chunk_workspace(handle(h), n_ids(seq_ids), s.data(), n.data(), (int32_t)window, (int32_t)sinks));
    at::Tensor out = at::empty(q.sizes(), q.options().dtype(at::kBFloat16));
    at::Tensor ws = at::empty({bytes}, q.options().dtype(at::kByte));
    check(ins_chunk_scan(handle(h), n_ids(seq_ids), s.data(), n.data(), (int32_t)window, (int32_t)sinks,
                         q.data_ptr<int32_t>(), out.data_ptr(), bytes ? ws.data_ptr() : nullptr, bytes,
                         at::cuda::getCurrentCUDAStream().stream()));
    return out;
}

int32_t element_type(at::ScalarType st) {
    TORCH_CHECK_VALUE(st == at::kFloat || st == at::kHalf || st == at::kBFloat16,
                      "insitu: the type must be float32, float16 or bfloat16, got ", st);
    return st == at::kFloat ? INS_F32 : st == at::kHalf ? INS_F16 : INS_BF16;
}

// ins_cache_dense into new (sum n, n_kv, 64) tensors k and v of `type`'s type.
std::tuple<at::Tensor, at::Tensor> dense(int64_t h, const at::Tensor &anchor, at::IntArrayRef seq_ids,
                                         at::IntArrayRef t0, at::IntArrayRef n, int64_t n_kv, at::ScalarType type,
                                         bool rotated) {
    c10::cuda::CUDAGuard guard(anchor.device());
    TORCH_CHECK_VALUE(t0.size() == seq_ids.size() && n.size() == seq_ids.size(),
                      "insitu: seq_ids, t0 and n disagree on their number");
    const int32_t dtype = element_type(type);
    const std::vector<int32_t> s = ids32(seq_ids);
    at::Tensor k = at::empty({cached_rows(h, s, t0, n), n_kv, 64}, anchor.options().dtype(type)), v = at::empty_like(k);
    check(ins_cache_dense(handle(h), n_ids(seq_ids), s.data(), t0.data(), n.data(), k.data_ptr(), v.data_ptr(), dtype,
                          rotated, at::cuda::getCurrentCUDAStream().stream()));
    return {k, v};
}

// ins_penalize: out = the logits under penalties, bias and mask; settings are
// device tensors of one value a row, or none.
void penalize(const at::Tensor &logits, const c10::optional<at::Tensor> &tokens,
                    const c10::optional<at::Tensor> &lengths, const c10::optional<at::Tensor> &prompts,
                    const c10::optional<at::Tensor> &of, const c10::optional<at::Tensor> &drafted,
                    const c10::optional<at::Tensor> &repetition, const c10::optional<at::Tensor> &presence,
                    const c10::optional<at::Tensor> &frequency, const c10::optional<at::Tensor> &bias,
                    const c10::optional<at::Tensor> &mask, const at::Tensor &out) {
    TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) < 2 || logits.stride(1) == 1),
                      "insitu: logits must be a (rows, vocab) CUDA tensor with adjacent columns");
    const int32_t dtype = element_type(logits.scalar_type());
    const int64_t n = logits.size(0), vocab = logits.size(1), words = (vocab + 31) / 32;
    TORCH_CHECK_VALUE(vocab >= 1 && vocab <= (1 << 18) && n <= (1 << 27), "insitu: vocab must be in [1, 262144], got ",
                      vocab);
    // a matrix with adjacent columns; returns its row stride
    auto matrix = [&](const at::Tensor &t, at::ScalarType type, const char *name) {
        TORCH_CHECK_VALUE(t.device() == logits.device() && t.scalar_type() == type && t.dim() == 2 &&
                              (t.size(1) < 2 || t.stride(1) == 1),
                          "insitu: ", name, " must be a 2-D ", type, " tensor with adjacent columns on logits' device");
        return t.size(0) > 1 ? t.stride(0) : 0;
    };
    // one value for each of `m` rows
    auto vector = [&](const c10::optional<at::Tensor> &t, at::ScalarType type, int64_t m, const char *name) -> void * {
        if (!t.has_value()) return nullptr;
        TORCH_CHECK_VALUE(t->device() == logits.device() && t->scalar_type() == type && t->is_contiguous() &&
                              t->dim() == 1 && t->size(0) == m,
                          "insitu: ", name, " must be a contiguous ", type, " tensor of ", m,
                          " values on logits' device");
        return t->data_ptr();
    };
    // one row for all rows of logits, or one each
    auto shared = [&](const at::Tensor &t, int64_t columns, const char *name) {
        TORCH_CHECK_VALUE(t.size(1) == columns && (t.size(0) == 1 || t.size(0) == n), "insitu: ", name,
                          " must hold 1 or ", n, " rows of ", columns, ", got ", t.sizes());
    };
    ins_penalties p{};
    if (tokens.has_value()) {
        p.tokens_stride = matrix(*tokens, at::kLong, "tokens");
        p.tokens = tokens->data_ptr<int64_t>();
        TORCH_CHECK_VALUE(tokens->size(0) <= INT32_MAX && tokens->size(1) <= INT32_MAX, "insitu: too many tokens");
        TORCH_CHECK_VALUE(of.has_value() || tokens->size(0) == n, "insitu: tokens hold ", tokens->size(0),
                          " rows; logits hold ", n);
        p.histories = (int32_t)tokens->size(0);
        p.history = (int32_t)tokens->size(1);
        p.lengths = static_cast<int32_t *>(vector(lengths, at::kInt, p.histories, "lengths"));
        p.prompts = static_cast<int32_t *>(vector(prompts, at::kInt, p.histories, "prompts"));
        p.of = static_cast<int32_t *>(vector(of, at::kInt, n, "of"));
    } else {
        TORCH_CHECK_VALUE(!lengths.has_value() && !prompts.has_value() && !of.has_value(),
                          "insitu: lengths, prompts and of need tokens");
    }
    if (drafted.has_value()) {
        p.drafted_stride = matrix(*drafted, at::kLong, "drafted");
        TORCH_CHECK_VALUE(drafted->size(0) == n && drafted->size(1) <= INT32_MAX, "insitu: drafted hold ",
                          drafted->size(0), " rows; logits hold ", n);
        p.drafted = drafted->data_ptr<int64_t>();
        p.n_drafted = (int32_t)drafted->size(1);
    }
    if (bias.has_value()) {
        p.bias_stride = matrix(*bias, at::kFloat, "bias");
        shared(*bias, vocab, "bias");
        p.bias = bias->data_ptr<float>();
    }
    if (mask.has_value()) {
        p.mask_stride = matrix(*mask, at::kInt, "mask");
        shared(*mask, words, "mask");
        p.mask = mask->data_ptr<int32_t>();
    }
    p.repetition = static_cast<float *>(vector(repetition, at::kFloat, n, "repetition"));
    p.presence = static_cast<float *>(vector(presence, at::kFloat, n, "presence"));
    p.frequency = static_cast<float *>(vector(frequency, at::kFloat, n, "frequency"));
    c10::cuda::CUDAGuard guard(logits.device());
    for (const auto *t : {&repetition, &presence, &frequency})
        if (t->has_value()) used_here(**t);
    TORCH_CHECK_VALUE(out.device() == logits.device() && out.scalar_type() == logits.scalar_type() &&
                          out.sizes() == logits.sizes() && (vocab < 2 || out.stride(1) == 1) &&
                          (n < 2 || out.stride(0) >= vocab),
                      "insitu: out must be a tensor of logits' shape, type and device whose rows do not overlap");
    auto span = [](const at::Tensor &t) {
        int64_t last = 0;
        for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
        const auto *from = static_cast<const char *>(t.data_ptr());
        return std::make_pair(from, t.numel() ? from + (last + 1) * t.element_size() : from);
    };
    const auto a = span(out);
    auto apart = [&](const at::Tensor &t) {
        const auto b = span(t);
        return a.second <= b.first || b.second <= a.first;
    };
    TORCH_CHECK_VALUE((out.data_ptr() == logits.data_ptr() && (n < 2 || out.stride(0) == logits.stride(0))) || apart(logits),
                      "insitu: out must be logits itself, or lie wholly before or after it in memory");
    // Rows of out are written while others still read what is theirs, or all
    // rows'. Other columns of the same wider rows are no overlap.
    auto beside = [&](const at::Tensor &t) {
        const int64_t size = t.element_size(), every = n > 1 ? out.stride(0) * out.element_size() : 0;
        if (every == 0 || t.dim() == 0 || (t.dim() == 2 && t.size(0) > 1 && t.stride(0) * size != every)) return false;
        const int64_t off = static_cast<const char *>(t.data_ptr()) - a.first, at = (off % every + every) % every;
        return at >= vocab * out.element_size() && at + t.size(-1) * size <= every;
    };
    for (const auto *t : {&tokens, &lengths, &prompts, &of, &drafted, &repetition, &presence, &frequency, &bias, &mask})
        TORCH_CHECK_VALUE(!t->has_value() || apart(**t) || beside(**t),
                          "insitu: out shares memory with an argument that is not logits");
    check(ins_penalize((int32_t)n, (int32_t)vocab, logits.data_ptr(), dtype, logits.stride(0), out.data_ptr(),
                       n > 1 ? out.stride(0) : vocab, &p, at::cuda::getCurrentCUDAStream().stream()));
}

// ins_sample: one token per row of logits (rows, vocab); the settings are
// device tensors of one value a row, or none.
std::tuple<at::Tensor, at::Tensor> sample(const at::Tensor &logits, const at::Tensor &uniform,
                                          const c10::optional<at::Tensor> &temperature,
                                          const c10::optional<at::Tensor> &top_k,
                                          const c10::optional<at::Tensor> &top_p,
                                          const c10::optional<at::Tensor> &min_p) {
    TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) < 2 || logits.stride(1) == 1),
                      "insitu: logits must be a (rows, vocab) CUDA tensor with adjacent columns");
    const auto st = logits.scalar_type();
    TORCH_CHECK_VALUE(st == at::kFloat || st == at::kHalf || st == at::kBFloat16,
                      "insitu: logits must be float32, float16 or bfloat16, got ", st);
    const int64_t n = logits.size(0), vocab = logits.size(1);
    TORCH_CHECK_VALUE(vocab >= 1 && vocab <= (1 << 18) && n <= (1 << 27), "insitu: vocab must be in [1, 262144], got ",
                      vocab);
    TORCH_CHECK_VALUE(uniform.device() == logits.device() && uniform.scalar_type() == at::kFloat &&
                          uniform.sizes() == logits.sizes() && (vocab < 2 || uniform.stride(1) == 1),
                      "insitu: uniform must be a float32 tensor of logits' shape and device with adjacent columns");
    auto setting = [&](const c10::optional<at::Tensor> &t, at::ScalarType type, const char *name) -> const void * {
        if (!t.has_value()) return nullptr;
        TORCH_CHECK_VALUE(t->device() == logits.device() && t->scalar_type() == type && t->is_contiguous() &&
                              t->dim() == 1 && t->size(0) == n,
                          "insitu: ", name, " must be a contiguous ", type, " tensor of ", n,
                          " values on logits' device");
        used_here(*t);
        return t->data_ptr();
    };
    c10::cuda::CUDAGuard guard(logits.device());
    const auto *t = static_cast<const float *>(setting(temperature, at::kFloat, "temperature"));
    const auto *k = static_cast<const int32_t *>(setting(top_k, at::kInt, "top_k"));
    const auto *p = static_cast<const float *>(setting(top_p, at::kFloat, "top_p"));
    const auto *m = static_cast<const float *>(setting(min_p, at::kFloat, "min_p"));
    at::Tensor tokens = at::empty({n}, logits.options().dtype(at::kLong));
    at::Tensor logprobs = at::empty({n}, logits.options().dtype(at::kFloat));
    check(ins_sample((int32_t)n, (int32_t)vocab, logits.data_ptr(),
                     st == at::kFloat ? INS_F32 : st == at::kHalf ? INS_F16 : INS_BF16, logits.stride(0),
                     uniform.data_ptr<float>(), uniform.stride(0), t, k, p, m, tokens.data_ptr<int64_t>(),
                     logprobs.data_ptr<float>(), at::cuda::getCurrentCUDAStream().stream()));
    return {tokens, logprobs};
}

}  // namespace

TORCH_LIBRARY(insitu, m) {
    m.def("fork(int handle, Tensor anchor, int[] src, int[] dst, int[]? lengths) -> ()");
    m.def("compact(int handle, Tensor anchor, int[] seq_ids, int[] base, int[] counts, Tensor keep) -> ()");
    m.def("truncate(int handle, Tensor anchor, int[] seq_ids, int[] lengths) -> ()");
    m.def("rows(int handle, Tensor anchor, int[] seq_ids, int[] t0, int[] n, int n_kv, int row_bytes) -> Tensor");
    m.def("put_rows(int handle, int[] seq_ids, int[] n, Tensor rows) -> ()");
    m.def("tree_scan(int handle, int[] seq_ids, int[] nodes, Tensor mask, Tensor q, int q_heads) -> Tensor");
    m.def("chunk_scan(int handle, int[] seq_ids, int[] counts, int window, int sinks, Tensor q, int q_heads) -> Tensor");
    m.def("dense(int handle, Tensor anchor, int[] seq_ids, int[] t0, int[] n, int n_kv, ScalarType type, "
          "bool rotated) -> (Tensor, Tensor)");
    m.def("penalize(Tensor logits, Tensor? tokens, Tensor? lengths, Tensor? prompts, Tensor? of, Tensor? drafted, "
          "Tensor? repetition, Tensor? presence, Tensor? frequency, Tensor? bias, Tensor? mask, Tensor(a!) out) -> ()");
    m.def("sample(Tensor logits, Tensor uniform, Tensor? temperature, Tensor? top_k, Tensor? top_p, "
          "Tensor? min_p) -> (Tensor, Tensor)");
    m.def("ingress(int handle, int[] seq_ids, Tensor k, Tensor v, Tensor? q, int n_kv, int q_heads, "
          "bool prerotated) -> Tensor?");
    m.def("scan(int handle, int[] seq_ids, int[]? lengths, Tensor q_rot, int n_kv, int mode, "
          "bool with_stats) -> (Tensor, Tensor?)");
    m.def("step(int handle, int[] seq_ids, Tensor q, Tensor k, Tensor v, int n_kv, int mode, "
          "bool with_stats) -> (Tensor, Tensor?)");
    m.def("project(Tensor w16, Tensor x, Tensor? bias) -> Tensor");
}

TORCH_LIBRARY_IMPL(insitu, CUDA, m) {
    m.impl("ingress", ingress);
    m.impl("scan", scan);
    m.impl("step", step);
    m.impl("project", project);
    m.impl("fork", fork);
    m.impl("compact", compact);
    m.impl("truncate", truncate);
    m.impl("rows", rows);
    m.impl("put_rows", put_rows);
    m.impl("tree_scan", tree_scan);
    m.impl("chunk_scan", chunk_scan);
    m.impl("dense", dense);
    m.impl("penalize", penalize);
    m.impl("sample", sample);
}
