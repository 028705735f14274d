// A call's host-built plan (a few descriptors), carried to its kernel.
//
// Up to PARAM_UPLOAD_MAX bytes ride in the kernel's own parameter (one launch
// in all); more go through the handle's upload ring and the kernel gets a
// pointer. A kernel takes the plan as a template parameter `Src` and reads it
// through data().
#pragma once

#include <cstring>
#include <vector>

#include "cache.h"

namespace ins {

template <int N>
struct PlanInline {
    alignas(16) uint8_t b[N];
    __device__ __forceinline__ const uint8_t *data() const { return b; }
};
struct PlanPtr {
    const uint8_t *p;
    __device__ __forceinline__ const uint8_t *data() const { return p; }
};

// The plan under construction: typed arrays one after another, each aligned
// to its element (the first to 16 bytes).
class Plan {
  public:
    template <typename T>
    size_t add(const T *v, size_t n) {
        const size_t at = (bytes_.size() + alignof(T) - 1) / alignof(T) * alignof(T);
        bytes_.resize(at + n * sizeof(T));
        if (n) std::memcpy(bytes_.data() + at, v, n * sizeof(T));
        return at;
    }
    template <typename T>
    size_t add(const std::vector<T> &v) { return add(v.data(), v.size()); }

    // Calls `launch(src)` with the plan as PlanInline<512>, PlanInline<3840>
    // or PlanPtr; launch returns a cudaError_t.
    template <typename F>
    int run(CacheBase *c, cudaStream_t s, F &&launch) const {
        const size_t n = bytes_.size();
        if (n <= 512) return inlined<512>(launch);
        if (n <= (size_t)PARAM_UPLOAD_MAX) return inlined<PARAM_UPLOAD_MAX>(launch);
        if (int rc = c->stage_p.reserve(n)) return rc;
        std::memcpy(c->stage_p.h, bytes_.data(), n);
        if (int rc = c->stage_p.upload(n, s)) return rc;
        CK(launch(PlanPtr{(const uint8_t *)c->stage_p.d}));
        return INS_OK;
    }

  private:
    template <int N, typename F>
    int inlined(F &&launch) const {
        PlanInline<N> p;
        if (!bytes_.empty()) std::memcpy(p.b, bytes_.data(), bytes_.size());
        CK(launch(p));
        return INS_OK;
    }
    std::vector<uint8_t> bytes_;
};

}  // namespace ins
