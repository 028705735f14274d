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
// to its element (the first to 16 bytes). It refers to the arrays, which must
// outlive run(): a long one is copied once, into the pinned upload buffer.
class Plan {
  public:
    template <typename T>
    size_t add(const T *v, size_t n) {
        const size_t at = (size_ + alignof(T) - 1) / alignof(T) * alignof(T);
        parts_[n_++] = Part{at, v, n * sizeof(T)};
        size_ = at + n * sizeof(T);
        return at;
    }
    template <typename T>
    size_t add(const std::vector<T> &v) { return add(v.data(), v.size()); }

    // Makes sure that run() will find its upload buffers for a plan of up to
    // `bytes`: run() then fails only where the device does.
    static int ready(CacheBase *c, size_t bytes) {
        return bytes > (size_t)PARAM_UPLOAD_MAX ? c->stage_p.grow(bytes) : INS_OK;
    }

    // Calls `launch(src)` with the plan as PlanInline<512>, PlanInline<3840>
    // or PlanPtr; launch returns a cudaError_t.
    template <typename F>
    int run(CacheBase *c, cudaStream_t s, F &&launch) const {
        if (size_ <= 512) return inlined<512>(launch);
        if (size_ <= (size_t)PARAM_UPLOAD_MAX) return inlined<PARAM_UPLOAD_MAX>(launch);
        if (int rc = c->stage_p.reserve(size_)) return rc;
        write(static_cast<uint8_t *>(c->stage_p.h));
        if (int rc = c->stage_p.upload(size_, s)) return rc;
        CK(launch(PlanPtr{(const uint8_t *)c->stage_p.d}));
        return INS_OK;
    }

  private:
    struct Part {
        size_t at;
        const void *from;
        size_t bytes;
    };
    void write(uint8_t *to) const {
        for (int i = 0; i < n_; ++i)
            if (parts_[i].bytes) std::memcpy(to + parts_[i].at, parts_[i].from, parts_[i].bytes);
    }
    template <int N, typename F>
    int inlined(F &&launch) const {
        PlanInline<N> p;
        write(p.b);
        CK(launch(p));
        return INS_OK;
    }
    Part parts_[4];                          // as many as any plan has
    int n_ = 0;
    size_t size_ = 0;
};

}  // namespace ins
