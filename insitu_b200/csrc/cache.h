// The cache handle's parts that several translation units work on: error
// reporting, the per-call upload ring, and the host's page bookkeeping.
#pragma once

#include <algorithm>
#include <climits>
#include <cstring>
#include <new>
#include <stdexcept>
#include <string>
#include <vector>

#include "common.cuh"

namespace ins {

// Records the thread's error message (ins_last_error) and returns `code`.
int fail(int code, const std::string &msg);

#define CK(call)                                                                       \
    do {                                                                               \
        cudaError_t e_ = (call);                                                       \
        if (e_ != cudaSuccess)                                                         \
            return fail(INS_ECUDA, std::string(#call " failed: ") + cudaGetErrorString(e_)); \
    } while (0)

struct DeviceGuard {
    int prev = -1;
    explicit DeviceGuard(int dev) {
        cudaGetDevice(&prev);
        if (prev != dev) cudaSetDevice(dev);
    }
    ~DeviceGuard() {
        int cur = -1;
        cudaGetDevice(&cur);
        if (prev >= 0 && cur != prev) cudaSetDevice(prev);
    }
};

// Per-call uploads (sequence ids, slots, plans, positions) go through a ring
// of pinned host / device buffer pairs. reserve() moves to the next slot and
// waits only for that slot's previous copy, so the host can run NSLOT calls
// ahead of the GPU rather than one; host writes into a slot wait on that
// slot's last copy, so an enqueued copy never reads a half-rewritten area. A
// slot that must grow takes the whole ring with it, so that steady-state
// calls never allocate.
struct Staging {
    static constexpr int NSLOT = 4;
    struct Slot {
        void *h = nullptr;
        void *d = nullptr;
        cudaEvent_t done = nullptr;
    };
    Slot ring[NSLOT];
    size_t cap = 0;                     // every slot's size
    int cur = NSLOT - 1;
    void *h = nullptr;                  // the current slot's buffers
    void *d = nullptr;
    int64_t *launches = nullptr;        // the cache's kernel count (an upload may be a launch)

    // Makes room for uploads of `bytes`: what can fail of a reserve, for a call
    // that has to know before it changes anything.
    int grow(size_t bytes) {
        if (bytes <= cap) return INS_OK;
        size_t want = cap ? cap : 4096;
        while (want < bytes) want *= 2;
        for (Slot &o : ring) {
            if (!o.done) CK(cudaEventCreateWithFlags(&o.done, cudaEventDisableTiming));
            CK(cudaEventSynchronize(o.done));
            if (o.h) cudaFreeHost(o.h);
            if (o.d) cudaFree(o.d);
            o.h = o.d = nullptr;
        }
        cap = 0;
        for (Slot &o : ring)
            if (cudaHostAlloc(&o.h, want, cudaHostAllocDefault) != cudaSuccess ||
                cudaMalloc(&o.d, want) != cudaSuccess) {
                cudaGetLastError();
                return fail(INS_ENOMEM, "allocation of " + std::to_string(want) + " B of upload buffers failed");
            }
        cap = want;
        return INS_OK;
    }
    int reserve(size_t bytes) {
        if (int rc = grow(bytes)) return rc;
        cur = (cur + 1) % NSLOT;
        Slot &sl = ring[cur];
        if (!sl.done) CK(cudaEventCreateWithFlags(&sl.done, cudaEventDisableTiming));
        CK(cudaEventSynchronize(sl.done));
        h = sl.h;
        d = sl.d;
        return INS_OK;
    }
    int upload(size_t bytes, cudaStream_t s) {
        int launched = 0;
        CK(small_upload(d, h, bytes, s, &launched));
        if (launched && launches) *launches += 1;
        CK(cudaEventRecord(ring[cur].done, s));
        return INS_OK;
    }
    void release() {
        for (Slot &o : ring) {
            if (o.done) cudaEventSynchronize(o.done), cudaEventDestroy(o.done);
            if (o.h) cudaFreeHost(o.h);
            if (o.d) cudaFree(o.d);
            o = Slot();
        }
        h = d = nullptr;
        cap = 0;
    }
};

// Limits of the kernels' bounded waits and the copies held back in tests
// (ins_cache_set_wait_test).
struct WaitTest {
    int32_t poll_limit = 1 << 22;
    int32_t item = -1, chunk = 0;
};

// What the host knows of a cache's pages. A page is free (on free_pages), or
// held by page_refs[page] sequences: the ingress opens pages for one
// sequence, ins_cache_fork adds holders. Only pages full of rows are shared;
// the page that the next appended row goes to always has one holder.
struct CacheBase {
    ins_config cfg;
    Geo g;
    int device = 0;
    DevTables *d_tables = nullptr;
    uint8_t *d_pool = nullptr;
    int32_t *d_page_table = nullptr;   // [max_seqs, max_pages]
    int32_t *d_status = nullptr;
    // host mirrors (pinned, so their copies can be asynchronous)
    int32_t *h_page_table = nullptr;
    int32_t *h_seq_lens = nullptr;
    cudaEvent_t mirror_done = nullptr;
    std::vector<int32_t> free_pages;
    std::vector<int32_t> page_refs;
    Staging stage_a;                    // per-call index uploads
    Staging stage_b;
    Staging stage_c;                    // positions of ins_seam
    Staging stage_p;                    // page operations and tree plans
    int64_t *launches = nullptr;        // the handle's kernel count
    WaitTest wait;
    // the sequences whose scores an ins_scan_maxima took, while ins_scan_part
    // may still use them
    std::vector<int32_t> split_seq;
    bool split_armed = false;
    double cent_max = 0.0;              // the largest centroid's magnitude, of keys and values
    // factors in [1, 2) under which the centroids' roundings to fp16 are smallest
    float k_unit = 1.0f, v_unit = 1.0f;

    int64_t capacity() const { return (int64_t)cfg.max_pages_per_seq * cfg.page_tokens; }
    int32_t *table_row(int32_t seq) const { return h_page_table + (size_t)seq * (size_t)cfg.max_pages_per_seq; }
    int32_t open_page() {
        const int32_t pg = free_pages.back();
        free_pages.pop_back();
        page_refs[(size_t)pg] = 1;
        return pg;
    }
    // Rows of `seq` have gone or moved (rows only added change nothing).
    void rows_changed(int32_t seq) {
        if (split_armed && std::find(split_seq.begin(), split_seq.end(), seq) != split_seq.end()) split_armed = false;
    }
    void release_page(int32_t pg) {
        if (--page_refs[(size_t)pg] == 0) free_pages.push_back(pg);
    }
};

// The base of a handle (the handle's own type is private to insitu.cu).
CacheBase *cache_base(ins_cache *c);

// Runs a C entry point's body; an exception (a failed host allocation) becomes
// a status instead of leaving the C boundary.
template <typename F>
int guarded(F &&body) {
    try {
        return body();
    } catch (const std::bad_alloc &) {
        return fail(INS_ENOMEM, "host allocation failed");
    } catch (const std::exception &e) {
        return fail(INS_EINVAL, e.what());
    }
}

}  // namespace ins
