// Page operations of the compressed cache: fork, compact, truncate, and the
// copies of packed rows out of and into the pool.
//
// The host owns lengths, page tables and reference counts, so sharing and
// freeing pages costs no device work; what the device does is move rows.
// A row of one KV head is three pieces in its region's planes (K codes, V
// codes, norms), 52 bytes at 4b/2b: every kernel here reads and writes each
// moved row once, and takes its one launch's time at a few rows, and at many
// the instructions that address pieces of 8 bytes.
#include <algorithm>

#include "plan.cuh"

namespace ins {

// ---------------------------------------------------------------------------
// moving rows inside the pool
// ---------------------------------------------------------------------------

// Destination positions [lo, hi) of one sequence. The source of position d is
// d itself below `base` or when keep < 0, else base + kept[keep + d - base].
// Position p's source page is pages[old_off + p / P], its destination page
// pages[new_off + p / P].
struct MoveUnit {
    int32_t lo, hi, base, keep, old_off, new_off;
};

constexpr int MOVE_ROWS = 128;
constexpr int MOVE_THREADS = 256;

// One CTA per (unit, KV head), chunk after chunk in rising order: a chunk's
// rows are all read (into shared memory) before any is written. Within a unit
// sources rise faster than destinations (source(d) >= d), so a row that a
// chunk writes is no later chunk's source, and pages may be compacted in
// place. Units that run side by side never write a page another one reads.
// 65,536 kept rows of 131,072 into pages of their own (8 heads, 4b/2b) read and
// write 54 MB in 24 us, 2.3 TB/s: a third of what the memory does, which is 26 %
// busy, as the issue slots are 63 %: each 8 bytes take a division and a 64-bit
// address. In place the chunks follow one another: 3.4 ms.
template <class Src>
__global__ void __launch_bounds__(MOVE_THREADS) k_move_rows(Geo g, uint8_t *__restrict__ pool,
                                                            int32_t *__restrict__ table, uint32_t kept_at,
                                                            uint32_t pages_at, uint32_t entries_at,
                                                            int32_t n_entries, const __grid_constant__ Src src) {
    __shared__ __align__(16) uint8_t rows[MOVE_ROWS * (2 * D + 4)];
    __shared__ int64_t src_at[MOVE_ROWS], dst_at[MOVE_ROWS];
    __shared__ int32_t src_t[MOVE_ROWS], dst_t[MOVE_ROWS];
    wait_prior_grid();
    const int tid = threadIdx.x;
    const int2 *entries = reinterpret_cast<const int2 *>(src.data() + entries_at);
    for (int i = blockIdx.x * MOVE_THREADS + tid; i < n_entries; i += gridDim.x * MOVE_THREADS)
        table[entries[i].x] = entries[i].y;
    const int unit = blockIdx.x / g.n_kv, head = blockIdx.x % g.n_kv;
    const MoveUnit u = reinterpret_cast<const MoveUnit *>(src.data())[unit];
    const int32_t *kept = reinterpret_cast<const int32_t *>(src.data() + kept_at);
    const int32_t *pages = reinterpret_cast<const int32_t *>(src.data() + pages_at);
    uint8_t *sk = rows, *sv = rows + MOVE_ROWS * D, *sn = rows + 2 * MOVE_ROWS * D;
    const int kw = g.kbytes / 8, vw = g.vbytes / 8;
    for (int lo = u.lo; lo < u.hi; lo += MOVE_ROWS) {
        const int n = min(MOVE_ROWS, u.hi - lo);
        if (tid < n) {
            const int d = lo + tid;
            const int s = (u.keep < 0 || d < u.base) ? d : u.base + kept[u.keep + (d - u.base)];
            src_at[tid] = region_off(g, pages[u.old_off + s / g.P], head);
            dst_at[tid] = region_off(g, pages[u.new_off + d / g.P], head);
            src_t[tid] = s % g.P;
            dst_t[tid] = d % g.P;
        }
        __syncthreads();
        for (int i = tid; i < n * kw; i += MOVE_THREADS) {
            const int r = i / kw, w = i - r * kw;
            reinterpret_cast<uint2 *>(sk)[i] = *reinterpret_cast<const uint2 *>(
                pool + src_at[r] + (int64_t)src_t[r] * g.kbytes + w * 8);
        }
        for (int i = tid; i < n * vw; i += MOVE_THREADS) {
            const int r = i / vw, w = i - r * vw;
            reinterpret_cast<uint2 *>(sv)[i] = *reinterpret_cast<const uint2 *>(
                pool + src_at[r] + vplane_off(g) + (int64_t)src_t[r] * g.vbytes + w * 8);
        }
        if (tid < n)
            reinterpret_cast<uint32_t *>(sn)[tid] =
                *reinterpret_cast<const uint32_t *>(pool + src_at[tid] + nplane_off(g) + (int64_t)src_t[tid] * 4);
        __syncthreads();
        for (int i = tid; i < n * kw; i += MOVE_THREADS) {
            const int r = i / kw, w = i - r * kw;
            *reinterpret_cast<uint2 *>(pool + dst_at[r] + (int64_t)dst_t[r] * g.kbytes + w * 8) =
                reinterpret_cast<const uint2 *>(sk)[i];
        }
        for (int i = tid; i < n * vw; i += MOVE_THREADS) {
            const int r = i / vw, w = i - r * vw;
            *reinterpret_cast<uint2 *>(pool + dst_at[r] + vplane_off(g) + (int64_t)dst_t[r] * g.vbytes + w * 8) =
                reinterpret_cast<const uint2 *>(sv)[i];
        }
        if (tid < n)
            *reinterpret_cast<uint32_t *>(pool + dst_at[tid] + nplane_off(g) + (int64_t)dst_t[tid] * 4) =
                reinterpret_cast<const uint32_t *>(sn)[tid];
        __syncthreads();
    }
}

// Page-table entries alone.
template <class Src>
__global__ void __launch_bounds__(256) k_table_entries(int32_t *__restrict__ table, int32_t n,
                                                       const __grid_constant__ Src src) {
    wait_prior_grid();
    const int2 *e = reinterpret_cast<const int2 *>(src.data());
    for (int i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) table[e[i].x] = e[i].y;
}

// ---------------------------------------------------------------------------
// packed rows out of and into the pool
// ---------------------------------------------------------------------------

// Rows [t0, t0 + n) of `seq`, at row `row` of the caller's buffer; the
// sequence's tiles of ROW_TILE rows are tiles [tile, next entry's tile).
struct RowSpan {
    int32_t seq, t0, n, tile;
    int64_t row;
};

constexpr int ROW_TILE = 32, ROW_HEADS = 8;

// One CTA per (tile of 32 rows, 8 KV heads). The pool is read (or, PUT,
// written) plane by plane, 8 bytes a thread; the caller's buffer
// ([rows][n_kv][row_bytes], the packed rows of CompressedCache.buf,
// cache/compressed.py:42-52) row by row, so both sides are contiguous runs;
// shared memory holds the tile in the buffer's order. 65,536 rows of 8 heads
// (4b/2b) out take 30 us, 131,072 in 51 us, 1.8 and 2.1 TB/s of reads and
// writes: bound by instructions (66 % of the issue slots; the divisions that
// find a piece's row and head), as the pool's and the buffer's orders differ.
template <bool PUT, class Src>
__global__ void __launch_bounds__(256) k_copy_rows(Geo g, uint8_t *__restrict__ pool,
                                                   const int32_t *__restrict__ table, uint8_t *__restrict__ buf,
                                                   int32_t n_spans, const __grid_constant__ Src src) {
    __shared__ __align__(16) uint32_t sm[ROW_TILE * ROW_HEADS * (2 * D + 4) / 4];
    __shared__ int64_t at[ROW_TILE];
    __shared__ int32_t tok[ROW_TILE];
    wait_prior_grid();
    const int tid = threadIdx.x;
    const int groups = (g.n_kv + ROW_HEADS - 1) / ROW_HEADS;
    const int tile = blockIdx.x / groups, h0 = (blockIdx.x % groups) * ROW_HEADS;
    const int H = min(ROW_HEADS, g.n_kv - h0);
    const RowSpan *spans = reinterpret_cast<const RowSpan *>(src.data());
    int lo = 0, hi = n_spans - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (spans[mid].tile <= tile) lo = mid;
        else hi = mid - 1;
    }
    const RowSpan sp = spans[lo];
    const int r0 = (tile - sp.tile) * ROW_TILE, n = min(ROW_TILE, sp.n - r0);
    if (tid < n) {
        const int p = sp.t0 + r0 + tid;
        at[tid] = (int64_t)table[(int64_t)sp.seq * g.max_pages + p / g.P] * g.page_bytes;
        tok[tid] = p % g.P;
    }
    const int rw = g.row_bytes / 4, kw = g.kbytes / 8, vw = g.vbytes / 8;
    uint32_t *out = reinterpret_cast<uint32_t *>(buf) + ((sp.row + r0) * g.n_kv + h0) * rw;
    const int per = H * rw;                      // words of one row of this CTA's heads
    const int64_t stride = (int64_t)g.n_kv * rw;
    if (PUT)
        for (int i = tid; i < n * per; i += 256) sm[i] = out[(i / per) * stride + i % per];
    __syncthreads();
    // (head, row, word of 8 bytes), a head's rows side by side as in the plane
    for (int i = tid; i < H * n * kw; i += 256) {
        const int w = i % kw, r = i / kw % n, h = i / (kw * n);
        uint2 *p = reinterpret_cast<uint2 *>(pool + at[r] + (h0 + h) * g.head_bytes + (int64_t)tok[r] * g.kbytes) + w;
        uint32_t *q = sm + r * per + h * rw + 2 * w;
        if (PUT) *p = make_uint2(q[0], q[1]);
        else {
            const uint2 v = *p;
            q[0] = v.x, q[1] = v.y;
        }
    }
    for (int i = tid; i < H * n * vw; i += 256) {
        const int w = i % vw, r = i / vw % n, h = i / (vw * n);
        uint2 *p = reinterpret_cast<uint2 *>(pool + at[r] + (h0 + h) * g.head_bytes + vplane_off(g) +
                                             (int64_t)tok[r] * g.vbytes) + w;
        uint32_t *q = sm + r * per + h * rw + 2 * kw + 2 * w;
        if (PUT) *p = make_uint2(q[0], q[1]);
        else {
            const uint2 v = *p;
            q[0] = v.x, q[1] = v.y;
        }
    }
    for (int i = tid; i < H * n; i += 256) {
        const int r = i % n, h = i / n;
        uint32_t *p = reinterpret_cast<uint32_t *>(pool + at[r] + (h0 + h) * g.head_bytes + nplane_off(g) +
                                                   (int64_t)tok[r] * 4);
        uint32_t *q = sm + r * per + h * rw + 2 * (kw + vw);
        if (PUT) *p = *q;
        else *q = *p;
    }
    if (PUT) return;
    __syncthreads();
    for (int i = tid; i < n * per; i += 256) out[(i / per) * stride + i % per] = sm[i];
}

namespace {

int check_seq(const CacheBase *c, int32_t s) {
    if (s < 0 || s >= c->cfg.max_seqs) return fail(INS_EINVAL, "sequence id " + std::to_string(s) + " out of range");
    return INS_OK;
}

int check_distinct(int32_t B, const int32_t *ids) {
    std::vector<int32_t> v(ids, ids + B);
    std::sort(v.begin(), v.end());
    if (std::adjacent_find(v.begin(), v.end()) != v.end())
        return fail(INS_EINVAL, "a sequence is named twice in one call");
    return INS_OK;
}

int64_t pages_for(const CacheBase *c, int64_t rows) { return (rows + c->cfg.page_tokens - 1) / c->cfg.page_tokens; }

// The device side of a fork or a compaction: the units' moves and the
// page-table entries that changed.
struct Moves {
    std::vector<MoveUnit> units;
    std::vector<int2> entries;
    std::vector<int32_t> kept, pages;

    // the pages of positions [first page, last page] of a sequence's row
    // appended to `pages`; returns the offset that pages[off + p / P] needs
    int32_t list(const int32_t *row, int64_t p0, int64_t p1) {
        const int32_t off = (int32_t)((int64_t)pages.size() - p0);
        pages.insert(pages.end(), row + p0, row + p1 + 1);
        return off;
    }
    // Room for what the vectors have reserved, before anything changes.
    int ready(CacheBase *c) const {
        if ((int64_t)units.capacity() * c->g.n_kv > INT32_MAX) return fail(INS_EBADLEN, "too many rows in one call");
        return Plan::ready(c, units.capacity() * sizeof(MoveUnit) + entries.capacity() * sizeof(int2) +
                                  (kept.size() + pages.capacity()) * sizeof(int32_t) + 64);
    }
    int launch(CacheBase *c, cudaStream_t s) const {
        Plan plan;
        if (units.empty()) {
            if (entries.empty()) return INS_OK;
            plan.add(entries);
            const int n = (int)entries.size(), grid = std::min((n + 255) / 256, 64);
            return plan.run(c, s, [&](const auto &src) {
                *c->launches += 1;
                return launch_after(k_table_entries<std::decay_t<decltype(src)>>, (unsigned)grid, 256u, 0, s,
                                    c->d_page_table, (int32_t)n, src);
            });
        }
        plan.add(units);
        const size_t entries_at = plan.add(entries), kept_at = plan.add(kept), pages_at = plan.add(pages);
        return plan.run(c, s, [&](const auto &src) {
            *c->launches += 1;
            return launch_after(k_move_rows<std::decay_t<decltype(src)>>, (unsigned)(units.size() * c->g.n_kv),
                                (unsigned)MOVE_THREADS, 0, s, c->g, c->d_pool, c->d_page_table, (uint32_t)kept_at,
                                (uint32_t)pages_at, (uint32_t)entries_at, (int32_t)entries.size(), src);
        });
    }
};

int sync_mirror(CacheBase *c) {
    CK(cudaEventSynchronize(c->mirror_done));
    return INS_OK;
}

int fork_body(CacheBase *c, int32_t B, const int32_t *src, const int32_t *dst, const int64_t *lengths,
              cudaStream_t s) {
    const int P = c->cfg.page_tokens;
    int64_t need = 0;
    if (int rc = check_distinct(B, dst)) return rc;
    // no source may be a target too: the lengths checked here are those that
    // are taken below, and no copy reads a page that another one writes
    std::vector<int32_t> targets(dst, dst + B);
    std::sort(targets.begin(), targets.end());
    for (int32_t b = 0; b < B; ++b) {
        if (int rc = check_seq(c, src[b])) return rc;
        if (int rc = check_seq(c, dst[b])) return rc;
        if (std::binary_search(targets.begin(), targets.end(), src[b]))
            return fail(INS_EINVAL, "fork: sequence " + std::to_string(src[b]) + " is a source and a target of one call");
        if (c->h_seq_lens[dst[b]])
            return fail(INS_EINVAL, "fork: sequence " + std::to_string(dst[b]) + " is not empty");
        const int64_t len = c->h_seq_lens[src[b]], n = lengths ? lengths[b] : len;
        if (n < 0 || n > len)
            return fail(INS_EBADLEN, "fork: length " + std::to_string(n) + " outside the sequence's " +
                                         std::to_string(len) + " cached tokens");
        need += n % P != 0;
    }
    if (need > (int64_t)c->free_pages.size())
        return fail(INS_EBADLEN, "page pool exhausted: need " + std::to_string(need) + " pages, " +
                                     std::to_string(c->free_pages.size()) + " free");
    Moves m;
    const size_t row = (size_t)c->cfg.max_pages_per_seq;
    size_t n_entries = 0;
    for (int32_t b = 0; b < B; ++b)
        n_entries += (size_t)pages_for(c, lengths ? lengths[b] : c->h_seq_lens[src[b]]);
    m.entries.reserve(n_entries);
    m.units.reserve((size_t)need);
    m.pages.reserve((size_t)need * 2);
    if (int rc = m.ready(c)) return rc;
    // nothing above changed the cache; nothing below can fail before the launch
    for (int32_t b = 0; b < B; ++b) {
        const int64_t n = lengths ? lengths[b] : c->h_seq_lens[src[b]], full = n / P;
        const int32_t *from = c->table_row(src[b]);
        int32_t *to = c->table_row(dst[b]);
        for (int64_t p = 0; p < full; ++p) {
            to[p] = from[p];
            c->page_refs[(size_t)to[p]] += 1;
            m.entries.push_back(make_int2((int32_t)((size_t)dst[b] * row + (size_t)p), to[p]));
        }
        if (n % P) {
            to[full] = c->open_page();
            m.entries.push_back(make_int2((int32_t)((size_t)dst[b] * row + (size_t)full), to[full]));
            MoveUnit u{(int32_t)(full * P), (int32_t)n, 0, -1, 0, 0};
            u.old_off = m.list(from, full, full);
            u.new_off = m.list(to, full, full);
            m.units.push_back(u);
        }
        c->h_seq_lens[dst[b]] = (int32_t)n;
    }
    return m.launch(c, s);
}

int compact_body(CacheBase *c, int32_t B, const int32_t *seq, const int64_t *base, const int64_t *counts,
                 const int64_t *keep, cudaStream_t s) {
    const int P = c->cfg.page_tokens;
    if (int rc = check_distinct(B, seq)) return rc;
    Moves m;
    int64_t total = 0;
    for (int32_t b = 0; b < B; ++b) {
        if (int rc = check_seq(c, seq[b])) return rc;
        const int64_t len = c->h_seq_lens[seq[b]], n = counts ? counts[b] : 0;
        if (base[b] < 0 || base[b] > len || n < 0 || n > len - base[b])
            return fail(INS_EBADLEN, "compact: rows outside sequence " + std::to_string(seq[b]) + "'s " +
                                         std::to_string(len) + " cached tokens");
        if (n && !keep) return fail(INS_EINVAL, "compact: keep is NULL");
        // checked and narrowed in one pass (a long keep list is most of the host's work)
        m.kept.resize((size_t)(total + n));
        const int64_t *k = keep + total, last = n ? k[n - 1] : -1;
        int32_t *to = m.kept.data() + total;
        int rising = n == 0 || k[0] >= 0;
        for (int64_t i = 0; i < n; ++i) to[i] = (int32_t)k[i];
        for (int64_t i = 1; i < n; ++i) rising &= k[i] > k[i - 1];
        if (!rising) return fail(INS_EINVAL, "compact: kept rows must be distinct, in rising order, from 0");
        if (last >= len - base[b])
            return fail(INS_EBADLEN, "compact: row " + std::to_string(base[b] + last) + " outside sequence " +
                                         std::to_string(seq[b]) + "'s " + std::to_string(len) + " cached tokens");
        total += n;
    }
    // What each sequence writes: positions [first, end). Pages of that range
    // (and the page that the next append goes to) that other sequences hold
    // too are replaced by pages of its own, whose earlier rows move as well.
    struct Job {
        int64_t first, end, p0, p1;      // written positions, pages [p0, p1) to examine
        int64_t keep_at;
        bool fresh;                      // every written page is a new one
    };
    std::vector<Job> jobs((size_t)B);
    int64_t need = 0, kept_at = 0;
    for (int32_t b = 0; b < B; ++b) {
        const int64_t n = counts ? counts[b] : 0, end = base[b] + n;
        int64_t same = 0;
        while (same < n && keep[kept_at + same] == same) ++same;
        Job &j = jobs[(size_t)b];
        j.first = base[b] + same;
        j.end = end;
        j.keep_at = kept_at;
        j.p0 = j.first < end ? j.first / P : (end % P ? end / P : pages_for(c, end));
        j.p1 = pages_for(c, end);
        j.fresh = true;
        kept_at += n;
        int64_t own = 0;
        for (int64_t p = j.p0; p < j.p1; ++p) {
            const bool shared = c->page_refs[(size_t)c->table_row(seq[b])[p]] > 1;
            need += shared;
            own += !shared;
        }
        j.fresh = own == 0;
    }
    if (need > (int64_t)c->free_pages.size())
        return fail(INS_EBADLEN, "page pool exhausted: need " + std::to_string(need) + " pages, " +
                                     std::to_string(c->free_pages.size()) + " free");
    // A long compaction within a sequence's own pages runs in order, one CTA
    // a head; into new pages it runs in parallel. So where it moves more than
    // a few chunks and the pool has room, it takes new pages too: every second
    // of 1,200 rows (8 heads) 9 us, in place 22; of 4,096 rows 32 and 74.
    int64_t room = (int64_t)c->free_pages.size() - need;
    for (int32_t b = 0; b < B; ++b) {
        Job &j = jobs[(size_t)b];
        if (j.fresh || j.end - j.first <= 4 * MOVE_ROWS) continue;
        int64_t more = 0;
        for (int64_t p = j.p0; p < j.p1; ++p) more += c->page_refs[(size_t)c->table_row(seq[b])[p]] == 1;
        if (more > room) continue;
        room -= more;
        j.fresh = true;
    }
    const size_t row = (size_t)c->cfg.max_pages_per_seq;
    // every allocation the plan needs happens before the cache changes
    size_t n_pages = 0, n_units = 0, n_listed = 0, n_dropped = 0;
    for (int32_t b = 0; b < B; ++b) {
        const Job &j = jobs[(size_t)b];
        n_pages += (size_t)(j.p1 - j.p0);
        n_units += j.p0 >= j.p1 ? 0 : j.fresh ? (size_t)((j.end - j.p0 * P + MOVE_ROWS - 1) / MOVE_ROWS) : 1;
        const size_t from_p0 = (size_t)(pages_for(c, c->h_seq_lens[seq[b]]) - j.p0);
        n_dropped += from_p0;
        n_listed += j.p0 < j.p1 ? from_p0 + (size_t)(j.p1 - j.p0) : 0;
    }
    std::vector<int32_t> dropped;
    m.units.reserve(n_units);
    m.entries.reserve(n_pages);
    m.pages.reserve(n_listed);
    dropped.reserve(n_dropped);
    if (int rc = m.ready(c)) return rc;
    bool any_kept = false;
    for (int32_t b = 0; b < B; ++b) {
        const Job &j = jobs[(size_t)b];
        int32_t *tab = c->table_row(seq[b]);
        const int64_t held = pages_for(c, c->h_seq_lens[seq[b]]);
        const int32_t old_off = j.p0 < j.p1 ? m.list(tab, j.p0, held - 1) : 0;
        bool replaced_first = false;
        for (int64_t p = j.p0; p < j.p1; ++p) {
            // reference counts as they were at the call: pages dropped below
            // are released only after every sequence has its own
            if (c->page_refs[(size_t)tab[p]] == 1 && !(j.fresh && j.first < j.end)) continue;
            dropped.push_back(tab[p]);
            tab[p] = c->open_page();
            m.entries.push_back(make_int2((int32_t)((size_t)seq[b] * row + (size_t)p), tab[p]));
            replaced_first |= p == j.p0;
        }
        for (int64_t p = j.p1; p < held; ++p) {
            dropped.push_back(tab[p]);
            tab[p] = -1;
        }
        if (j.first < j.end || j.end < c->h_seq_lens[seq[b]]) c->rows_changed(seq[b]);
        c->h_seq_lens[seq[b]] = (int32_t)j.end;
        if (j.p0 >= j.p1) continue;
        // a replaced page's rows before the first moved one come along
        const int64_t lo = replaced_first ? j.p0 * P : j.first;
        if (lo >= j.end) continue;
        MoveUnit u{(int32_t)lo, (int32_t)j.end, (int32_t)base[b], j.first < j.end ? (int32_t)j.keep_at : -1, old_off, 0};
        u.new_off = m.list(tab, j.p0, j.p1 - 1);
        any_kept |= u.keep >= 0;
        if (!j.fresh) {
            m.units.push_back(u);
            continue;
        }
        for (int64_t x = lo; x < j.end; x += MOVE_ROWS) {
            u.lo = (int32_t)x;
            u.hi = (int32_t)std::min<int64_t>(x + MOVE_ROWS, j.end);
            m.units.push_back(u);
        }
    }
    for (int32_t pg : dropped) c->release_page(pg);
    if (!any_kept) m.kept.clear();
    return m.launch(c, s);
}

int rows_launch(CacheBase *c, const std::vector<RowSpan> &spans, int64_t tiles, uint8_t *buf, bool put,
                cudaStream_t s) {
    const int64_t grid = tiles * ((c->g.n_kv + ROW_HEADS - 1) / ROW_HEADS);
    if (grid == 0) return INS_OK;
    if (grid > INT32_MAX) return fail(INS_EBADLEN, "too many rows in one call");
    Plan plan;
    plan.add(spans);
    return plan.run(c, s, [&](const auto &src) {
        using S = std::decay_t<decltype(src)>;
        *c->launches += 1;
        return launch_after(put ? k_copy_rows<true, S> : k_copy_rows<false, S>, (unsigned)grid, 256u, 0, s, c->g,
                            c->d_pool, (const int32_t *)c->d_page_table, buf, (int32_t)spans.size(), src);
    });
}

int rows_body(CacheBase *c, int32_t B, const int32_t *seq, const int64_t *t0, const int64_t *n, uint8_t *rows,
              cudaStream_t s) {
    std::vector<RowSpan> spans;
    spans.reserve((size_t)B);
    int64_t tiles = 0, total = 0;
    for (int32_t b = 0; b < B; ++b) {
        if (int rc = check_seq(c, seq[b])) return rc;
        const int64_t len = c->h_seq_lens[seq[b]];
        if (t0[b] < 0 || n[b] < 0 || t0[b] > len || n[b] > len - t0[b])
            return fail(INS_EBADLEN, "rows outside sequence " + std::to_string(seq[b]) + "'s " + std::to_string(len) +
                                         " cached tokens");
        if (n[b] == 0) continue;
        spans.push_back(RowSpan{seq[b], (int32_t)t0[b], (int32_t)n[b], (int32_t)tiles, total});
        tiles += (n[b] + ROW_TILE - 1) / ROW_TILE;
        total += n[b];
        if (tiles > INT32_MAX) return fail(INS_EBADLEN, "too many rows in one call");
    }
    if (total && !rows) return fail(INS_EINVAL, "rows is NULL");
    return rows_launch(c, spans, tiles, rows, false, s);
}

int put_rows_body(CacheBase *c, int32_t B, const int32_t *seq, const int64_t *n, const uint8_t *rows,
                  cudaStream_t s) {
    if (int rc = check_distinct(B, seq)) return rc;
    int64_t need = 0, total = 0;
    for (int32_t b = 0; b < B; ++b) {
        if (int rc = check_seq(c, seq[b])) return rc;
        const int64_t len = c->h_seq_lens[seq[b]];
        if (n[b] < 0 || n[b] > c->capacity() - len)
            return fail(INS_EBADLEN, "cache holds " + std::to_string(len) + " of " + std::to_string(c->capacity()) +
                                         " tokens for sequence " + std::to_string(seq[b]) + "; cannot append " +
                                         std::to_string(n[b]));
        need += pages_for(c, len + n[b]) - pages_for(c, len);
        total += n[b];
    }
    if (total && !rows) return fail(INS_EINVAL, "rows is NULL");
    if (need > (int64_t)c->free_pages.size())
        return fail(INS_EBADLEN, "page pool exhausted: need " + std::to_string(need) + " pages, " +
                                     std::to_string(c->free_pages.size()) + " free");
    std::vector<RowSpan> spans;
    Moves m;
    spans.reserve((size_t)B);
    m.entries.reserve((size_t)need);
    int64_t tiles = 0;
    for (int32_t b = 0; b < B; ++b) tiles += (n[b] + ROW_TILE - 1) / ROW_TILE;
    if (tiles * ((c->g.n_kv + ROW_HEADS - 1) / ROW_HEADS) > INT32_MAX)
        return fail(INS_EBADLEN, "too many rows in one call");
    if (int rc = Plan::ready(c, std::max((size_t)need * sizeof(int2), (size_t)B * sizeof(RowSpan)) + 64)) return rc;
    tiles = total = 0;
    const size_t row = (size_t)c->cfg.max_pages_per_seq;
    for (int32_t b = 0; b < B; ++b) {
        if (n[b] == 0) continue;
        const int64_t len = c->h_seq_lens[seq[b]];
        int32_t *tab = c->table_row(seq[b]);
        for (int64_t p = pages_for(c, len); p < pages_for(c, len + n[b]); ++p) {
            tab[p] = c->open_page();
            m.entries.push_back(make_int2((int32_t)((size_t)seq[b] * row + (size_t)p), tab[p]));
        }
        c->h_seq_lens[seq[b]] = (int32_t)(len + n[b]);
        spans.push_back(RowSpan{seq[b], (int32_t)len, (int32_t)n[b], (int32_t)tiles, total});
        tiles += (n[b] + ROW_TILE - 1) / ROW_TILE;
        total += n[b];
    }
    if (int rc = m.launch(c, s)) return rc;
    return rows_launch(c, spans, tiles, const_cast<uint8_t *>(rows), true, s);
}

template <typename F>
int entry(ins_cache *cache, int32_t B, bool args, F &&body) {
    if (!cache) return fail(INS_EINVAL, "cache is NULL");
    if (B < 0 || (B > 0 && !args)) return fail(INS_EINVAL, "page operation arguments");
    if (B == 0) return INS_OK;
    CacheBase *c = cache_base(cache);
    return guarded([&] {
        DeviceGuard dg(c->device);
        if (int rc = sync_mirror(c)) return rc;
        return body(c);
    });
}

}  // namespace
}  // namespace ins

using namespace ins;

extern "C" {

int64_t ins_cache_free_pages(const ins_cache *cache) {
    return cache ? (int64_t)cache_base(const_cast<ins_cache *>(cache))->free_pages.size() : -1;
}

int ins_cache_fork(ins_cache *cache, int32_t B, const int32_t *src, const int32_t *dst, const int64_t *lengths,
                   void *stream) {
    return entry(cache, B, src && dst,
                 [&](CacheBase *c) { return fork_body(c, B, src, dst, lengths, (cudaStream_t)stream); });
}

int ins_cache_compact(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int64_t *base,
                      const int64_t *counts, const int64_t *keep, void *stream) {
    return entry(cache, B, seq_ids && base && counts, [&](CacheBase *c) {
        return compact_body(c, B, seq_ids, base, counts, keep, (cudaStream_t)stream);
    });
}

int ins_cache_truncate(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int64_t *lengths, void *stream) {
    return entry(cache, B, seq_ids && lengths, [&](CacheBase *c) {
        return compact_body(c, B, seq_ids, lengths, nullptr, nullptr, (cudaStream_t)stream);
    });
}

int ins_cache_rows(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int64_t *t0, const int64_t *n,
                   uint8_t *rows, void *stream) {
    if ((uintptr_t)rows & 3u) return fail(INS_EINVAL, "rows must be 4-byte aligned");
    return entry(cache, B, seq_ids && t0 && n,
                 [&](CacheBase *c) { return rows_body(c, B, seq_ids, t0, n, rows, (cudaStream_t)stream); });
}

int ins_cache_put_rows(ins_cache *cache, int32_t B, const int32_t *seq_ids, const int64_t *n, const uint8_t *rows,
                       void *stream) {
    if ((uintptr_t)rows & 3u) return fail(INS_EINVAL, "rows must be 4-byte aligned");
    return entry(cache, B, seq_ids && n,
                 [&](CacheBase *c) { return put_rows_body(c, B, seq_ids, n, rows, (cudaStream_t)stream); });
}

}  // extern "C"
