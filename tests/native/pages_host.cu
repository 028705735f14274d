// The page operations' host side, for a runtime without a GPU (fake_cuda.cpp):
// the tests read the bookkeeping that the calls leave behind.
#include "../../insitu_b200/csrc/pages.cu"

static std::string last;
struct ins_cache : ins::CacheBase {};
int ins::fail(int code, const std::string &msg) { return last = msg, code; }
ins::CacheBase *ins::cache_base(ins_cache *c) { return c; }

extern "C" {

ins_cache *host_create(int n_kv, int page_tokens, int max_seqs, int max_pages, int n_pages) {
    ins_cache *c = new ins_cache();
    c->cfg = ins_config{};
    c->cfg.n_kv_heads = n_kv;
    c->cfg.page_tokens = page_tokens;
    c->cfg.max_seqs = max_seqs;
    c->cfg.max_pages_per_seq = max_pages;
    c->cfg.n_pages = n_pages;
    c->g = ins::Geo{};
    c->g.n_kv = n_kv;
    c->g.P = page_tokens;
    c->h_page_table = new int32_t[(size_t)max_seqs * max_pages];
    std::fill_n(c->h_page_table, (size_t)max_seqs * max_pages, -1);
    c->h_seq_lens = new int32_t[(size_t)max_seqs]();
    c->page_refs.assign((size_t)n_pages, 0);
    for (int p = n_pages - 1; p >= 0; --p) c->free_pages.push_back(p);
    c->launches = new int64_t(0);
    return c;
}
void host_destroy(ins_cache *c) {
    c->stage_p.release();
    delete[] c->h_page_table;
    delete[] c->h_seq_lens;
    delete c->launches;
    delete c;
}
const char *host_error(void) { return last.c_str(); }
const int32_t *host_table(ins_cache *c) { return c->h_page_table; }
const int32_t *host_lengths(ins_cache *c) { return c->h_seq_lens; }
const int32_t *host_refs(ins_cache *c) { return c->page_refs.data(); }
int host_free(ins_cache *c, int32_t *out) {
    std::copy(c->free_pages.begin(), c->free_pages.end(), out);
    return (int)c->free_pages.size();
}

}  // extern "C"
