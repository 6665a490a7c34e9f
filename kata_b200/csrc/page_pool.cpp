// C entry points of the host-only page table (include/kata_paged.h).
#include <exception>

#include "page_pool.hpp"

extern "C" {

int kata_pages_create(int32_t n_pages, int32_t page_size, int32_t n_seqs, int32_t max_slots, kata_pages** out) {
    if (!out) return KATA_ERR_ARG;
    *out = nullptr;
    if (n_pages < 1 || n_seqs < 1 || max_slots < 1 || max_slots > KATA_PAGED_MAX_SLOTS || page_size < 16 || page_size > 1024 || (page_size & (page_size - 1))) return KATA_ERR_ARG;
    try { *out = new kata_pages(n_pages, page_size, n_seqs, max_slots); } catch (const std::exception&) { return KATA_ERR_NOMEM; }
    return KATA_OK;
}
int kata_pages_destroy(kata_pages* p) { if (!p) return KATA_ERR_ARG; delete p; return KATA_OK; }
int kata_pages_reserve(kata_pages* p, int32_t seq, int32_t n_slots) { return p ? p->reserve(seq, n_slots) : KATA_ERR_ARG; }
int kata_pages_trim(kata_pages* p, int32_t seq, int32_t n_slots) { return p ? p->trim(seq, n_slots) : KATA_ERR_ARG; }
int kata_pages_fork(kata_pages* p, int32_t src, int32_t dst, int32_t n_slots, int32_t* copy_from, int32_t* copy_to, int32_t* copy_slots) {
    if (!p || !copy_from || !copy_to || !copy_slots) return KATA_ERR_ARG;
    return p->fork(src, dst, n_slots, *copy_from, *copy_to, *copy_slots);
}
int32_t kata_pages_count(const kata_pages* p, int32_t seq) { return p && seq >= 0 && seq < p->n_seqs ? p->count[seq] : -1; }
int32_t kata_pages_get(const kata_pages* p, int32_t seq, int32_t* out, int32_t cap) {
    if (!p || seq < 0 || seq >= p->n_seqs || cap < 0 || (cap && !out)) return -1;
    for (int32_t i = 0; i < p->count[seq] && i < cap; i++) out[i] = p->row(seq)[i];
    return p->count[seq];
}
int32_t kata_pages_free_count(const kata_pages* p) { return p ? (int32_t)p->free_heap.size() : -1; }
int32_t kata_pages_owners(const kata_pages* p, int32_t page) { return p && page >= 0 && page < p->n_pages ? p->owners[page] : -1; }

}  // extern "C"
