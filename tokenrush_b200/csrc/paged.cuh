// Views of a paged cache and of a batch of sequences, shared by the batched append and attention kernels.
#pragma once
#include "common.cuh"

namespace trb {

constexpr int PG_MAX_SEQS = 1024;

struct PagedView {
    uint8_t *k, *v;              // codes or bf16, [num_pages, hkv, page_size, d]
    float *ks, *vs;
    int hkv, page_shift;
    long long num_pages;
};

struct BatchView {
    const int *table;
    long long table_stride;
    const void *lens;
    int lens_width, n_seqs, table_pages;
};

__host__ inline int make_paged_view(const trb_paged_t *c, PagedView *o) {
    if (!c || !c->k || !c->v) return TRB_E_ARG;
    if (c->d != 128 && c->d != 256) return TRB_E_UNSUPPORTED;
    if (c->hkv < 1 || c->num_pages < 1 || c->page_size < 1) return TRB_E_ARG;
    if (c->kv_dtype != TRB_KV_BF16 && c->kv_dtype != TRB_KV_FP8) return TRB_E_ARG;
    if (c->kv_dtype == TRB_KV_FP8 && (!c->k_scale || !c->v_scale)) return TRB_E_ARG;
    if (c->hkv > 64 || c->page_size < 16 || c->page_size > 65536 || (c->page_size & (c->page_size - 1))) return TRB_E_UNSUPPORTED;
    if (c->num_pages > 0x7fffffffLL / c->hkv) return TRB_E_UNSUPPORTED;
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return TRB_E_ALIGN;
    if (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 15) return TRB_E_ALIGN;
    o->k = (uint8_t *)c->k; o->v = (uint8_t *)c->v;
    o->ks = c->kv_dtype == TRB_KV_FP8 ? c->k_scale : nullptr;
    o->vs = c->kv_dtype == TRB_KV_FP8 ? c->v_scale : nullptr;
    o->hkv = c->hkv; o->num_pages = c->num_pages;
    o->page_shift = __builtin_ctz((unsigned)c->page_size);
    return TRB_OK;
}

__host__ inline int make_batch_view(const trb_batch_t *b, BatchView *o) {
    if (!b || !b->table || !b->lens || b->n_seqs < 1 || b->table_pages < 1) return TRB_E_ARG;
    if (b->lens_width != 4 && b->lens_width != 8) return TRB_E_ARG;
    if (b->n_seqs > PG_MAX_SEQS) return TRB_E_UNSUPPORTED;
    if (b->n_seqs > 1 && b->table_stride < b->table_pages) return TRB_E_ARG;
    if (((uintptr_t)b->table & 3) || ((uintptr_t)b->lens & (b->lens_width - 1))) return TRB_E_ALIGN;
    o->table = b->table; o->table_stride = b->table_stride; o->lens = b->lens;
    o->lens_width = b->lens_width; o->n_seqs = b->n_seqs; o->table_pages = b->table_pages;
    return TRB_OK;
}

__device__ __forceinline__ long long load_len(const BatchView &b, int i) {
    return b.lens_width == 4 ? (long long)((const int *)b.lens)[i] : ((const long long *)b.lens)[i];
}

// Rows of the prefix, and rows of one sequence's own pages, that this step may see (clamped to what the tables hold).
__device__ __forceinline__ int paged_prefix_rows(const Cursor &len, int pages, int page_shift, bool report) {
    long long n = pages > 0 ? load_cursor(len) : 0;
    const long long most = (long long)pages << page_shift;
    if (n < 0 || n > most) {
        if (report) raise_status(TRB_ST_CURSOR_RANGE);
        n = n < 0 ? 0 : most;
    }
    return (int)n;
}
__device__ __forceinline__ int paged_own_rows(const BatchView &b, int seq, int m, int page_shift, bool report) {
    const long long len = load_len(b, seq);
    if (len < 0) return -1;                                            // an empty slot
    const long long most = (long long)b.table_pages << page_shift;
    if (len > most - m) {                                              // (no sum: a length may be anything)
        if (report) raise_status(TRB_ST_CURSOR_RANGE);
        return (int)most;
    }
    return (int)(len + m);
}

}  // namespace trb
