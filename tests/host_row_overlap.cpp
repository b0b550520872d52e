// csrc/row_overlap.h and rows_apart of csrc/paged_plan.h, for tests/test_row_overlap.py.
#include "../slai_b200/csrc/row_overlap.h"
extern "C" int host_rows_overlap(uint64_t a, int64_t ld_a, int64_t w_a, uint64_t b, int64_t ld_b, int64_t w_b, int64_t n) { return rows_overlap(a, ld_a, w_a, b, ld_b, w_b, n); }

// csrc/paged_plan.h: rows of a layer's pages
#include "../slai_b200/csrc/paged_plan.h"
extern "C" int host_rows_apart(int hs, int n_pages, int n_kv, int page_size, int64_t page_stride, int64_t head_stride, int64_t pos_stride) {
    paged::Config c = {};
    c.head_size = hs;
    c.n_pages = n_pages;
    c.n_kv_heads = n_kv;
    c.page_size = page_size;
    return paged::rows_apart(c, page_stride, head_stride, pos_stride);
}
