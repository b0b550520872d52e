// csrc/row_overlap.h for tests/test_row_overlap.py.
#include "../slai_b200/csrc/row_overlap.h"
extern "C" int host_rows_overlap(uint64_t a, int64_t ld_a, int64_t w_a, uint64_t b, int64_t ld_b, int64_t w_b, int64_t n) { return rows_overlap(a, ld_a, w_a, b, ld_b, w_b, n); }
