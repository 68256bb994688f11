// fa::may_overlap of libfa_mi355x.so for tests/test_row_overlap.py.
#include <stdint.h>

#include "fa_host.h"

// base in bytes; stride and size of n dimensions, rows of `row` elements of 2 bytes
extern "C" int row_overlap(int64_t base_a, const int64_t* stride_a, const int64_t* size_a, int n_a, int64_t row_a,
                           int64_t base_b, const int64_t* stride_b, const int64_t* size_b, int n_b, int64_t row_b) {
  fa::RowSet a = {reinterpret_cast<const void*>(base_a), {}, {}, n_a, row_a};
  fa::RowSet b = {reinterpret_cast<const void*>(base_b), {}, {}, n_b, row_b};
  for (int i = 0; i < n_a; ++i) a.stride[i] = stride_a[i], a.size[i] = size_a[i];
  for (int i = 0; i < n_b; ++i) b.stride[i] = stride_b[i], b.size[i] = size_b[i];
  return fa::may_overlap(a, b);
}
