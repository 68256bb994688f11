// Host helpers of the C ABI's sources and of the binding: the error string, the
// device's size, tensors that share memory.
#pragma once

#include <stdint.h>

#include "fa_mi355x.h"

namespace fa {

// Sets fa_last_error's text and returns s.
fa_status fail(fa_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();

// Compute units of the calling thread's current device (queried once per
// device; launch plans depend on it).
fa_status current_compute_units(int* cus);

// Rows of 2-byte elements, contiguous each, of up to three dimensions; strides in
// elements, not negative.
struct RowSet {
  const void* base;
  int64_t stride[3], size[3];
  int n;
  int64_t row;
};
// Whether two sets of rows share an element.  Exact for rows of the same strides
// that do not overlap among themselves (views of one buffer); else true unless
// their addresses, whole or modulo all strides, keep them apart.
bool may_overlap(const RowSet& a, const RowSet& b);

}  // namespace fa
