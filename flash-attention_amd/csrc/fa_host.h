// Host helpers of the C ABI's sources: the error string and the device's size.
#pragma once

#include "fa_mi355x.h"

namespace fa {

// Sets fa_last_error's text and returns s.
fa_status fail(fa_status s, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
void clear_error();

// Compute units of the calling thread's current device (queried once per
// device; launch plans depend on it).
fa_status current_compute_units(int* cus);

}  // namespace fa
