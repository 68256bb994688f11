// Argument checks and launch helpers that the C ABI's sources share.  Host code
// that touches no GPU.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "fa_host.h"
#include "fa_mi355x_attention.h"
#include "fa_score.h"

namespace fa {
namespace {

constexpr int64_t kMaxKeyStride = int64_t(1) << 24;  // as the forward's seq stride
// Rows of a call: the kernels number the rows of whole tiles, up to 128 past the
// last one, in 31 bits.
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 256;

inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Strides of a 2-byte tensor whose rows are read in 16-byte pieces.
inline fa_status check_rows(const char* name, const void* ptr, const int64_t* st, int n) {
  if (ptr == nullptr) return fail(FA_ERR_NULL, "%s is NULL", name);
  for (int i = 0; i < n; ++i) {
    if (st[i] < 0)
      return fail(FA_ERR_STRIDE, "%s stride[%d] = %lld is negative", name, i, (long long)st[i]);
    if (st[i] % 8 != 0)
      return fail(FA_ERR_STRIDE,
                  "%s stride[%d] = %lld is not a multiple of 8 elements (16-byte rows required)",
                  name, i, (long long)st[i]);
  }
  if (!aligned(ptr, 16)) return fail(FA_ERR_STRIDE, "%s pointer is not 16-byte aligned", name);
  return FA_OK;
}

// Rows of `row` elements of a written tensor must not overlap: each stride, in
// ascending order, spans what the smaller ones reach.  (n <= 3)
inline fa_status check_written(const char* name, const int64_t* st, const int64_t* size, int n, int64_t row) {
  int order[3] = {0, 1, 2};
  std::sort(order, order + n, [&](int i, int j) { return st[i] < st[j]; });
  __int128 reach = row;
  for (int o = 0; o < n; ++o) {
    const int i = order[o];
    if (size[i] <= 1) continue;
    if (st[i] < reach)
      return fail(FA_ERR_STRIDE, "%s stride[%d] = %lld is smaller than the %lld elements it must step over"
                  " (rows overlap)", name, i, (long long)st[i], (long long)reach);
    reach += (__int128)st[i] * (size[i] - 1);
  }
  return FA_OK;
}

inline fa_status check_dtype(int32_t dtype) {
  if (dtype != FA_DTYPE_F16 && dtype != FA_DTYPE_BF16)
    return fail(FA_ERR_DTYPE, "dtype %d is not fp16 (0) or bf16 (1)", (int)dtype);
  return FA_OK;
}

inline fa_status check_head_dim(int32_t d) {
  if (d != 64 && d != 128)
    return fail(FA_ERR_HEADDIM, "Only head_dim 64 and 128 are supported (got %d)", (int)d);
  return FA_OK;
}

inline fa_status check_flag(const char* name, int32_t v) {
  if (v != 0 && v != 1) return fail(FA_ERR_ARG, "%s must be 0 or 1 (got %d)", name, (int)v);
  return FA_OK;
}

#define FA_TRY(expr)                     \
  do {                                   \
    const fa_status s_ = (expr);         \
    if (s_ != FA_OK) return s_;          \
  } while (0)

inline fa_status check_int32(const char* name, const void* p, bool required = true) {
  if (p == nullptr) return required ? fail(FA_ERR_NULL, "%s is NULL", name) : FA_OK;
  if (!aligned(p, 4)) return fail(FA_ERR_STRIDE, "%s pointer is not 4-byte aligned", name);
  return FA_OK;
}

// A normal number: the offset's headroom is divided by it; its product with
// log2(e) is finite.
inline fa_status check_scale(float scale) {
  if (!(scale >= FLT_MIN) || !(scale <= FLT_MAX / 2))
    return fail(FA_ERR_ARG, "softmax_scale must be from %g to %g (got %g)", (double)FLT_MIN,
                (double)FLT_MAX / 2, (double)scale);
  return FA_OK;
}

constexpr double kLog2e = 1.4426950408889634;
constexpr float kLeastCap = 1e-3f, kMostCap = 1e3f;

inline fa_status check_score(const fa_score_params& s, float scale) {
  if (s.softcap != 0.0f) {
    if (!(s.softcap >= kLeastCap) || !(s.softcap <= kMostCap))
      return fail(FA_ERR_ARG, "softcap must be 0 or from %g to %g (got %g)", (double)kLeastCap, (double)kMostCap,
                  (double)s.softcap);
    const double in = 2.0 * scale * kLog2e / s.softcap;
    if (in < FLT_MIN || in > FLT_MAX)
      return fail(FA_ERR_ARG, "softmax_scale / softcap = %g is out of range", (double)scale / s.softcap);
  }
  if (s.window < 0) return fail(FA_ERR_ARG, "window must be >= 0 (got %d)", (int)s.window);
  if (!aligned(s.slopes, 4)) return fail(FA_ERR_STRIDE, "slopes pointer is not 4-byte aligned");
  return FA_OK;
}

// No key is 2^30 or more from a row: such a window leaves all.
inline ScoreArgs score_args(const fa_score_params& s, float scale) {
  ScoreArgs a = {};
  if (s.softcap != 0.0f) {
    a.cap = (float)(s.softcap * kLog2e);
    a.cap_twice = 2.0f * a.cap;
    a.cap_in = (float)(2.0 * scale * kLog2e / s.softcap);
  }
  a.slope_unit = (float)(s.softcap != 0.0f ? kLog2e / a.cap_twice : 1.0 / scale);
  a.slopes = s.slopes;
  a.window = s.window < (1 << 30) ? s.window : 0;
  return a;
}

inline fa_status check_workspace(void* ws, uint64_t have, uint64_t need) {
  if (need == 0) return FA_OK;
  if (ws == nullptr)
    return fail(FA_ERR_NULL, "workspace is NULL but %llu bytes are needed", (unsigned long long)need);
  if (have < need)
    return fail(FA_ERR_ARG, "workspace of %llu bytes is smaller than the %llu bytes needed",
                (unsigned long long)have, (unsigned long long)need);
  if (!aligned(ws, 16)) return fail(FA_ERR_STRIDE, "workspace pointer is not 16-byte aligned");
  return FA_OK;
}

inline fa_status launched(hipError_t e) {
  if (e != hipSuccess) return fail(FA_ERR_HIP, "kernel launch failed: %s", hipGetErrorString(e));
  return FA_OK;
}

}  // namespace
}  // namespace fa
