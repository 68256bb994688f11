// Scores of attention beside the plain scale q.k: the cap, the bias by distance
// and the window, as the host passes them and as the kernels apply them.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>

#include "fa_device_ops.h"
#endif

namespace fa {

struct ScoreArgs {
  float cap;            // softcap * log2(e); 0: none
  float cap_twice;      // twice that
  float cap_in;         // 2 softmax_scale log2(e) / softcap
  float slope_unit;     // of the scores as products, or tails, that the bias is added to: log2(e) over
                        // their factor, log2(e) softmax_scale or cap_twice
  const float* slopes;  // of each query head; NULL: no bias
  int32_t window;       // keys at a distance below it are seen; 0: all
};

#if defined(__HIPCC__)
namespace {

// The scores of a wave, to a factor: times log2(e) softmax_scale, or 2 caps in units of log2.
//   cap tanh(x) = cap - 2 cap tail,  tail = (1 - tanh(x)) / 2 = 1 / (1 + e^2x)
// The first cap is the same for all keys: it is left out and added to the logsumexp.
// The error, about 1.2e-7 cap, is that of 1 + e^2x: of no weight for scores up to some hundreds.
// Two instructions beside two of a quarter of the rate.
struct Score {
  bool capped, biased;
  float in, out, twice;  // capped: e^2x = 2^(in z), the cap, 2 caps
  __device__ __forceinline__ void init(const ScoreArgs& a) {
    capped = a.cap > 0.0f;
    biased = a.slopes != nullptr;
    in = a.cap_in;
    out = a.cap;
    twice = a.cap_twice;
  }
  __device__ __forceinline__ float tail(float z) const {
    return __builtin_amdgcn_rcpf(1.0f + dev::fast_exp2(z * in));
  }
  __device__ __forceinline__ float minus_tail(float z) const {
    return __builtin_amdgcn_rcpf(-(1.0f + dev::fast_exp2(z * in)));
  }
  // What the scores are less than those of the formula.
  __device__ __forceinline__ float left_out() const { return capped ? out : 0.0f; }
};

}  // namespace
#endif

}  // namespace fa
