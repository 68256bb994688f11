// Helpers that the sources of the _C extension share: checks of tensors, memory
// from the caching allocator, autograd.
#pragma once

#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/HIPGraphsUtils.cuh>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>

#include <cmath>
#include <initializer_list>
#include <optional>

#include "fa_mi355x_attention.h"

namespace {

using torch::Tensor;

inline void check_status(fa_status s, const char* what) {
  TORCH_CHECK(s == FA_OK, what, " failed: ", fa_status_str(s), ": ", fa_last_error());
}

inline void check_no_grad(const char* name, std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t->requires_grad(), name, " computes no gradients: call it under torch.no_grad() or detach "
                "its inputs");
}

// No call carries tangents on: none may be dropped.  (no_grad does not stop them.)
inline void check_no_tangent(const char* name, std::initializer_list<const Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(t->unsafeGetTensorImpl()->autograd_meta() == nullptr || !t->_fw_grad(0).defined(), name,
                " has no forward-mode derivative: an input has a tangent");
}

// Both, for a call without derivatives.
inline void check_no_derivative(const char* name, std::initializer_list<const Tensor*> tensors) {
  check_no_grad(name, tensors);
  check_no_tangent(name, tensors);
}

// Tensors that a call has written: a new version of each, so that an autograd
// graph that had saved one notices.  (Inference tensors have no versions.)
inline void wrote(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors)
    if (!t->is_inference()) torch::autograd::impl::bump_version(*t);
}

inline void check_half(const Tensor& t, const char* name, int64_t dims, const char* shape) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == dims, name, " must be a ", dims, "D tensor with shape ", shape);
  TORCH_CHECK(t.dtype() == torch::kFloat16 || t.dtype() == torch::kBFloat16, name,
              " must be float16 or bfloat16");
  TORCH_CHECK(t.size(dims - 1) <= 1 || t.stride(dims - 1) == 1, name,
              " must have unit stride in the last dimension");
}

inline void check_like(const Tensor& t, const char* name, const Tensor& ref) {
  TORCH_CHECK(t.device() == ref.device(), name, " must be on the same device as the others");
  TORCH_CHECK(t.dtype() == ref.dtype(), name, " must have the same dtype as the others");
}

// An int32 index tensor in rows of unit stride.
inline const int32_t* index_ptr(const Tensor& t, const char* name, int64_t dims, const Tensor& ref) {
  TORCH_CHECK(t.is_cuda() && t.device() == ref.device(), name,
              " must be a CUDA tensor on the same device as the others");
  TORCH_CHECK(t.dtype() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.dim() == dims, name, " must have ", dims, " dimension(s)");
  TORCH_CHECK(t.size(dims - 1) <= 1 || t.stride(dims - 1) == 1, name,
              " must have unit stride in the last dimension");
  return t.numel() == 0 ? nullptr : t.data_ptr<int32_t>();
}

inline int32_t int32_of(int64_t v, const char* name) {
  TORCH_CHECK(v >= INT32_MIN && v <= INT32_MAX, name, " does not fit 32 bits");
  return static_cast<int32_t>(v);
}

inline void set_strides(int64_t* out, const Tensor& t, int n) {
  for (int i = 0; i < n; ++i) out[i] = t.size(i) > 1 ? t.stride(i) : 0;
  // (the stride of a dimension of one entry means nothing, and may be anything)
}

inline void* stream_of(const Tensor& t) {
  return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

inline float scale_of(std::optional<double> scale, int64_t d) {
  return static_cast<float>(scale.value_or(1.0 / std::sqrt((double)d)));
}

// Memory from the caching allocator without the dispatcher, which costs a
// microsecond a tensor in calls whose kernels take five.
inline Tensor new_tensor(c10::IntArrayRef sizes, c10::ScalarType type, const Tensor& ref) {
  return at::detail::empty_cuda(sizes, type, ref.device(), c10::nullopt);
}
inline Tensor new_like(const Tensor& t) {
  if (!t.is_non_overlapping_and_dense()) return torch::empty_like(t);
  return at::detail::empty_strided_cuda(t.sizes(), t.strides(), t.scalar_type(), t.device());
}

inline Tensor workspace(uint64_t bytes, const Tensor& ref) {
  Tensor t;
  if (bytes > 0) t = new_tensor({(int64_t)bytes}, torch::kUInt8, ref);
  return t;
}

// A gradient as the kernel reads it: unit stride, 16-byte rows.
inline Tensor readable(const Tensor& g) {
  bool ok = g.size(3) <= 1 || g.stride(3) == 1;
  for (int i = 0; i < 3; ++i) ok = ok && (g.size(i) <= 1 || (g.stride(i) >= 0 && g.stride(i) % 8 == 0));
  ok = ok && (reinterpret_cast<uintptr_t>(g.data_ptr()) & 15u) == 0;
  return ok ? g : g.clone(at::MemoryFormat::Contiguous);
}

// Whether a leaf's gradient accumulator lives on, kept by an autograd graph,
// on another stream than the current one: a backward pass that is captured
// here would have to wait for that stream, which ends the capture.
inline bool accumulates_elsewhere(const Tensor& t) {
  if (!t.requires_grad() || !t.is_leaf()) return false;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return false;
  const auto s = node->stream();
  return s.has_value() &&
         *s != at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).unwrap();
}

// The results of a backward pass that is recorded (create_graph): a second
// derivative is refused when it is asked for.
inline torch::autograd::variable_list once(torch::autograd::variable_list out, const char* name) {
  if (!at::GradMode::is_enabled()) return out;
  for (Tensor& t : out) t.requires_grad_();
  auto refuse = std::make_shared<torch::autograd::DelayedError>(
      std::string("trying to differentiate twice ") + name + ", which is once_differentiable", out.size());
  return (*refuse)(std::move(out));
}

// In a graph capture, a call whose backward pass would have to wait for the
// stream of an older autograd graph.
inline void check_capture(const char* name, const char* instead, std::initializer_list<const Tensor*> leaves) {
  if (at::hip::currentStreamCaptureStatusMayInitCtx() == at::hip::CaptureStatus::None) return;
  for (const Tensor* t : leaves)
    TORCH_CHECK(!accumulates_elsewhere(*t), name,
                ": an autograd graph made on another stream still holds these leaves, "
                "and the backward pass of this capture would have to wait for that stream: release "
                "that graph first, or use ", instead);
}

// The scores of a call beside scale q.k.
inline fa_score_params score_params(std::optional<double> softcap, std::optional<int64_t> window,
                                    const std::optional<Tensor>& slopes, int64_t heads, const Tensor& ref) {
  fa_score_params s{};
  if (softcap) {
    TORCH_CHECK(*softcap > 0.0, "softcap must be positive (None: no cap)");
    s.softcap = static_cast<float>(*softcap);
    TORCH_CHECK(s.softcap > 0.0f, "softcap is too small");
  }
  if (window) {
    TORCH_CHECK(*window > 0, "window must be positive (None: no window)");
    s.window = static_cast<int32_t>(std::min<int64_t>(*window, INT32_MAX));
  }
  if (slopes) {
    TORCH_CHECK(slopes->is_cuda() && slopes->device() == ref.device(),
                "slopes must be a CUDA tensor on the same device as the others");
    TORCH_CHECK(slopes->dtype() == torch::kFloat32 && slopes->dim() == 1 && slopes->size(0) == heads &&
                    slopes->is_contiguous(),
                "slopes must be contiguous float32 with one entry per query head");
    s.slopes = slopes->data_ptr<float>();
  }
  return s;
}

}  // namespace
