// PyTorch host binding of attention with gradients (include/fa_mi355x_attention.h),
// part of the _C extension.
#include <string>

#include "fa_torch_common.h"

namespace {

struct Options {
  bool causal;
  std::optional<int64_t> window;
  std::optional<double> softcap, scale;
};

fa_attn_params attn_params(const Tensor& q, const Tensor& k, const Tensor& v,
                           const std::optional<Tensor>& ranges, const std::optional<Tensor>& slopes,
                           const Options& opt) {
  check_half(q, "q", 4, "[B, H, N, D]");
  check_half(k, "k", 4, "[B, H, N, D]");
  check_half(v, "v", 4, "[B, H, N, D]");
  check_like(k, "k", q);
  check_like(v, "v", q);
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have the same shape");
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(3) == k.size(3), "q and k must have the same batch and head_dim");
  fa_attn_params p{};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  set_strides(p.q_stride, q, 3);
  set_strides(p.k_stride, k, 3);
  set_strides(p.v_stride, v, 3);
  if (ranges) {
    const int64_t dims = ranges->dim();
    p.ranges = index_ptr(*ranges, "key_ranges", dims == 3 ? 3 : 2, q);
    TORCH_CHECK(ranges->size(-1) == 2 && ranges->size(-2) == q.size(2) && (dims == 2 || ranges->size(0) == q.size(0)),
                "key_ranges must have shape [N, 2] or [B, N, 2]");
    TORCH_CHECK(ranges->size(-2) <= 1 || ranges->stride(-2) == 2, "key_ranges must have contiguous rows");
    p.range_stride = dims == 3 && ranges->size(0) > 1 ? ranges->stride(0) : 0;
  }
  p.batch = int32_of(q.size(0), "batch");
  p.heads = int32_of(q.size(1), "heads");
  p.kv_heads = int32_of(k.size(1), "kv_heads");
  p.seq_len = int32_of(q.size(2), "seq_len");
  p.keys = int32_of(k.size(2), "keys");
  p.head_dim = int32_of(q.size(3), "head_dim");
  p.dtype = q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16;
  p.causal = opt.causal;
  p.softmax_scale = scale_of(opt.scale, q.size(3));
  p.score = score_params(opt.softcap, opt.window, slopes, q.size(1), q);
  return p;
}

struct Forward {
  Tensor o, lse, o_low;
};

// for_gradients: with lse and o_low.
Forward attn_forward(const Tensor& q, const Tensor& k, const Tensor& v,
                                       const std::optional<Tensor>& ranges,
                                       const std::optional<Tensor>& slopes, const Options& opt, bool with_lse,
                     bool for_gradients) {
  fa_attn_params p = attn_params(q, k, v, ranges, slopes, opt);
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor o = new_like(q), lse, o_low;
  if (with_lse || for_gradients) lse = new_tensor({q.size(0), q.size(1), q.size(2)}, torch::kFloat32, q);
  p.o = o.data_ptr();
  p.lse = lse.defined() ? lse.data_ptr<float>() : nullptr;
  if (for_gradients) o_low = new_tensor(q.sizes(), q.scalar_type(), q);
  p.o_low = for_gradients ? o_low.data_ptr() : nullptr;
  set_strides(p.o_stride, o, 3);
  check_status(fa_attn_fwd(&p, stream_of(q)), "attention");
  return {o, lse, o_low};
}

// glse and o_low may be undefined.
std::array<Tensor, 3> attn_backward(const Tensor& go, const Tensor& glse, const Tensor& q, const Tensor& k,
                                    const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& o_low,
                                    const std::optional<Tensor>& ranges, const std::optional<Tensor>& slopes,
                                    const Options& opt) {
  fa_attn_bwd_params p{};
  p.fwd = attn_params(q, k, v, ranges, slopes, opt);
  check_half(o, "o", 4, "[B, H, N, D]");
  check_like(o, "o", q);
  TORCH_CHECK(o.sizes() == q.sizes(), "o must have q's shape");
  TORCH_CHECK(go.is_cuda() && go.sizes() == q.sizes(), "o's gradient must have o's shape");
  check_like(go, "o's gradient", q);
  for (const auto& [x, name] : {std::make_pair(&lse, "lse"), std::make_pair(&glse, "lse's gradient")}) {
    if (!x->defined()) continue;
    TORCH_CHECK(x->is_cuda() && x->device() == q.device(), name, " must be on the same device as the others");
    TORCH_CHECK(x->dtype() == torch::kFloat32 && x->dim() == 3 && x->size(0) == q.size(0) &&
                    x->size(1) == q.size(1) && x->size(2) == q.size(2),
                name, " must be float32 with shape [B, H, N]");
  }
  TORCH_CHECK(lse.is_contiguous(), "lse must be contiguous");
  const c10::OptionalDeviceGuard guard(q.device());
  const Tensor g = readable(go);
  const Tensor gl = glse.defined() ? glse.contiguous() : Tensor();
  Tensor gq = new_like(q), gk = new_like(k), gv = new_like(v);
  p.fwd.o = o.data_ptr();
  p.fwd.lse = lse.data_ptr<float>();
  p.fwd.o_low = o_low.defined() ? o_low.data_ptr() : nullptr;
  set_strides(p.fwd.o_stride, o, 3);
  p.go = g.data_ptr();
  set_strides(p.go_stride, g, 3);
  p.glse = gl.defined() ? gl.data_ptr<float>() : nullptr;
  p.gq = gq.data_ptr();
  p.gk = gk.data_ptr();
  p.gv = gv.data_ptr();
  set_strides(p.gq_stride, gq, 3);
  set_strides(p.gk_stride, gk, 3);
  set_strides(p.gv_stride, gv, 3);
  uint64_t bytes = 0;
  check_status(fa_attn_bwd_workspace_size(&p, &bytes), "attention_backward");
  Tensor ws = workspace(bytes, q);
  check_status(fa_attn_bwd(&p, ws.data_ptr(), bytes, stream_of(q)), "attention_backward");
  return {gq, gk, gv};
}

std::optional<Tensor> optional_of(const Tensor& t) {
  return t.defined() ? std::optional<Tensor>(t) : std::nullopt;
}

// Attention in autograd, differentiable once in q, k and v; returns o and lse.
struct Attention : torch::autograd::Function<Attention> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q,
                                                const Tensor& k, const Tensor& v,
                                                const std::optional<Tensor>& ranges,
                                                const std::optional<Tensor>& slopes, bool causal,
                                                std::optional<int64_t> window, std::optional<double> softcap,
                                                std::optional<double> scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Forward y = attn_forward(q, k, v, ranges, slopes, Options{causal, window, softcap, scale}, true, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({q, k, v, y.o, y.lse, ranges.value_or(Tensor()), slopes.value_or(Tensor()), y.o_low});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["window"] = window;
    ctx->saved_data["softcap"] = softcap;
    ctx->saved_data["scale"] = scale;
    return {y.o, y.lse};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list g) {
    torch::autograd::variable_list out(9);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto s = ctx->get_saved_variables();
    std::array<Tensor, 3> d;
    {
      at::NoGradGuard no_grad;
      const Options opt{ctx->saved_data["causal"].toBool(), ctx->saved_data["window"].toOptional<int64_t>(),
                        ctx->saved_data["softcap"].toOptional<double>(),
                        ctx->saved_data["scale"].toOptional<double>()};
      const Tensor go = g[0].defined() ? g[0] : torch::zeros_like(s[3]);
      d = attn_backward(go, g[1], s[0], s[1], s[2], s[3], s[4], s[7], optional_of(s[5]), optional_of(s[6]), opt);
    }
    out = once({d.begin(), d.end()}, "attention");
    out.resize(9);
    return out;
  }
};

pybind11::object attention(const Tensor& q, const Tensor& k, const Tensor& v, std::optional<Tensor> ranges,
                           bool causal, std::optional<int64_t> window, std::optional<double> softcap,
                           std::optional<Tensor> slopes, std::optional<double> softmax_scale, bool return_lse) {
  check_no_tangent("attention", {&q, &k, &v});
  if (slopes) {
    check_no_tangent("attention", {&*slopes});
    TORCH_CHECK(!at::GradMode::is_enabled() || !slopes->requires_grad(), "slopes get no gradient: detach them");
  }
  Tensor o, lse;
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad())) {
    check_capture("attention", "attention_backward", {&q, &k, &v});
    const auto y = Attention::apply(q, k, v, ranges, slopes, causal, window, softcap, softmax_scale);
    o = y[0];
    lse = y[1];
  } else {
    const Forward y =
        attn_forward(q, k, v, ranges, slopes, Options{causal, window, softcap, softmax_scale}, return_lse, false);
    o = y.o;
    lse = y.lse;
  }
  if (return_lse) return pybind11::make_tuple(o, lse);
  return pybind11::cast(o);
}

pybind11::tuple attention_backward(const Tensor& go, const Tensor& q, const Tensor& k, const Tensor& v,
                                   const Tensor& o, const Tensor& lse, std::optional<Tensor> ranges, bool causal,
                                   std::optional<int64_t> window, std::optional<double> softcap,
                                   std::optional<Tensor> slopes, std::optional<double> softmax_scale,
                                   std::optional<Tensor> glse) {
  check_no_tangent("attention_backward", {&go, &q, &k, &v, &o, &lse});
  at::NoGradGuard no_grad;
  const auto d = attn_backward(go, glse.value_or(Tensor()), q, k, v, o, lse, Tensor(), ranges, slopes,
                               Options{causal, window, softcap, softmax_scale});
  return pybind11::make_tuple(d[0], d[1], d[2]);
}

}  // namespace

void bind_attention(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("attention", &attention, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("key_ranges"),
        py::arg("causal"), py::arg("window"), py::arg("softcap"), py::arg("slopes"), py::arg("softmax_scale"),
        py::arg("return_lse"));
  m.def("attention_backward", &attention_backward, py::arg("do"), py::arg("q"), py::arg("k"), py::arg("v"),
        py::arg("o"), py::arg("lse"), py::arg("key_ranges"), py::arg("causal"), py::arg("window"),
        py::arg("softcap"), py::arg("slopes"), py::arg("softmax_scale"), py::arg("dlse"));
}
