// PyTorch host binding of the paged cache's operators and of the q/k norm with
// rotation (include/fa_mi355x_cache.h), part of the _C extension.  As
// fa_torch_ext.cpp it holds no kernels: tensors become parameter blocks,
// workspaces come from torch's caching allocator on the current stream of the
// tensors' device.
#include <array>
#include <cstring>
#include <string>
#include <utility>

#include "fa_host.h"
#include "fa_torch_common.h"

namespace {

fa_paged_cache make_cache(const Tensor& k, const std::optional<Tensor>& v, const Tensor& table,
                          const std::optional<Tensor>& cu, const Tensor& lens) {
  check_half(k, "k_cache", 4, "[pages, kv_heads, page_size, head_dim]");
  fa_paged_cache c{};
  c.k = k.data_ptr();
  set_strides(c.k_stride, k, 3);
  if (v) {
    check_half(*v, "v_cache", 4, "[pages, kv_heads, page_size, head_dim]");
    check_like(*v, "v_cache", k);
    TORCH_CHECK(v->sizes() == k.sizes(), "k_cache and v_cache must have the same shape");
    c.v = v->data_ptr();
    set_strides(c.v_stride, *v, 3);
  }
  c.block_table = index_ptr(table, "block_table", 2, k);
  c.seq_lens = index_ptr(lens, "seq_lens", 1, k);
  TORCH_CHECK(lens.size(0) == table.size(0), "seq_lens must have one entry per row of block_table");
  if (cu) {
    c.cu_seqlens = index_ptr(*cu, "cu_seqlens", 1, k);
    TORCH_CHECK(cu->size(0) == table.size(0) + 1,
                "cu_seqlens must have one entry more than block_table has rows");
  }
  c.table_stride = table.stride(0);
  c.batch = int32_of(table.size(0), "batch");
  c.max_pages = int32_of(table.size(1), "block_table's width");
  c.num_pages = int32_of(k.size(0), "the number of pages");
  c.kv_heads = int32_of(k.size(1), "kv_heads");
  c.page_size = int32_of(k.size(2), "page_size");
  c.head_dim = int32_of(k.size(3), "head_dim");
  c.dtype = k.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16;
  return c;
}

int32_t kv_limit(const fa_paged_cache& c, std::optional<int64_t> max_kv) {
  const int64_t all = (int64_t)c.max_pages * c.page_size;
  return int32_of(max_kv.value_or(std::min<int64_t>(all, INT32_MAX)), "max_kv");
}

void check_packed(const Tensor& t, const char* name, const Tensor& k, int64_t tokens = -1,
                  int64_t heads = -1) {
  check_half(t, name, 3, "[tokens, heads, head_dim]");
  check_like(t, name, k);
  TORCH_CHECK(t.size(2) == k.size(3), name, " must have the cache's head_dim");
  TORCH_CHECK(tokens < 0 || t.size(0) == tokens, name, " must have as many tokens as q");
  TORCH_CHECK(heads < 0 || t.size(1) == heads, name, " has the wrong number of heads");
}

// The rows of a tensor of 2-byte elements with unit stride along its last
// dimension (check_half), and the end of their memory.
struct Rows : fa::RowSet {
  const char* end;
  explicit Rows(const Tensor& t) : RowSet{t.data_ptr(), {}, {}, (int)t.dim() - 1, t.sizes().back()} {
    const auto sizes = t.sizes(), strides = t.strides();
    int64_t reach = row;
    for (int d = 0; d < n; ++d) {
      stride[d] = strides[d];
      size[d] = sizes[d];
      reach += stride[d] * (size[d] - 1);
    }
    end = static_cast<const char*>(base) + 2 * reach;
  }
};

// `out` is written while the call still reads `in`.  (Nearly always their memory
// is apart as a whole, which is seen here.)
void check_apart(const Rows& out, const char* out_name, const Rows& in, const char* in_name) {
  if (out.end <= in.base || in.end <= out.base) return;
  TORCH_CHECK(!fa::may_overlap(out, in), out_name, " must not overlap ", in_name);
}

// A result in the place of its input, row for row.
bool same_rows(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.sizes() != b.sizes()) return false;
  for (int d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

float* key_weight_ptr(const Tensor& w, const Tensor& k, int64_t stride[2]) {
  TORCH_CHECK(w.is_cuda() && w.device() == k.device(),
              "key_weights must be a CUDA tensor on the same device as the others");
  TORCH_CHECK(w.dtype() == torch::kFloat32, "key_weights must be float32");
  TORCH_CHECK(w.dim() == 3 && w.size(0) == k.size(0) && w.size(1) == k.size(1) && w.size(2) == k.size(2),
              "key_weights must have shape [pages, kv_heads, page_size]");
  TORCH_CHECK(w.stride(2) == 1 || w.size(2) == 1,
              "key_weights must have unit stride in the last dimension");
  set_strides(stride, w, 2);
  return w.data_ptr<float>();
}

const float* lse_ptr(const Tensor& lse, const Tensor& q) {
  TORCH_CHECK(lse.is_cuda() && lse.device() == q.device(),
              "lse must be a CUDA tensor on the same device as the others");
  TORCH_CHECK(lse.dtype() == torch::kFloat32 && lse.is_contiguous(), "lse must be contiguous float32");
  TORCH_CHECK(lse.dim() == 2 && lse.size(0) == q.size(0) && lse.size(1) == q.size(1),
              "lse must have shape [tokens, heads]");
  return lse.data_ptr<float>();
}

pybind11::object paged_forward(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache,
                              const Tensor& block_table, const Tensor& cu_seqlens,
                              const Tensor& seq_lens, std::optional<Tensor> out, int64_t max_q,
                              std::optional<int64_t> max_kv, bool causal,
                              std::optional<double> softmax_scale, bool return_lse,
                              std::optional<double> softcap, std::optional<int64_t> window,
                              std::optional<Tensor> slopes) {
  check_no_derivative("paged_forward", {&q, &k_cache, &v_cache});
  if (slopes) check_no_derivative("paged_forward", {&*slopes});
  if (out) check_no_derivative("paged_forward", {&*out});
  fa_paged_fwd_params p{};
  p.cache = make_cache(k_cache, v_cache, block_table, cu_seqlens, seq_lens);
  check_packed(q, "q", k_cache);
  const c10::OptionalDeviceGuard guard(q.device());
  if (out) {
    check_packed(*out, "out", k_cache, q.size(0), q.size(1));
    TORCH_CHECK(!out->is_alias_of(q) || out->data_ptr() != q.data_ptr() || out->numel() == 0,
                "out must not be q");
    const Rows rows(*out);
    check_apart(rows, "out", Rows(q), "q");
    check_apart(rows, "out", Rows(k_cache), "k_cache");
    check_apart(rows, "out", Rows(v_cache), "v_cache");
  }
  Tensor o = out ? *out : new_tensor(q.sizes(), q.scalar_type(), q);
  Tensor lse;
  if (return_lse) lse = new_tensor({q.size(0), q.size(1)}, torch::kFloat32, q);
  p.q = q.data_ptr();
  p.o = o.data_ptr();
  p.lse = return_lse ? lse.data_ptr<float>() : nullptr;
  set_strides(p.q_stride, q, 2);
  set_strides(p.o_stride, o, 2);
  p.tokens = int32_of(q.size(0), "tokens");
  p.heads = int32_of(q.size(1), "heads");
  p.max_q = int32_of(max_q, "max_q");
  p.max_kv = kv_limit(p.cache, max_kv);
  p.softmax_scale = scale_of(softmax_scale, q.size(2));
  p.causal = causal;
  const fa_score_params score = score_params(softcap, window, slopes, q.size(1), q);
  uint64_t bytes = 0;
  check_status(fa_paged_fwd_scored_workspace_size(&p, &score, &bytes), "paged_forward");
  Tensor ws = workspace(bytes, q);
  check_status(fa_paged_fwd_scored(&p, &score, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
               "paged_forward");
  if (out) wrote({&o});
  if (return_lse) return pybind11::make_tuple(o, lse);
  return pybind11::cast(o);
}

void paged_key_weights(const Tensor& q, const Tensor& lse, const Tensor& k_cache,
                       const Tensor& block_table, const Tensor& cu_seqlens, const Tensor& seq_lens,
                       Tensor key_weights, int64_t max_q, std::optional<int64_t> max_kv, bool causal,
                       std::optional<double> softmax_scale) {
  check_no_derivative("paged_key_weights", {&q, &lse, &k_cache, &key_weights});
  fa_paged_weights_params p{};
  p.cache = make_cache(k_cache, std::nullopt, block_table, cu_seqlens, seq_lens);
  check_packed(q, "q", k_cache);
  const c10::OptionalDeviceGuard guard(q.device());
  p.q = q.data_ptr();
  p.lse = lse_ptr(lse, q);
  p.key_weights = key_weight_ptr(key_weights, k_cache, p.w_stride);
  set_strides(p.q_stride, q, 2);
  p.tokens = int32_of(q.size(0), "tokens");
  p.heads = int32_of(q.size(1), "heads");
  p.max_q = int32_of(max_q, "max_q");
  p.max_kv = kv_limit(p.cache, max_kv);
  p.softmax_scale = scale_of(softmax_scale, q.size(2));
  p.causal = causal;
  uint64_t bytes = 0;
  check_status(fa_paged_key_weights_workspace_size(&p, &bytes), "paged_key_weights");
  Tensor ws = workspace(bytes, q);
  check_status(fa_paged_key_weights(&p, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
               "paged_key_weights");
  wrote({&key_weights});
}

pybind11::tuple paged_evict(Tensor k_cache, Tensor v_cache, Tensor key_weights,
                            const Tensor& block_table, const Tensor& seq_lens, const Tensor& new_table,
                            int64_t keep, int64_t recent, std::optional<int64_t> max_kv) {
  check_no_derivative("paged_evict", {&k_cache, &v_cache, &key_weights});
  fa_paged_evict_params p{};
  p.cache = make_cache(k_cache, v_cache, block_table, std::nullopt, seq_lens);
  check_apart(Rows(k_cache), "k_cache", Rows(v_cache), "v_cache");
  const c10::OptionalDeviceGuard guard(k_cache.device());
  p.key_weights = key_weight_ptr(key_weights, k_cache, p.w_stride);
  p.new_table = index_ptr(new_table, "new_table", 2, k_cache);
  TORCH_CHECK(new_table.size(0) == block_table.size(0),
              "new_table must have as many rows as block_table");
  p.new_table_stride = new_table.stride(0);
  p.new_pages = int32_of(new_table.size(1), "new_table's width");
  p.keep = int32_of(keep, "keep");
  p.recent = int32_of(recent, "recent");
  p.max_kv = kv_limit(p.cache, max_kv);
  // Refused before anything is allocated by sizes that are not checked yet.
  int32_t none = 0;
  p.new_lens = p.kept = &none;
  check_status(fa_paged_evict_validate(&p), "paged_evict");
  Tensor new_lens = new_tensor({block_table.size(0)}, torch::kInt32, k_cache);
  Tensor kept = new_tensor({block_table.size(0), k_cache.size(1), keep}, torch::kInt32, k_cache);
  if (block_table.size(0) > 0) {
    p.new_lens = new_lens.data_ptr<int32_t>();
    p.kept = kept.data_ptr<int32_t>();
  }
  check_status(fa_paged_evict(&p, stream_of(k_cache)), "paged_evict");
  wrote({&k_cache, &v_cache, &key_weights});
  return pybind11::make_tuple(new_lens, kept);
}

// The norm's weights and tables, the same for every entry point.
struct NormTables {
  int32_t rot, rows, fp32;
  NormTables(const Tensor& ref, const Tensor& qw, const Tensor& kw, const Tensor& cos, const Tensor& sin) {
    const int64_t d = ref.size(ref.dim() - 1);
    for (const Tensor* w : {&qw, &kw}) {
      TORCH_CHECK(w->is_cuda() && w->device() == ref.device(),
                  "norm weights must be CUDA tensors on the same device as the others");
      TORCH_CHECK(w->dim() == 1 && w->size(0) == d && w->is_contiguous(),
                  "norm weights must be contiguous with shape [head_dim]");
      TORCH_CHECK(w->dtype() == torch::kFloat32 || w->dtype() == ref.dtype(),
                  "norm weights must be float32 or have q's dtype");
    }
    TORCH_CHECK(qw.dtype() == kw.dtype(), "q_weight and k_weight must have the same dtype");
    for (const Tensor* t : {&cos, &sin}) {
      TORCH_CHECK(t->is_cuda() && t->device() == ref.device(),
                  "cos and sin must be CUDA tensors on the same device as the others");
      TORCH_CHECK(t->dtype() == torch::kFloat32 && t->dim() == 2 && t->is_contiguous(),
                  "cos and sin must be contiguous float32 with shape [rows, rotated dims / 2]");
    }
    TORCH_CHECK(cos.sizes() == sin.sizes(), "cos and sin must have the same shape");
    rot = int32_of(2 * cos.size(1), "the rotated dims");
    rows = int32_of(cos.size(0), "the tables' rows");
    fp32 = qw.dtype() == torch::kFloat32;
  }
};

// Axes of the pairs of rotated dims, a byte each; none: one position a token.
using Axes = std::optional<std::string>;

// Their number is that of the positions' first dimension.
fa_rotary_axes rotary_axes(const std::string& axes, int32_t rot, const Tensor& positions) {
  TORCH_CHECK((int64_t)axes.size() == rot / 2 && axes.size() <= 64,
              "axes must have one entry per pair of rotated dims");
  fa_rotary_axes a{};
  std::memcpy(a.axis, axes.data(), axes.size());
  a.axes = int32_of(positions.size(0), "the number of axes");
  a.axis_stride = positions.size(0) > 1 ? positions.stride(0) : 0;
  return a;
}

// With axes, a is filled in.
fa_qk_norm_params norm_params(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw,
                              const Tensor& cos, const Tensor& sin, const std::optional<Tensor>& positions,
                              double eps, bool interleaved, const Axes& axes, fa_rotary_axes& a) {
  check_half(q, "q", 4, "[B, H, N, D]");
  check_half(k, "k", 4, "[B, H, N, D]");
  check_like(k, "k", q);
  TORCH_CHECK(q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3),
              "q and k must have the same batch, length and head_dim");
  const NormTables t(q, qw, kw, cos, sin);
  fa_qk_norm_params p{};
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  set_strides(p.q_stride, q, 3);
  set_strides(p.k_stride, k, 3);
  p.q_weight = qw.data_ptr();
  p.k_weight = kw.data_ptr();
  p.cos = cos.data_ptr<float>();
  p.sin = sin.data_ptr<float>();
  if (axes) {
    TORCH_CHECK(positions, "axes need positions");
    const int64_t dims = positions->dim();
    p.positions = index_ptr(*positions, "positions", dims == 3 ? 3 : 2, q);
    TORCH_CHECK(positions->size(-1) == q.size(2) && (dims == 2 || positions->size(1) == q.size(0)),
                "with axes, positions must have shape [axes, N] or [axes, B, N]");
    p.pos_stride = dims == 3 && positions->size(1) > 1 ? positions->stride(1) : 0;
    a = rotary_axes(*axes, t.rot, *positions);
  } else if (positions) {
    p.positions = index_ptr(*positions, "positions", positions->dim() == 2 ? 2 : 1, q);
    TORCH_CHECK(positions->size(-1) == q.size(2) &&
                    (positions->dim() == 1 || positions->size(0) == q.size(0)),
                "positions must have shape [N] or [B, N]");
    p.pos_stride = positions->dim() == 2 && positions->size(0) > 1 ? positions->stride(0) : 0;
  }
  p.batch = int32_of(q.size(0), "batch");
  p.heads = int32_of(q.size(1), "heads");
  p.kv_heads = int32_of(k.size(1), "kv_heads");
  p.seq_len = int32_of(q.size(2), "seq_len");
  p.head_dim = int32_of(q.size(3), "head_dim");
  p.rot = t.rot;
  p.table_rows = t.rows;
  p.interleaved = interleaved;
  p.dtype = q.dtype() == torch::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_F16;
  p.weight_fp32 = t.fp32;
  p.eps = static_cast<float>(eps);
  return p;
}

using Pair = std::pair<Tensor, Tensor>;

Pair norm_forward(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& cos,
                  const Tensor& sin, const std::optional<Tensor>& positions, double eps,
                  bool interleaved, const Axes& axes) {
  fa_rotary_axes a{};
  fa_qk_norm_params p = norm_params(q, k, qw, kw, cos, sin, positions, eps, interleaved, axes, a);
  const c10::OptionalDeviceGuard guard(q.device());
  Tensor qo = new_like(q), ko = new_like(k);
  p.q_out = qo.data_ptr();
  p.k_out = ko.data_ptr();
  set_strides(p.q_out_stride, qo, 3);
  set_strides(p.k_out_stride, ko, 3);
  check_status(axes ? fa_qk_norm_rope_axes(&p, &a, stream_of(q)) : fa_qk_norm_rope(&p, stream_of(q)),
               "qk_norm_rope");
  return {qo, ko};
}

std::array<Tensor, 4> norm_backward(const Tensor& dq_out, const Tensor& dk_out, const Tensor& q,
                                    const Tensor& k, const Tensor& qw, const Tensor& kw,
                                    const Tensor& cos, const Tensor& sin,
                                    const std::optional<Tensor>& positions, double eps,
                                    bool interleaved, const Axes& axes) {
  fa_qk_norm_bwd_params p{};
  fa_rotary_axes a{};
  p.fwd = norm_params(q, k, qw, kw, cos, sin, positions, eps, interleaved, axes, a);
  for (const auto& [g, x, name] : {std::make_tuple(&dq_out, &q, "q's gradient"),
                                   std::make_tuple(&dk_out, &k, "k's gradient")}) {
    TORCH_CHECK(g->is_cuda() && g->sizes() == x->sizes(), name, " must have its tensor's shape");
    check_like(*g, name, q);
  }
  const c10::OptionalDeviceGuard guard(q.device());
  const Tensor gq = readable(dq_out), gk = readable(dk_out);
  Tensor dq = new_like(q), dk = new_like(k);
  Tensor dqw = new_tensor({q.size(3)}, torch::kFloat32, q), dkw = new_tensor({q.size(3)}, torch::kFloat32, q);
  p.fwd.q_out = gq.data_ptr();
  p.fwd.k_out = gk.data_ptr();
  set_strides(p.fwd.q_out_stride, gq, 3);
  set_strides(p.fwd.k_out_stride, gk, 3);
  p.dq = dq.data_ptr();
  p.dk = dk.data_ptr();
  set_strides(p.dq_stride, dq, 3);
  set_strides(p.dk_stride, dk, 3);
  p.dq_weight = dqw.data_ptr<float>();
  p.dk_weight = dkw.data_ptr<float>();
  uint64_t bytes = 0;
  check_status(fa_qk_norm_rope_bwd_workspace_size(&p, &bytes), "qk_norm_rope_backward");
  Tensor ws = workspace(bytes, q);
  check_status(axes ? fa_qk_norm_rope_bwd_axes(&p, &a, ws.data_ptr(), bytes, stream_of(q))
                    : fa_qk_norm_rope_bwd(&p, ws.data_ptr(), bytes, stream_of(q)),
               "qk_norm_rope_backward");
  if (qw.dtype() != torch::kFloat32) {
    dqw = dqw.to(qw.dtype());
    dkw = dkw.to(kw.dtype());
  }
  return {dq, dk, dqw, dkw};
}

// The norm in autograd, differentiable once.  (A node of its own here: one
// written in Python costs 60 us more per training step.)
struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q,
                                                const Tensor& k, const Tensor& qw, const Tensor& kw,
                                                const Tensor& cos, const Tensor& sin,
                                                const std::optional<Tensor>& positions, double eps,
                                                bool interleaved, const Axes& axes) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Pair y = norm_forward(q, k, qw, kw, cos, sin, positions, eps, interleaved, axes);
    ctx->save_for_backward({q, k, qw, kw, cos, sin, positions.value_or(Tensor())});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["axes"] = axes;
    return {y.first, y.second};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list g) {
    const auto v = ctx->get_saved_variables();
    std::optional<Tensor> positions;
    if (v[6].defined()) positions = v[6];
    std::array<Tensor, 4> d;
    {
      at::NoGradGuard no_grad;
      for (int i = 0; i < 2; ++i)
        if (!g[i].defined()) g[i] = torch::zeros_like(v[i]);
      d = norm_backward(g[0], g[1], v[0], v[1], v[2], v[3], v[4], v[5], positions,
                        ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool(),
                        ctx->saved_data["axes"].toOptional<std::string>());
    }
    torch::autograd::variable_list out = once({d.begin(), d.end()}, "qk_norm_rope");
    out.resize(10);
    return out;
  }
};

pybind11::tuple qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw,
                             const Tensor& cos, const Tensor& sin, std::optional<Tensor> positions,
                             double eps, bool interleaved, Axes axes) {
  check_no_tangent("qk_norm_rope", {&q, &k, &qw, &kw, &cos, &sin});
  if (at::GradMode::is_enabled()) {
    TORCH_CHECK(!cos.requires_grad() && !sin.requires_grad(),
                "cos and sin get no gradients: detach them");
    if (q.requires_grad() || k.requires_grad() || qw.requires_grad() || kw.requires_grad()) {
      check_capture("qk_norm_rope", "qk_norm_rope_backward", {&q, &k, &qw, &kw});
      const auto y = QkNormRope::apply(q, k, qw, kw, cos, sin, positions, eps, interleaved, axes);
      return pybind11::make_tuple(y[0], y[1]);
    }
  }
  const Pair y = norm_forward(q, k, qw, kw, cos, sin, positions, eps, interleaved, axes);
  return pybind11::make_tuple(y.first, y.second);
}

pybind11::tuple qk_norm_rope_backward(const Tensor& dq_out, const Tensor& dk_out, const Tensor& q,
                                      const Tensor& k, const Tensor& qw, const Tensor& kw,
                                      const Tensor& cos, const Tensor& sin,
                                      std::optional<Tensor> positions, double eps, bool interleaved,
                                      Axes axes) {
  check_no_tangent("qk_norm_rope_backward", {&dq_out, &dk_out, &q, &k, &qw, &kw, &cos, &sin});
  at::NoGradGuard no_grad;
  const auto d = norm_backward(dq_out, dk_out, q, k, qw, kw, cos, sin, positions, eps, interleaved, axes);
  return pybind11::make_tuple(d[0], d[1], d[2], d[3]);
}

Tensor paged_store(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& qw, const Tensor& kw,
                   const Tensor& cos, const Tensor& sin, const Tensor& positions, Tensor k_cache,
                   Tensor v_cache, const Tensor& block_table, const Tensor& cu_seqlens,
                   const Tensor& seq_lens, std::optional<Tensor> out, double eps, bool interleaved,
                   Axes axes) {
  check_no_derivative("paged_store", {&q, &k, &v, &qw, &kw, &cos, &sin, &k_cache, &v_cache});
  if (out) check_no_derivative("paged_store", {&*out});
  fa_paged_store_params p{};
  p.cache = make_cache(k_cache, v_cache, block_table, cu_seqlens, seq_lens);
  check_packed(q, "q", k_cache);
  check_packed(k, "k", k_cache, q.size(0), k_cache.size(1));
  check_packed(v, "v", k_cache, q.size(0), k_cache.size(1));
  const Rows pools[2] = {Rows(k_cache), Rows(v_cache)};
  const Rows rows[3] = {Rows(q), Rows(k), Rows(v)};
  const char* const pool_names[2] = {"k_cache", "v_cache"};
  const char* const names[3] = {"q, unless it is q", "k", "v"};
  check_apart(pools[0], "k_cache", pools[1], "v_cache");
  for (int i = 0; i < 2; ++i)
    for (int j = 0; j < 3; ++j) check_apart(pools[i], pool_names[i], rows[j], j == 0 ? "q" : names[j]);
  const c10::OptionalDeviceGuard guard(q.device());
  if (out) {
    check_packed(*out, "out", k_cache, q.size(0), q.size(1));
    const Rows result(*out);
    for (int j = same_rows(*out, q) ? 1 : 0; j < 3; ++j) check_apart(result, "out", rows[j], names[j]);
    for (int i = 0; i < 2; ++i) check_apart(result, "out", pools[i], pool_names[i]);
  }
  Tensor o = out ? *out : new_tensor(q.sizes(), q.scalar_type(), q);
  const NormTables t(q, qw, kw, cos, sin);
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.q_out = o.data_ptr();
  set_strides(p.q_stride, q, 2);
  set_strides(p.k_stride, k, 2);
  set_strides(p.v_stride, v, 2);
  set_strides(p.q_out_stride, o, 2);
  p.q_weight = qw.data_ptr();
  p.k_weight = kw.data_ptr();
  p.cos = cos.data_ptr<float>();
  p.sin = sin.data_ptr<float>();
  p.positions = index_ptr(positions, "positions", axes ? 2 : 1, q);
  TORCH_CHECK(positions.size(-1) == q.size(0), axes ? "with axes, positions must have shape [axes, tokens]"
                                                    : "positions must have one entry per token");
  p.tokens = int32_of(q.size(0), "tokens");
  p.heads = int32_of(q.size(1), "heads");
  p.rot = t.rot;
  p.table_rows = t.rows;
  p.interleaved = interleaved;
  p.weight_fp32 = t.fp32;
  p.eps = static_cast<float>(eps);
  if (axes) {
    const fa_rotary_axes a = rotary_axes(*axes, t.rot, positions);
    check_status(fa_paged_store_axes(&p, &a, stream_of(q)), "paged_store");
  } else {
    check_status(fa_paged_store(&p, stream_of(q)), "paged_store");
  }
  wrote({&k_cache, &v_cache});
  if (out) wrote({&o});
  return o;
}

}  // namespace

void bind_cache(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("paged_forward", &paged_forward, py::arg("q"), py::arg("k_cache"), py::arg("v_cache"),
        py::arg("block_table"), py::arg("cu_seqlens"), py::arg("seq_lens"), py::arg("out"),
        py::arg("max_q"), py::arg("max_kv"), py::arg("causal"), py::arg("softmax_scale"),
        py::arg("return_lse"), py::arg("softcap") = std::optional<double>{},
        py::arg("window") = std::optional<int64_t>{}, py::arg("slopes") = std::optional<Tensor>{});
  m.def("paged_key_weights", &paged_key_weights, py::arg("q"), py::arg("lse"), py::arg("k_cache"),
        py::arg("block_table"), py::arg("cu_seqlens"), py::arg("seq_lens"), py::arg("key_weights"),
        py::arg("max_q"), py::arg("max_kv"), py::arg("causal"), py::arg("softmax_scale"));
  m.def("paged_evict", &paged_evict, py::arg("k_cache"), py::arg("v_cache"), py::arg("key_weights"),
        py::arg("block_table"), py::arg("seq_lens"), py::arg("new_table"), py::arg("keep"),
        py::arg("recent"), py::arg("max_kv"));
  m.def("qk_norm_rope", &qk_norm_rope, py::arg("q"), py::arg("k"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("cos"), py::arg("sin"), py::arg("positions"), py::arg("eps"),
        py::arg("interleaved"), py::arg("axes") = Axes{});
  m.def("qk_norm_rope_backward", &qk_norm_rope_backward, py::arg("dq_out"), py::arg("dk_out"),
        py::arg("q"), py::arg("k"), py::arg("q_weight"), py::arg("k_weight"), py::arg("cos"),
        py::arg("sin"), py::arg("positions"), py::arg("eps"), py::arg("interleaved"),
        py::arg("axes") = Axes{});
  m.def("paged_store", &paged_store, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("cos"), py::arg("sin"), py::arg("positions"), py::arg("k_cache"),
        py::arg("v_cache"), py::arg("block_table"), py::arg("cu_seqlens"), py::arg("seq_lens"),
        py::arg("out"), py::arg("eps"), py::arg("interleaved"), py::arg("axes") = Axes{});
}
