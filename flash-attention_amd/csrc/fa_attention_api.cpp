// C ABI of attention with gradients (declared in include/fa_mi355x_attention.h):
// argument checks, launch plans and workspace layout.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "fa_attention_kernels.h"
#include "fa_checks.h"
#include "fa_host.h"
#include "fa_mi355x_attention.h"

namespace fa {

namespace {
constexpr int kXcds = 8;
}

GridOrder grid_order(int units, int places, int compute_units, int per_cu) {
  GridOrder o = {};
  o.units = units;
  o.places = places;
  o.xcd_cus = compute_units / kXcds;
  o.per_xcd = units % kXcds == 0 ? units / kXcds : 0;
  o.xcds = o.per_xcd == 0 && kXcds % units == 0 ? kXcds / units : 0;
  // The fewest units at once that give each CU its workgroups, of those that divide an
  // XCD's evenly; all of them if none does.
  o.unit_group = std::max(o.per_xcd, 1);
  for (int g = 1; g < o.per_xcd && g <= per_cu * o.xcd_cus; ++g)
    if (o.per_xcd % g == 0 && (int64_t)g * places >= per_cu * o.xcd_cus) {
      o.unit_group = g;
      break;
    }
  o.turn = per_cu > 1 && (int64_t)units * places > (int64_t)kXcds * o.xcd_cus;
  o.by_group_places = make_fast_div((uint32_t)(o.unit_group * places));
  o.by_unit_group = make_fast_div((uint32_t)o.unit_group);
  o.by_units = make_fast_div((uint32_t)units);
  return o;
}

int64_t grid_size(const GridOrder& o) {
  if (o.xcds > 0) return (int64_t)kXcds * ((o.places + o.xcds - 1) / o.xcds);
  return (int64_t)o.units * o.places;
}

AttnBwdPlan plan_attn_bwd(const AttnArgs& a, int head_dim, bool bf16, int compute_units) {
  AttnBwdPlan p = {};
  const int64_t bh = (int64_t)a.batch * a.heads;
  // (1 KiB from a record's start is staged, at most 512 bytes behind it)
  p.records = (uint64_t)bh * a.spans * record_floats(bf16) * 4 + 512;
  p.bounds = (uint64_t)a.batch * a.spans * 16;
  const int64_t tiles = (int64_t)a.batch * a.kv_heads * a.key_tiles;
  // Teams where a CU has one workgroup at most; or two of different lengths, which a
  // team more evens out (D = 128, us with one and with teams: 16 causal heads of 4096 rows 206
  // and 186, 32 heads without a mask of 2048 rows 142 and 172); or any number of lengths
  // that only the device knows, the longest first (documents of 21 to 3960 rows in 16384, 32 heads
  // on 8: 1190 and 970; of 2048 each: 650 and 775).
  const bool ranked = a.ranges != nullptr && tiles > 2 * compute_units && a.key_tiles <= kMaxOrdered;
  const bool uneven = a.ranges != nullptr || (a.causal && a.score.window == 0);
  p.order = ranked ? ((uint64_t)a.batch * a.key_tiles * 4 + 15) / 16 * 16 : 0;
  p.teams = ranked || tiles <= (uneven ? 2 : 1) * compute_units ? key_teams(head_dim) : 1;
  int64_t splits = ((int64_t)compute_units + tiles - 1) / tiles;
  splits = std::max<int64_t>(1, std::min<int64_t>(splits, a.spans / (4 * p.teams)));
  p.splits = (int32_t)splits;
  p.parts = splits > 1 ? (uint64_t)splits * a.batch * a.kv_heads * a.m * 2 * head_dim * 4 : 0;
  return p;
}

namespace {

constexpr int32_t kMaxLength = 1 << 28;

fa_status check_attn(const fa_attn_params& p, bool backward) {
  FA_TRY(check_dtype(p.dtype));
  FA_TRY(check_head_dim(p.head_dim));
  if (p.batch < 1 || p.heads < 1 || p.kv_heads < 1 || p.seq_len < 1 || p.keys < 1)
    return fail(FA_ERR_SHAPE, "batch=%d heads=%d kv_heads=%d seq_len=%d keys=%d must all be >= 1", (int)p.batch,
                (int)p.heads, (int)p.kv_heads, (int)p.seq_len, (int)p.keys);
  if (p.heads % p.kv_heads != 0)
    return fail(FA_ERR_SHAPE, "heads=%d must be a multiple of kv_heads=%d", (int)p.heads, (int)p.kv_heads);
  if (p.seq_len > kMaxLength || p.keys > kMaxLength)
    return fail(FA_ERR_UNSUPPORTED, "seq_len=%d and keys=%d must be at most 2^28", (int)p.seq_len, (int)p.keys);
  // (workgroups of 64 rows, and of 128 keys in parts of 4 spans of rows)
  const int64_t rows = ((int64_t)p.seq_len + 63) / 64, keys = ((int64_t)p.keys + kAttnKeys - 1) / kAttnKeys;
  if ((__int128)p.batch * p.heads * (rows + keys) > (int64_t(1) << 30))
    return fail(FA_ERR_UNSUPPORTED, "batch*heads and the lengths exceed the kernel's range");
  const int64_t qs[3] = {p.batch, p.heads, p.seq_len};
  FA_TRY(check_rows("q", p.q, p.q_stride, 3));
  FA_TRY(check_rows("k", p.k, p.k_stride, 3));
  FA_TRY(check_rows("v", p.v, p.v_stride, 3));
  FA_TRY(check_rows("o", p.o, p.o_stride, 3));
  if (!backward) FA_TRY(check_written("o", p.o_stride, qs, 3, p.head_dim));
  for (const int64_t* st : {p.q_stride, p.k_stride, p.v_stride, p.o_stride})
    if (st[2] > kMaxKeyStride)
      return fail(FA_ERR_UNSUPPORTED, "row stride %lld exceeds %lld elements", (long long)st[2],
                  (long long)kMaxKeyStride);
  if (backward && p.lse == nullptr) return fail(FA_ERR_NULL, "lse is NULL");
  if (!aligned(p.lse, 4)) return fail(FA_ERR_STRIDE, "lse pointer is not 4-byte aligned");
  if (!aligned(p.o_low, 16)) return fail(FA_ERR_STRIDE, "o_low pointer is not 16-byte aligned");
  if (!aligned(p.ranges, 8)) return fail(FA_ERR_STRIDE, "ranges pointer is not 8-byte aligned");
  if (p.range_stride < 0 || p.range_stride % 2 != 0)
    return fail(FA_ERR_STRIDE, "range_stride %lld is negative or odd", (long long)p.range_stride);
  FA_TRY(check_flag("causal", p.causal));
  FA_TRY(check_scale(p.softmax_scale));
  return check_score(p.score, p.softmax_scale);
}

Rows3 rows3(const void* p, const int64_t st[3]) {
  return Rows3{static_cast<char*>(const_cast<void*>(p)), 2 * st[0], 2 * st[1], 2 * st[2]};
}

AttnArgs attn_args(const fa_attn_params& p, int compute_units) {
  AttnArgs a = {};
  a.q = rows3(p.q, p.q_stride);
  a.k = rows3(p.k, p.k_stride);
  a.v = rows3(p.v, p.v_stride);
  a.o = rows3(p.o, p.o_stride);
  a.lse = p.lse;
  a.o_low = static_cast<char*>(p.o_low);
  a.ranges = p.ranges;
  a.range_sb = p.range_stride;
  a.batch = p.batch;
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.group = p.heads / p.kv_heads;
  a.n = p.seq_len;
  a.m = p.keys;
  a.causal = p.causal;
  a.scale = p.softmax_scale;
  a.scale_log2 = (float)(p.softmax_scale * kLog2e);
  a.score = score_args(p.score, p.softmax_scale);
  a.tiles = (p.seq_len + kAttnRows - 1) / kAttnRows;
  a.by_group = make_fast_div((uint32_t)a.group);
  a.by_kvh = make_fast_div((uint32_t)a.kv_heads);
  const int64_t row_tiles = (int64_t)a.batch * a.heads * a.tiles;
  // Two teams where a CU has one workgroup at most: 16 heads of 2048 rows, D = 128, us with
  // one and two: forward 51 and 43, dq 70 and 60; with two workgroups a CU (2 x 2000 rows in
  // documents) 66 and 68, 72 and 76.
  a.row_teams = row_tiles <= compute_units ? 2 : 1;
  a.rows = grid_order(a.batch * a.kv_heads, a.tiles * a.group, compute_units, a.row_teams == 1 ? 2 : 1);
  a.spans = (p.seq_len + kSpan - 1) / kSpan;
  a.key_tiles = (p.keys + kAttnKeys - 1) / kAttnKeys;
  return a;
}

fa_status bwd_plan(const fa_attn_bwd_params& p, AttnArgs* args, AttnBwdPlan* plan) {
  int cus = 0;
  FA_TRY(current_compute_units(&cus));
  *args = attn_args(p.fwd, cus);
  *plan = plan_attn_bwd(*args, p.fwd.head_dim, p.fwd.dtype == FA_DTYPE_BF16, cus);
  args->splits = plan->splits;
  args->cols = grid_order(args->batch * args->kv_heads, args->key_tiles * plan->splits, cus, plan->teams == 1 ? 2 : 1);
  args->key_teams = plan->teams;
  return FA_OK;
}

uint64_t total(const AttnBwdPlan& p) { return p.records + p.bounds + p.parts + p.order; }

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

fa_status fa_attn_fwd_validate(const fa_attn_params* p) {
  clear_error();
  if (p == nullptr) return fail(FA_ERR_NULL, "params is NULL");
  return check_attn(*p, false);
}

fa_status fa_attn_bwd_validate(const fa_attn_bwd_params* p) {
  clear_error();
  if (p == nullptr) return fail(FA_ERR_NULL, "params is NULL");
  const fa_attn_params& f = p->fwd;
  FA_TRY(check_attn(f, true));
  const int64_t qs[3] = {f.batch, f.heads, f.seq_len}, ks[3] = {f.batch, f.kv_heads, f.keys};
  FA_TRY(check_rows("o's gradient", p->go, p->go_stride, 3));
  if (p->go_stride[2] > kMaxKeyStride)
    return fail(FA_ERR_UNSUPPORTED, "row stride %lld of o's gradient exceeds %lld elements",
                (long long)p->go_stride[2], (long long)kMaxKeyStride);
  FA_TRY(check_rows("gq", p->gq, p->gq_stride, 3));
  FA_TRY(check_rows("gk", p->gk, p->gk_stride, 3));
  FA_TRY(check_rows("gv", p->gv, p->gv_stride, 3));
  FA_TRY(check_written("gq", p->gq_stride, qs, 3, f.head_dim));
  FA_TRY(check_written("gk", p->gk_stride, ks, 3, f.head_dim));
  FA_TRY(check_written("gv", p->gv_stride, ks, 3, f.head_dim));
  if (!aligned(p->glse, 4)) return fail(FA_ERR_STRIDE, "lse's gradient is not 4-byte aligned");
  return FA_OK;
}

fa_status fa_attn_fwd(const fa_attn_params* p, void* stream) {
  FA_TRY(fa_attn_fwd_validate(p));
  int cus = 0;
  FA_TRY(current_compute_units(&cus));
  return launched(launch_attn_fwd(attn_args(*p, cus), p->head_dim, p->dtype == FA_DTYPE_BF16,
                                  static_cast<hipStream_t>(stream)));
}

fa_status fa_attn_bwd_workspace_size(const fa_attn_bwd_params* p, uint64_t* bytes) {
  if (bytes == nullptr) return fail(FA_ERR_NULL, "bytes is NULL");
  *bytes = 0;
  FA_TRY(fa_attn_bwd_validate(p));
  AttnArgs a;
  AttnBwdPlan plan;
  FA_TRY(bwd_plan(*p, &a, &plan));
  *bytes = total(plan);
  return FA_OK;
}

fa_status fa_attn_bwd(const fa_attn_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream) {
  FA_TRY(fa_attn_bwd_validate(p));
  AttnArgs a;
  AttnBwdPlan plan;
  FA_TRY(bwd_plan(*p, &a, &plan));
  FA_TRY(check_workspace(workspace, workspace_bytes, total(plan)));
  a.go = rows3(p->go, p->go_stride);
  a.gq = rows3(p->gq, p->gq_stride);
  a.gk = rows3(p->gk, p->gk_stride);
  a.gv = rows3(p->gv, p->gv_stride);
  a.glse = p->glse;
  char* ws = static_cast<char*>(workspace);
  a.records = reinterpret_cast<float*>(ws);
  a.bounds = reinterpret_cast<int32_t*>(ws + plan.records);
  ws += plan.records + plan.bounds;
  a.parts = plan.parts > 0 ? reinterpret_cast<float*>(ws) : nullptr;
  a.key_order = plan.order > 0 ? reinterpret_cast<int32_t*>(ws + plan.parts) : nullptr;
  a.by_splits = make_fast_div((uint32_t)a.splits);
  return launched(launch_attn_bwd(a, p->fwd.head_dim, p->fwd.dtype == FA_DTYPE_BF16,
                                  static_cast<hipStream_t>(stream)));
}

}  // extern "C"
