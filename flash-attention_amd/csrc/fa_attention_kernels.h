// Internal interface between the C ABI of attention with gradients
// (fa_attention_api.cpp) and its HIP kernels.  Strides are in bytes here.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_fwd_kernel.h"
#include "fa_score.h"

namespace fa {

// Rows of whole tensors [batch, heads, rows, head_dim].
struct Rows3 {
  char* p;
  int64_t sb, sh, st;  // batch, head, row
};

// Order of a grid: `places` workgroups of each unit (batch entry and kv head), the
// longest of a causal mask first.
struct GridOrder {
  int32_t units, places, per_xcd, unit_group, xcds, xcd_cus, turn;
  FastDiv by_group_places, by_unit_group, by_units;
};

struct AttnArgs {
  Rows3 q, k, v, o;
  float* lse;               // [batch, heads, n] contiguous
  char* o_low;              // [batch, heads, n, head_dim] contiguous: what o's rounding left out; NULL: none
  const int32_t* ranges;    // pairs (first key, end) of each row; NULL: all keys
  int64_t range_sb;         // elements
  int32_t batch, heads, kv_heads, group;
  int32_t n, m;             // rows, keys
  int32_t causal;
  float scale, scale_log2;
  ScoreArgs score;
  int32_t tiles;            // row tiles of a head (kAttnRows)
  FastDiv by_group, by_kvh;
  GridOrder rows;           // forward and dq: tiles * group places
  int32_t row_teams, key_teams;  // teams of four waves of their workgroups, of dk and dv's
  // backward
  Rows3 go, gq, gk, gv;     // gradients of o, q, k, v
  const float* glse;        // of lse; may be NULL
  float* records;           // [batch, heads, spans][record_floats], see fa_attention_bwd.hip
  int32_t* bounds;          // [batch, spans][4]: limits of a span's rows
  int32_t spans;            // spans of kSpan rows
  int32_t key_tiles, splits;
  FastDiv by_splits;
  GridOrder cols;           // dk, dv: key_tiles * splits places
  int32_t* key_order;       // [batch, key_tiles]: the tiles of keys, the longest first; NULL: as they lie
  float* parts;             // [splits][batch, kv_heads, m][2][D] gradients of k and v; NULL: one split
};

constexpr int kAttnRows = 128;  // rows of a forward or dq workgroup
constexpr int kAttnKeys = 128;  // keys of a dk, dv workgroup
constexpr int kSpan = 32;       // rows that it stages at a time
constexpr int kMaxOrdered = 1024;  // tiles of keys that key_order ranks

// Teams of a workgroup of few: as many as fill a CU.
constexpr int key_teams(int head_dim) { return head_dim == 128 ? 2 : 3; }

// Of the record of a span: four of each row, and with fp16 one more, one of all and filling.
constexpr int record_floats(bool bf16) { return bf16 ? 4 * kSpan : 5 * kSpan + 4; }

struct AttnBwdPlan {
  int32_t teams, splits;
  uint64_t records, bounds, parts, order;  // bytes, each a multiple of 16
};
GridOrder grid_order(int units, int places, int compute_units, int per_cu);
int64_t grid_size(const GridOrder& o);
AttnBwdPlan plan_attn_bwd(const AttnArgs& a, int head_dim, bool bf16, int compute_units);

hipError_t launch_attn_fwd(const AttnArgs& args, int head_dim, bool bf16, hipStream_t stream);
hipError_t launch_attn_bwd(const AttnArgs& args, int head_dim, bool bf16, hipStream_t stream);

}  // namespace fa
