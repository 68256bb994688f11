/*
 * fa_mi355x_attention.h — C ABI of attention with gradients, whose scores may be
 * capped, biased by distance and masked; of the same scores over the paged cache;
 * and of the rotation by positions of several axes.  Same library, status codes,
 * error string, ownership, streams and threading as fa_mi355x.h.  None of these
 * has a counterpart in the reference.
 *
 *   fa_attn_fwd            attention of whole tensors
 *   fa_attn_bwd            its gradients
 *   fa_paged_fwd_scored    fa_paged_fwd with these scores
 *   fa_qk_norm_rope_axes   fa_qk_norm_rope with several positions a token
 *   fa_qk_norm_rope_bwd_axes, fa_paged_store_axes   likewise
 *
 * Scores.  Row i stands at p = i + keys - seq_len among the keys (the last row at
 * the last key); of the paged cache at its token's key.
 *   z = softmax_scale q_i.k_j
 *   c = softcap tanh(z / softcap)              (softcap 0: c = z)
 *   x = c - slopes[head] |p - j|               (slopes NULL: x = c)
 * Row i sees the keys j of its range that, with causal, are j <= p and, with a
 * window, are at |p - j| < window.  Distances are fp32: whole numbers to 2^24, beyond
 * that to 24 bits.
 */
#ifndef FA_MI355X_ATTENTION_H
#define FA_MI355X_ATTENTION_H

#include "fa_mi355x.h"
#include "fa_mi355x_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

/* All zero: plain scores. */
typedef struct {
  float softcap;       /* 0: none; else from 0.001 to 1000 (its error is about 1e-7 of it) */
  int32_t window;      /* 0: none */
  const float* slopes; /* [heads], device memory; slopes over softmax_scale are finite; NULL: none */
} fa_score_params;

/* o_i = sum_j exp(x_ij - lse_i) v_j,  lse_i = ln sum_j exp(x_ij), over the keys
 * that row i sees.  Query head h reads kv head h / (heads / kv_heads).  A row that
 * sees no key has o = 0 and lse = -inf.  A key that a row does not see contributes
 * nothing to it, whatever its K and V hold (infinities and NaN included). */
typedef struct {
  const void* q;          /* [batch, heads, seq_len, head_dim], unit stride along head_dim */
  const void* k;          /* [batch, kv_heads, keys, head_dim] */
  const void* v;
  void* o;                /* like q */
  float* lse;             /* [batch, heads, seq_len] contiguous, natural log; may be NULL in fa_attn_fwd */
  void* o_low;            /* [batch, heads, seq_len, head_dim] contiguous, 16-byte aligned: what the rounding
                             of o left out, rounded likewise; fa_attn_bwd takes delta from both.  NULL: none,
                             at the price of delta's exactness where few keys have most of the weight */
  int64_t q_stride[3];    /* batch, head, row; multiples of 8 elements */
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t o_stride[3];
  const int32_t* ranges;  /* [batch][seq_len][2], 8-byte aligned: first key and end of the keys that a
                             row sees, any values (limited to 0 .. keys); NULL: all keys */
  int64_t range_stride;   /* elements from one batch entry to the next; 0: shared; even */
  int32_t batch, heads, kv_heads, seq_len, keys, head_dim; /* head_dim 64 or 128; lengths to 2^28 */
  int32_t dtype;          /* fa_dtype of q, k, v, o and their gradients */
  int32_t causal;
  float softmax_scale;    /* a normal positive number, at most FLT_MAX / 2 */
  fa_score_params score;
} fa_attn_params;

/* Gradients of fa_attn_fwd:  delta_i = go_i.(o_i + o_low_i) - glse_i,
 *   dx_ij = P_ij (go_i.v_j - delta_i),  P = exp(x - lse),
 *   dz = dx (1 - (c / softcap)^2),  gv_j = sum_i P go_i,
 *   gk_j = softmax_scale sum_i dz q_i,  gq_i = softmax_scale sum_j dz k_j,
 * those of k and v summed over the query heads that read them.  Sums run in a fixed
 * order (no atomics).  fwd: as given to fa_attn_fwd, o, lse and o_low as it wrote
 * them (read only).  Rows and keys that do not see each other contribute nothing to each
 * other, whatever they hold.  A result that takes in an infinity or a NaN of a row or
 * key that it sees is one of them; so may be the others of that row or key. */
typedef struct {
  fa_attn_params fwd;
  const void* go;         /* like q */
  const float* glse;      /* gradient of lse, contiguous; NULL: 0 */
  void* gq;
  void* gk;
  void* gv;
  int64_t go_stride[3];
  int64_t gq_stride[3];
  int64_t gk_stride[3];
  int64_t gv_stride[3];
} fa_attn_bwd_params;

/* The axis of each pair of rotated dims: pair i turns by the angles of row
 * positions[axis[i]] of the tables (at its own column i).  With axes, positions
 * holds the axes' positions one after the other, axis_stride elements apart. */
typedef struct {
  uint8_t axis[64];       /* of the first rot / 2 pairs; below axes */
  int32_t axes;           /* 1 to 4 */
  int64_t axis_stride;
} fa_rotary_axes;

/* Host-only argument checks; they touch no GPU. */
fa_status fa_attn_fwd_validate(const fa_attn_params* p);
fa_status fa_attn_bwd_validate(const fa_attn_bwd_params* p);
fa_status fa_paged_fwd_scored_validate(const fa_paged_fwd_params* p, const fa_score_params* score);
fa_status fa_qk_norm_rope_axes_validate(const fa_qk_norm_params* p, const fa_rotary_axes* axes);
fa_status fa_qk_norm_rope_bwd_axes_validate(const fa_qk_norm_bwd_params* p, const fa_rotary_axes* axes);
fa_status fa_paged_store_axes_validate(const fa_paged_store_params* p, const fa_rotary_axes* axes);

/* Workspace bytes on the calling thread's current device, by the arguments alone. */
fa_status fa_attn_bwd_workspace_size(const fa_attn_bwd_params* p, uint64_t* bytes);
fa_status fa_paged_fwd_scored_workspace_size(const fa_paged_fwd_params* p, const fa_score_params* score,
                                             uint64_t* bytes);

/* Validate, then launch asynchronously on `stream`; as the calls of
 * fa_mi355x_cache.h each can be captured into a graph.  fa_qk_norm_rope_bwd_axes
 * takes the workspace of fa_qk_norm_rope_bwd_workspace_size. */
fa_status fa_attn_fwd(const fa_attn_params* p, void* stream);
fa_status fa_attn_bwd(const fa_attn_bwd_params* p, void* workspace, uint64_t workspace_bytes, void* stream);
fa_status fa_paged_fwd_scored(const fa_paged_fwd_params* p, const fa_score_params* score, void* workspace,
                              uint64_t workspace_bytes, void* stream);
fa_status fa_qk_norm_rope_axes(const fa_qk_norm_params* p, const fa_rotary_axes* axes, void* stream);
fa_status fa_qk_norm_rope_bwd_axes(const fa_qk_norm_bwd_params* p, const fa_rotary_axes* axes,
                                   void* workspace, uint64_t workspace_bytes, void* stream);
fa_status fa_paged_store_axes(const fa_paged_store_params* p, const fa_rotary_axes* axes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FA_MI355X_ATTENTION_H */
