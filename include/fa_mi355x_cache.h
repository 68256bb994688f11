/*
 * fa_mi355x_cache.h — C ABI of the operators around a paged key/value cache,
 * and of the q/k norm with rotation that stands in front of attention.  Same
 * library, status codes, error string, ownership, streams and threading as
 * fa_mi355x.h.  None of these has a counterpart in the reference.
 *
 *   fa_qk_norm_rope      per-head RMS norm of q and k and the position rotation
 *   fa_qk_norm_rope_bwd  its gradients
 *   fa_paged_store       the same for new tokens, k and v written to the cache
 *   fa_paged_fwd         attention of the new tokens over the cache
 *   fa_paged_key_weights attention weight that each cached key has received
 *   fa_paged_evict       keeps the newest and the heaviest keys of each head
 *
 * The cache.  k and v are pools of pages: [num_pages, kv_heads, page_size,
 * head_dim] with unit stride along head_dim and free strides otherwise (a
 * [num_pages, page_size, kv_heads, head_dim] pool is a view).  Key j of
 * sequence b is row j % page_size of page block_table[b][j / page_size].
 * New tokens of all sequences are packed: rows cu_seqlens[b] up to
 * cu_seqlens[b + 1] of q, k, v, o, lse are sequence b's, oldest first, and
 * seq_lens[b] counts its keys in the cache, these new ones included: with n
 * new tokens of length L, token i is key L - n + i.
 *
 * The table, cu_seqlens and seq_lens are device memory, so that a captured
 * graph can be replayed with other lengths, and no kernel trusts them: a page
 * id outside [0, num_pages) is an absent page (its keys are masked, read as
 * weight 0 and never written), seq_lens is limited to [0, max_kv] and to the
 * table's max_pages pages, cu_seqlens to [0, tokens].  Rows of q that belong
 * to no sequence are not written to in o and lse.  cu_seqlens must not
 * descend: the rows and keys of sequences that do get unspecified values, and
 * nothing else is written.
 *
 * What a call writes shares no element with what it reads, nor k's pool with
 * v's where both are written, unless a field says that it may.
 */
#ifndef FA_MI355X_CACHE_H
#define FA_MI355X_CACHE_H

#include "fa_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A paged cache and the sequences in it.  Strides are in elements: [0] page,
 * [1] kv head, [2] key; multiples of 8, pointers 16-byte aligned. */
typedef struct {
  void* k;
  void* v; /* not read by fa_paged_key_weights, where it may be NULL */
  int64_t k_stride[3];
  int64_t v_stride[3];
  const int32_t* block_table; /* [batch][max_pages], row stride table_stride */
  int64_t table_stride;
  const int32_t* cu_seqlens;  /* [batch + 1]; not read by fa_paged_evict */
  const int32_t* seq_lens;    /* [batch] */
  int32_t batch;              /* >= 0 */
  int32_t num_pages;          /* >= 1 */
  int32_t page_size;          /* a power of two, 16 to 4096 */
  int32_t max_pages;          /* >= 1; max_pages * page_size <= 2^30 */
  int32_t kv_heads;
  int32_t head_dim;           /* 64 or 128 */
  int32_t dtype;              /* fa_dtype of the cache, q, k, v and o */
  int32_t reserved;           /* 0 */
} fa_paged_cache;

/* Attention of new tokens over the cache:
 *   o[t,h] = sum_j softmax_j(scale q[t,h].k_j) v_j over the keys j that token t
 *   sees: with causal those up to its own, else all of its sequence.
 * Query head h reads kv head h / (heads / kv_heads).  A row that sees no key
 * has o = 0 and lse = -inf.  A masked or absent key contributes nothing,
 * whatever its row holds (infinities and NaN included). */
typedef struct {
  fa_paged_cache cache;
  const void* q;        /* [tokens, heads, head_dim] */
  void* o;              /* the same shape */
  float* lse;           /* [tokens, heads] contiguous, natural log; may be NULL */
  int64_t q_stride[2];  /* token, head; multiples of 8 elements */
  int64_t o_stride[2];
  int32_t tokens;       /* >= 0 */
  int32_t heads;        /* a multiple of kv_heads */
  int32_t max_q;        /* most new tokens of one sequence; those past it are not computed */
  int32_t max_kv;       /* most keys of one sequence; seq_lens above it are taken as max_kv */
  float softmax_scale;  /* a normal positive number, at most FLT_MAX / 2 */
  int32_t causal;
} fa_paged_fwd_params;

/* Adds to key_weights the attention weight that each key receives from the new
 * tokens of its kv head's query heads:
 *   add[j] = sum_{t,h} exp(scale q[t,h].k_j - lse[t,h]) over the rows that see j.
 * A key that is itself one of the new tokens is seen for the first time: its
 * weight is set to the sum, so that the slot of a reused page needs no
 * clearing.  Rows whose lse is -inf add nothing.  Sums run in a fixed order
 * (no atomics); a page must belong to one sequence of the call only. */
typedef struct {
  fa_paged_cache cache;   /* v unused */
  const void* q;          /* [tokens, heads, head_dim] */
  const float* lse;       /* [tokens, heads] contiguous, as fa_paged_fwd writes it (not fa_paged_fwd_scored:
                             the weights are those of plain scores) */
  float* key_weights;     /* [num_pages, kv_heads, page_size], unit key stride */
  int64_t q_stride[2];    /* token, head */
  int64_t w_stride[2];    /* page, kv head */
  int32_t tokens;
  int32_t heads;
  int32_t max_q;
  int32_t max_kv;
  float softmax_scale;
  int32_t causal;
} fa_paged_weights_params;

/* Per sequence and kv head: keeps the `recent` last keys and, of the others,
 * the ones of largest key weight, `keep` keys in all (every key of a sequence
 * that has no more).  Equal weights: the lower index is kept; NaN counts as
 * the largest.  The kept keys, values and weights are copied in their order
 * to the pages of new_table, each listed once there and none among the pages
 * being read; the old pages are left as they are.  A sequence with an absent page among its keys'
 * or its new pages is not copied: its new length is 0 and its kept indices
 * are -1. */
typedef struct {
  fa_paged_cache cache;      /* cu_seqlens unused */
  float* key_weights;        /* as above */
  int64_t w_stride[2];       /* page, kv head */
  const int32_t* new_table;  /* [batch][new_pages], row stride new_table_stride */
  int64_t new_table_stride;
  int32_t* new_lens;         /* [batch]: min(length, keep); may be cache.seq_lens itself */
  int32_t* kept;             /* [batch, kv_heads, keep] contiguous: index of the key now at t, or -1 */
  int32_t new_pages;         /* new_pages * page_size >= min(keep, max_pages * page_size) */
  int32_t keep;              /* 1 to 2^30 */
  int32_t recent;            /* 0 to keep */
  int32_t max_kv;            /* as in fa_paged_fwd_params */
} fa_paged_evict_params;

/* y = R(pos) (x rstd w), rstd = (mean(x^2) + eps)^(-1/2), for each head's row x
 * of q and k.  R turns the pairs (i, i + rot/2), or with interleaved (2i,
 * 2i + 1), of the first rot dims by the angle whose cosine and sine are row
 * pos of the tables: (a, b) -> (a cos - b sin, b cos + a sin); the other dims
 * keep their value.  All in fp32, rounded once; the mean square overflows for
 * rows of values above about 1e18, which become 0.  A position outside the
 * tables gives rows of NaN. */
typedef struct {
  const void* q;         /* [batch, heads, seq_len, head_dim], unit stride along head_dim */
  const void* k;         /* [batch, kv_heads, seq_len, head_dim] */
  void* q_out;           /* same shapes; may be q and k themselves */
  void* k_out;
  int64_t q_stride[3];   /* batch, head, token; multiples of 8 elements */
  int64_t k_stride[3];
  int64_t q_out_stride[3];
  int64_t k_out_stride[3];
  const void* q_weight;  /* [head_dim] of weight_dtype */
  const void* k_weight;
  const float* cos;      /* [table_rows, rot / 2] contiguous */
  const float* sin;
  const int32_t* positions; /* [batch][seq_len], row stride pos_stride (0: shared); NULL: 0, 1, ... */
  int64_t pos_stride;
  int32_t batch, heads, kv_heads, seq_len, head_dim;
  int32_t rot;           /* rotated dims, a multiple of 16 up to head_dim */
  int32_t table_rows;
  int32_t interleaved;   /* 0 or 1 */
  int32_t dtype;         /* of q and k */
  int32_t weight_fp32;   /* 1: the weights are fp32; 0: they have q's dtype */
  float eps;             /* finite, >= 0 */
} fa_qk_norm_params;

/* Gradients of fa_qk_norm_rope: with g = R(pos)^T dy and xh = x rstd,
 *   dx = rstd (g w - xh mean(g w xh)),  dw = sum over rows of g xh.
 * fwd: as given to fa_qk_norm_rope, with q_out and k_out holding the incoming
 * gradients (read only).  dq and dk have q's and k's shapes; they may be q_out
 * and k_out themselves where their strides agree.  The weights' gradients are
 * fp32, summed in a fixed order.  Rows at positions outside the tables give NaN. */
typedef struct {
  fa_qk_norm_params fwd;
  void* dq;
  void* dk;
  int64_t dq_stride[3];
  int64_t dk_stride[3];
  float* dq_weight; /* [head_dim] */
  float* dk_weight;
} fa_qk_norm_bwd_params;

/* fa_qk_norm_rope of packed new tokens: q_out as there ([tokens, heads,
 * head_dim]), k's result and v go to the tokens' places in the cache.  The
 * pages that receive new tokens must belong to one sequence only.  Tokens past
 * a sequence's keys (more new tokens than keys: the first ones) or on absent
 * pages are not stored.  seq_lens is limited by the table alone: a length that
 * fa_paged_fwd cuts at a smaller max_kv has its tokens at other keys there. */
typedef struct {
  fa_paged_cache cache;
  const void* q;        /* [tokens, heads, head_dim] */
  const void* k;        /* [tokens, kv_heads, head_dim] */
  const void* v;
  void* q_out;          /* may be q itself */
  int64_t q_stride[2];  /* token, head */
  int64_t k_stride[2];
  int64_t v_stride[2];
  int64_t q_out_stride[2];
  const void* q_weight;
  const void* k_weight;
  const float* cos;
  const float* sin;
  const int32_t* positions; /* [tokens] */
  int32_t tokens, heads;
  int32_t rot, table_rows, interleaved, weight_fp32;
  float eps;
} fa_paged_store_params;

/* Host-only argument checks; they touch no GPU. */
fa_status fa_paged_fwd_validate(const fa_paged_fwd_params* p);
fa_status fa_paged_key_weights_validate(const fa_paged_weights_params* p);
fa_status fa_paged_evict_validate(const fa_paged_evict_params* p);
fa_status fa_qk_norm_rope_validate(const fa_qk_norm_params* p);
fa_status fa_qk_norm_rope_bwd_validate(const fa_qk_norm_bwd_params* p);
fa_status fa_paged_store_validate(const fa_paged_store_params* p);

/* Workspace bytes of the calls below on the calling thread's current device
 * (0: none needed).  They go by the arguments alone, never by device memory. */
fa_status fa_paged_fwd_workspace_size(const fa_paged_fwd_params* p, uint64_t* bytes);
fa_status fa_paged_key_weights_workspace_size(const fa_paged_weights_params* p, uint64_t* bytes);
fa_status fa_qk_norm_rope_bwd_workspace_size(const fa_qk_norm_bwd_params* p, uint64_t* bytes);

/* Validate, then launch asynchronously on `stream`.  Workspaces are device
 * memory, 16-byte aligned, contents undefined on entry; calls that share one
 * must be ordered.  No call allocates, clears memory with a memset or waits, so
 * each can be captured into a graph. */
fa_status fa_paged_fwd(const fa_paged_fwd_params* p, void* workspace, uint64_t workspace_bytes,
                       void* stream);
fa_status fa_paged_key_weights(const fa_paged_weights_params* p, void* workspace,
                               uint64_t workspace_bytes, void* stream);
fa_status fa_paged_evict(const fa_paged_evict_params* p, void* stream);
fa_status fa_qk_norm_rope(const fa_qk_norm_params* p, void* stream);
fa_status fa_qk_norm_rope_bwd(const fa_qk_norm_bwd_params* p, void* workspace,
                              uint64_t workspace_bytes, void* stream);
fa_status fa_paged_store(const fa_paged_store_params* p, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FA_MI355X_CACHE_H */
