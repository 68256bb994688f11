// Internal interface between the C ABI of the paged cache's operators
// (fa_cache_api.cpp) and their HIP kernels.  Strides are in bytes here.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <math.h>

#include "fa_fwd_kernel.h"
#include "fa_score.h"

// Arithmetic that the host's plans and the kernels share.
#if defined(__HIPCC__)
#define FA_PLAN_FN __host__ __device__ __forceinline__
#else
#define FA_PLAN_FN inline
#endif

namespace fa {

// Sequences over a paged cache (fa_paged_cache): table, lengths and limits.
struct PageTable {
  const int32_t* table;
  const int32_t* cu;
  const int32_t* lens;
  int64_t table_stride;  // elements
  int32_t batch, num_pages, page_shift;
  int32_t tokens;        // cu's limit
  int32_t max_kv;        // lens' limit, at most the table's capacity
};

// Rows of a workgroup: the new tokens of a sequence times the query heads of
// one kv head, row r = token r / group, head r % group of them, so that every
// key row read serves the whole group.
struct PagedFwdArgs {
  PageTable pt;
  const char* q;
  const char* k;
  const char* v;
  char* o;
  float* lse;
  int64_t q_st, q_sh, o_st, o_sh;  // token, head
  int64_t k_sp, k_sh, v_sp, v_sh;  // page, head
  uint32_t k_ss, v_ss;             // key
  int32_t heads, kv_heads, group;
  int32_t max_q, causal;
  float scale_log2;                // softmax scale * log2(e)
  // Grids.  Decode kernel: slots (sequences) x kv heads x splits of `chunk` keys.
  // Chunk kernel: at most `slots` row tiles per kv head, and up to max_pieces
  // pieces of the last ones (LastRound; 0: none is cut).
  int32_t slots, splits, chunk;
  int32_t conc, max_pieces;        // workgroups of a kv head that run at once, its most pieces
  float piece_cost;
  // Merge: lane groups of a row; rows of a workgroup (tiles), of a slot (decode).
  int32_t join, merge_rows, most_rows;
  FastDiv by_group, by_kvh, by_splits, by_conc;
  // Order of the chunk kernel's grid (set_order).
  int32_t places, per_xcd, unit_group, xcds, xcd_cus;
  FastDiv by_group_places, by_unit_group;
  float* ws_o;                     // [slot or piece][BM][D] partial o, fp32, of each kv head
  float* ws_e;                     // the same rows: (log2 of the rounded P's sum, of the plain one's)
  ScoreArgs score;                 // read by the scored kernels only
};

// Cost of a piece of a tile beside its keys (LastRound): the time of 768 keys,
// in units of a tile that sees max_kv of them.
inline float piece_cost(int64_t max_kv) { return 768.0f / (float)(max_kv > 768 ? max_kv : 768); }

// Tiles of the chunk kernel's list, of `found` that the offsets make: offsets
// that ascend make at most `slots`, others may make more, which are left out.
FA_PLAN_FN int listed_tiles(int found, int slots) { return found < slots ? found : slots; }

// Time of the last round's tiles cut into q pieces each, `all` in all, in units
// of a tile: rounds of pieces, each 1 / q of a tile and a piece's own cost.  The
// workspace holds max_pieces of them, so more are never cut.
FA_PLAN_FN float cut_cost(int all, int rounds, int q, int max_pieces, float piece_cost) {
  return q > 1 && all > max_pieces ? INFINITY : (float)rounds * (1.0f / (float)q + piece_cost);
}

// Place in the workspace, in tiles, of a piece of the tile-th tile of the last
// round: below max_pieces for each kv head (tile * pieces + piece < all).
FA_PLAN_FN int64_t partial_tile(int kvh, int max_pieces, int tile, int pieces, int piece) {
  return (int64_t)kvh * max_pieces + tile * pieces + piece;
}

// How a call is launched (plan_paged): on the decode kernel where no sequence
// has more than kDecodeRows rows, else on the chunk kernel.
constexpr int kDecodeRows = 32;
constexpr int kChunkRows = 128;

struct PagedGrid {
  int32_t rows;  // rows of a slot (BM): kChunkRows, or 16 or 32
  int32_t slots;
  int32_t splits, chunk;  // decode
  int32_t conc, pieces;   // chunk: at once per kv head, most pieces per kv head
  int32_t keys;           // most keys that a tile sees
  uint64_t ws_rows;       // rows of partials
};
struct PagedPlan {
  PagedGrid grid;
  int32_t compute_units;
  uint64_t workspace_bytes;
};
PagedPlan plan_paged(int tokens, int batch, int kv_heads, int group, int head_dim, int max_q,
                     int max_kv, bool causal, int compute_units, int window = 0);

hipError_t launch_paged_fwd(const PagedFwdArgs& args, const PagedPlan& plan, int head_dim, bool bf16,
                            void* workspace, hipStream_t stream);
// The same with args.score.
hipError_t launch_paged_scored(const PagedFwdArgs& args, const PagedPlan& plan, int head_dim, bool bf16,
                               void* workspace, hipStream_t stream);

struct PagedWeightsArgs {
  PageTable pt;
  const char* q;
  const char* k;
  const float* lse;
  float* w;
  int64_t q_st, q_sh, k_sp, k_sh;
  int64_t w_sp, w_sh;  // elements
  uint32_t k_ss;
  int32_t heads, kv_heads, group, max_q, causal;
  float scale_log2;
  // Many rows, sequences of min_rows or more; grid: sequences x kv heads x
  // places x row splits, a place being a key tile, or with `pairs` the n-th and
  // the n-th last.
  int32_t min_rows;
  int32_t key_tiles, splits, pairs, places;
  FastDiv by_group, by_kvh, by_tiles, by_places, by_batch, by_splits;
  float* ws;           // [splits][batch][kv_heads][key_tiles * 256] partial sums
  // Few rows, at most max_rows; grid: sequences x kv heads x chunks of keys.
  int32_t max_rows, few_keys, few_chunks;
  FastDiv by_few;
};
constexpr int kWeightKeys = 256;    // keys of a workgroup, many rows
constexpr int kWeightChunk = 2048;  // most keys of a workgroup, few rows
struct WeightsPlan {
  int32_t few_rows;  // 16 or 32: sequences of at most so many rows apart; 0: none
  int32_t few_keys;  // their keys a workgroup
  int32_t splits;    // row splits of the others (1: no workspace); 0: none
  int32_t pairs;     // 1: key tiles in pairs
};
WeightsPlan plan_weights(int tokens, int batch, int kv_heads, int group, int head_dim, int max_q,
                         int max_kv, int compute_units);
hipError_t launch_paged_weights(const PagedWeightsArgs& args, const WeightsPlan& plan, int head_dim,
                                bool bf16, hipStream_t stream);

struct PagedEvictArgs {
  PageTable pt;  // cu unused
  char* k;
  char* v;
  float* w;
  int64_t k_sp, k_sh, v_sp, v_sh;
  int64_t w_sp, w_sh;  // elements
  uint32_t k_ss, v_ss;
  int32_t kv_heads;
  const int32_t* new_table;
  int64_t new_table_stride;
  int32_t* new_lens;
  int32_t* kept;
  int32_t keep, recent;
};
hipError_t launch_paged_evict(const PagedEvictArgs& args, int head_dim, hipStream_t stream);

// Rows of q and k (and v, to be copied, when storing) of a grid of tokens;
// [0] q, [1] k, [2] v.
struct NormArgs {
  const char* x[3];
  char* y[3];                     // outputs; storing: y[1], y[2] are the cache
  int64_t x_sb[3], x_sh[3], x_st[3];  // batch, head, token
  int64_t y_sb[3], y_sh[3], y_st[3];  // storing: page, head, key for [1] and [2]
  const void* weight[2];
  const float* cos;
  const float* sin;
  const int32_t* positions;
  int64_t pos_stride;             // elements
  int32_t axes;                   // positions of a token; 0: one for all pairs of dims
  int64_t axis_stride;            // elements from one axis's positions to the next's
  uint64_t axis_bits[2];          // two bits a pair: its axis
  PageTable pt;                   // storing only
  int32_t tokens;                 // of all sequences: batch * seq_len
  int32_t seq_len;                // tokens of one batch entry
  int32_t heads, kv_heads, head_dim;
  int32_t rot, table_rows, interleaved, weight_fp32;
  float eps;
  FastDiv by_seq;
  // backward: dx's; the weights' partial sums [blocks][2][D] and results
  char* dx[2];
  int64_t dx_sb[2], dx_sh[2], dx_st[2];
  float* ws;
  float* dw[2];
  int32_t blocks_x, head_chunk;   // grid: token blocks x chunks of heads
};
hipError_t launch_norm(const NormArgs& args, bool bf16, bool store, int compute_units,
                       hipStream_t stream);
// Workgroups of the backward pass, each with 2 * D partial sums.
int norm_bwd_blocks(int64_t tokens, int heads, int head_dim, int compute_units);
hipError_t launch_norm_bwd(const NormArgs& args, bool bf16, int compute_units, hipStream_t stream);

}  // namespace fa
