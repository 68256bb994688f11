// C ABI of the paged cache's operators and of the q/k norm with rotation
// (declared in include/fa_mi355x_cache.h): argument checks, launch plans and
// workspace layout.  The checks are host code that touches no GPU, as
// fa_fwd_validate's.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "fa_cache_kernels.h"
#include "fa_checks.h"
#include "fa_host.h"
#include "fa_mi355x_attention.h"
#include "fa_mi355x_cache.h"

namespace fa {

// Whether the chunk kernel may cut the tiles of its last round in pieces
// (LastRound), for every number of tiles that sequences of `rows` rows in all
// can have.  Where it may not, the call is spared the launch that joins them.
static bool cuts_tiles(int64_t rows, int batch, int conc, int max_pieces, float piece_cost) {
  if (conc == 1) return false;  // whole rounds only
  if (batch > 8) return true;
  const int64_t least = (rows + kChunkRows - 1) / kChunkRows;
  const int64_t most = std::max(least, (rows - batch) / kChunkRows + batch);
  for (int64_t n = least; n <= most; ++n) {
    const int64_t rest = n % conc;
    for (int q = 2; rest > 0 && q <= 64; ++q) {
      const int64_t all = rest * q;
      if (cut_cost((int)all, (int)((all + conc - 1) / conc), q, max_pieces, piece_cost) < 1.0f + piece_cost)
        return true;
    }
  }
  return false;
}

PagedPlan plan_paged(int tokens, int batch, int kv_heads, int group, int head_dim, int max_q,
                     int max_kv, bool causal, int compute_units, int window) {
  PagedPlan p = {};
  p.compute_units = compute_units;
  PagedGrid& g = p.grid;
  const int64_t most = (int64_t)std::min(max_q, tokens) * group;  // rows of a sequence
  int64_t keys = std::max(max_kv, 1);
  if (window > 0) {
    // What the tokens of a tile see in a window, from a tile of keys on.
    const int64_t tokens_of = most > kDecodeRows ? std::min<int64_t>(max_q, (kChunkRows + group - 1) / group + 1) : max_q;
    keys = std::min<int64_t>(keys, (causal ? 1 : 2) * (int64_t)window + tokens_of + 63);
    causal = false;  // (tiles of a window are of one length)
  }
  g.keys = (int)keys;
  if (most > kDecodeRows) {
    // All sequences of the call, those of few rows too: one launch after the
    // other for the two kinds was 10 to 30 % slower in mixes of like lengths (us,
    // two launches and one: 63 sequences of one token and one of 64, of up to 8000
    // keys, 32 heads on 8, D = 128: 341, 297; 60 and 4 of 512: 493, 387; 16 of
    // up to 64 tokens over 3000 keys: 74, 55).  It is not where a sequence of few
    // rows is far longer than the others, whose tile is a whole one here: one
    // token over 131072 keys and a prompt of 2048, 102 and 49 in two calls, 2336
    // in one.
    g.rows = kChunkRows;
    const int64_t rows = (int64_t)tokens * group;
    g.slots = (int)(rows / kChunkRows + batch);
    // Two workgroups per CU; the tiles of the last round go in pieces of 512
    // keys or more, two rounds of them at most.  No pieces, and no launch that
    // joins them (5 us), for up to 1024 keys; where LastRound would cut none; and
    // where causal tiles get so much shorter that those of a last round are
    // short (prompts of 2048, 2800 and 4096 tokens, 32 heads on 8, D = 128: 50, 74
    // and 130 us without, 55, 82 and 133 with; but fewer tiles than workgroups
    // hold the longest ones: 2048 tokens, 8 heads on 2: 43 and 34).
    g.conc = std::max(1, 2 * compute_units / kv_heads);
    g.pieces = (int)std::min<int64_t>(2 * (int64_t)g.conc, 64 * (int64_t)g.slots);
    const bool falling = causal && 4 * (int64_t)max_q >= keys;
    if (keys <= 1024 || (falling && rows / kChunkRows >= g.conc) ||
        !cuts_tiles(rows, batch, g.conc, g.pieces, piece_cost(keys)))
      g.pieces = 0;
    g.ws_rows = (uint64_t)g.pieces * kv_heads * g.rows;
  } else {
    g.rows = most <= 16 ? 16 : 32;
    g.slots = batch;
    // One workgroup per CU, of 128 to 8192 keys in whole 64-key tiles (the
    // upper end for batches with one long sequence among short ones); up to 512
    // keys are not split, for the join's launch.  Ragged
    // lengths need no finer cut: a CU whose workgroup ended leaves its bandwidth
    // to the others.  us for 1, 2, 4, 8 workgroups per CU: 32 sequences of up
    // to 8192 keys, 8 kv heads, D = 128: 144, 147, 151, 157; one of 131072: 99,
    // 100, 104, 113; 4 of up to 16000: 44, 44, 48, 48.
    const int64_t base = (int64_t)batch * kv_heads;
    // (the cut for long sequences as far as its partials stay within 128 MiB)
    const int64_t part = base * g.rows * (head_dim + 2) * 4;
    const int64_t want = std::max<int64_t>(
        std::min((keys + 8191) / 8192, std::max<int64_t>(1, (int64_t(128) << 20) / part)),
        keys <= 512 ? 1 : std::min((compute_units + base - 1) / base, (keys + 127) / 128));
    g.chunk = (int)(((keys + want - 1) / want + 63) / 64 * 64);
    g.splits = (int)((keys + g.chunk - 1) / g.chunk);
    g.ws_rows = g.splits > 1 ? (uint64_t)base * g.splits * g.rows : 0;
  }
  p.workspace_bytes = g.ws_rows * (head_dim + 2) * 4;
  return p;
}

WeightsPlan plan_weights(int tokens, int batch, int kv_heads, int group, int head_dim, int max_q,
                         int max_kv, int compute_units) {
  WeightsPlan p = {};
  const int64_t most = (int64_t)std::min(max_q, tokens) * group;  // rows of a sequence
  // Beside sequences of many rows, those of few get a kernel of their own where
  // the cache is large (K of more than 384 MiB; us, two kernels and one: 63
  // sequences of one token and one of 64, of up to 8000 keys, D = 128: 8 kv heads,
  // 1 GB, 178 and 212; 2 kv heads, 0.26 GB, 63 and 53), and where there may be any:
  // no sequence can have so few tokens if the others, at max_q, leave it more.
  const int64_t least = tokens - (int64_t)(batch - 1) * max_q;
  const int64_t k_bytes = (int64_t)batch * kv_heads * max_kv * head_dim * 2;
  if (most <= kDecodeRows || (batch > 1 && k_bytes > (int64_t(384) << 20) && least * group <= kDecodeRows)) {
    p.few_rows = most <= 16 ? 16 : kDecodeRows;
    // Four workgroups per CU, which run at once, of 256 to 2048 keys in whole
    // 64-key tiles.
    const int64_t bk = (int64_t)batch * kv_heads;
    const int64_t cut = (4 * (int64_t)compute_units + bk - 1) / bk;
    const int64_t keys = ((max_kv + cut - 1) / cut + 63) / 64 * 64;
    p.few_keys = (int)std::max<int64_t>(256, std::min<int64_t>(keys, kWeightChunk));
  }
  if (most > kDecodeRows) {
    // Three workgroups per CU run at once; row splits fill them, of a row tile or
    // more.  Where new tokens are many of the keys, causal masks leave the first
    // key tile all rows and the last one few: then tiles go in pairs of equal
    // work if that is long (4 prompts of 4096 tokens, 4 kv heads: 251 -> 151
    // us), and are cut finer if it is short, twice over for splits of four row
    // tiles (28 prompts of up to 1613, one kv head: 45 -> 33 us; a pair starts
    // twice, 46 us), else up to two workgroups per CU (prompts of 256, 512 and
    // 1000 tokens, 8 kv heads, group 4: 9.6, 12 and 21 us; 15, 16 and 23 with four
    // row tiles at least, 9.6, 12 and 27 with one at any number).
    const int64_t tiles = (max_kv + kWeightKeys - 1) / kWeightKeys;
    const int64_t bk = (int64_t)batch * kv_heads;
    // (Up to 256 rows are not split, for the launch that adds the splits up; 512
    // over 2000 keys, 8 kv heads: 21 us without, 12 with.)
    auto cut = [&](int64_t places, int per_cu, int rows) {
      if (most <= 256) return 1;
      const int64_t want = per_cu * (int64_t)compute_units / std::max<int64_t>(bk * places, 1);
      return (int)std::max<int64_t>(1, std::min(want, most / rows));
    };
    p.splits = cut(tiles, 3, 64);
    if (4 * (int64_t)max_q >= max_kv) {
      p.pairs = most / 64 >= 32 * (int64_t)p.splits;
      p.splits = p.pairs ? cut((tiles + 1) / 2, 3, 64) : std::max(cut(tiles, 6, 256), cut(tiles, 2, 64));
    }
  }
  return p;
}

namespace {

using Wide = __int128;  // strides times sizes

Wide floor_div(Wide a, Wide b) { return a / b - (a % b < 0 ? 1 : 0); }

// Whether some i[d] of lo[d]..hi[d] make -row_a < delta + sum i[d] stride[d] < row_b,
// strides descending.  A stride that spans what the smaller ones reach leaves two
// or three values to look at; overlapping rows, more, count as a meeting.
bool meets(Wide delta, const int64_t* stride, const int64_t* lo, const int64_t* hi, int n, int64_t row_a,
           int64_t row_b) {
  if (n == 0) return -row_a < delta && delta < row_b;
  Wide least = 0, most = 0;  // of the smaller strides' sum
  for (int d = 1; d < n; ++d) {
    least += (Wide)lo[d] * stride[d];
    most += (Wide)hi[d] * stride[d];
  }
  const Wide s = stride[0];
  const Wide first = std::max<Wide>(lo[0], -floor_div(-(-row_a + 1 - delta - most), s));
  const Wide last = std::min<Wide>(hi[0], floor_div(row_b - 1 - delta - least, s));
  if (last - first > 3) return true;
  for (Wide i = first; i <= last; ++i)
    if (meets(delta + i * s, stride + 1, lo + 1, hi + 1, n - 1, row_a, row_b)) return true;
  return false;
}

int64_t gcd(int64_t a, int64_t b) { return b == 0 ? a : gcd(b, a % b); }

}  // namespace

bool may_overlap(const RowSet& a, const RowSet& b) {
  Wide reach[2];
  const RowSet* sets[2] = {&a, &b};
  for (int x = 0; x < 2; ++x) {
    reach[x] = sets[x]->row;
    for (int d = 0; d < sets[x]->n; ++d) {
      if (sets[x]->size[d] == 0) return false;
      if (sets[x]->size[d] == 1) continue;
      reach[x] += (Wide)sets[x]->stride[d] * (sets[x]->size[d] - 1);
    }
  }
  const Wide bytes = (Wide)(intptr_t)b.base - (Wide)(intptr_t)a.base;
  if (bytes >= 2 * reach[0] || -bytes >= 2 * reach[1]) return false;
  if (bytes % 2 != 0) return true;
  const Wide delta = bytes / 2;  // of b's first row behind a's
  int64_t stride[3], lo[3], hi[3];
  int n = 0;
  bool same = a.n == b.n;
  for (int d = 0; same && d < a.n; ++d) {
    same = a.size[d] == 1 || b.size[d] == 1 || a.stride[d] == b.stride[d];
    const int64_t s = a.size[d] > 1 ? a.stride[d] : b.stride[d];
    if (s == 0 || (a.size[d] == 1 && b.size[d] == 1)) continue;
    int at = n++;
    for (; at > 0 && stride[at - 1] < s; --at) {
      stride[at] = stride[at - 1];
      lo[at] = lo[at - 1];
      hi[at] = hi[at - 1];
    }
    stride[at] = s;
    lo[at] = -(a.size[d] - 1);
    hi[at] = b.size[d] - 1;
  }
  // b's rows start at delta + sum i_b stride, a's at sum i_a stride
  if (same) return meets(delta, stride, lo, hi, n, b.row, a.row);
  int64_t common = 0;
  for (const RowSet* r : sets)
    for (int d = 0; d < r->n; ++d)
      if (r->size[d] > 1) common = gcd(common, r->stride[d]);
  if (common == 0) return true;
  const Wide at = ((delta % common) + common) % common;
  return at < a.row || at + b.row > common;
}

namespace {

// written: the call writes k and v.  v may be absent where with_v is false.
fa_status check_cache(const fa_paged_cache& c, bool with_v, bool with_cu, bool written) {
  FA_TRY(check_dtype(c.dtype));
  FA_TRY(check_head_dim(c.head_dim));
  if (c.batch < 0 || c.num_pages < 1 || c.max_pages < 1 || c.kv_heads < 1)
    return fail(FA_ERR_SHAPE, "batch=%d must be >= 0, num_pages=%d max_pages=%d kv_heads=%d >= 1",
                (int)c.batch, (int)c.num_pages, (int)c.max_pages, (int)c.kv_heads);
  if (c.page_size < 16 || c.page_size > 4096 || (c.page_size & (c.page_size - 1)) != 0)
    return fail(FA_ERR_SHAPE, "page_size %d is not a power of two from 16 to 4096", (int)c.page_size);
  if ((int64_t)c.max_pages * c.page_size > (int64_t(1) << 30))
    return fail(FA_ERR_UNSUPPORTED, "max_pages * page_size = %lld exceeds 2^30",
                (long long)c.max_pages * c.page_size);
  const int64_t size[3] = {c.num_pages, c.kv_heads, c.page_size};
  FA_TRY(check_rows("k_cache", c.k, c.k_stride, 3));
  FA_TRY(check_written("k_cache", c.k_stride + 2, size + 2, 1, c.head_dim));
  if (c.k_stride[2] > kMaxKeyStride)
    return fail(FA_ERR_UNSUPPORTED, "k_cache key stride %lld exceeds %lld elements",
                (long long)c.k_stride[2], (long long)kMaxKeyStride);
  if (with_v) {
    FA_TRY(check_rows("v_cache", c.v, c.v_stride, 3));
    FA_TRY(check_written("v_cache", c.v_stride + 2, size + 2, 1, c.head_dim));
    if (c.v_stride[2] > kMaxKeyStride)
      return fail(FA_ERR_UNSUPPORTED, "v_cache key stride %lld exceeds %lld elements",
                  (long long)c.v_stride[2], (long long)kMaxKeyStride);
  }
  if (written) {
    FA_TRY(check_written("k_cache", c.k_stride, size, 3, c.head_dim));
    FA_TRY(check_written("v_cache", c.v_stride, size, 3, c.head_dim));
  }
  if (c.batch == 0) return FA_OK;  // no sequence: the tables are not read
  FA_TRY(check_int32("block_table", c.block_table));
  FA_TRY(check_int32("seq_lens", c.seq_lens));
  if (with_cu) FA_TRY(check_int32("cu_seqlens", c.cu_seqlens));
  if (c.batch > 1 && c.table_stride < c.max_pages)
    return fail(FA_ERR_STRIDE, "block_table row stride %lld is smaller than max_pages %d",
                (long long)c.table_stride, (int)c.max_pages);
  return FA_OK;
}

// Packed queries: tokens, heads, limits.
fa_status check_queries(const fa_paged_cache& c, int32_t tokens, int32_t heads, int32_t max_q,
                        int32_t max_kv, float scale, int32_t causal) {
  if (tokens < 0) return fail(FA_ERR_SHAPE, "tokens=%d must be >= 0", (int)tokens);
  if (heads < 1 || heads % c.kv_heads != 0)
    return fail(FA_ERR_SHAPE, "heads=%d must be a positive multiple of kv_heads=%d", (int)heads,
                (int)c.kv_heads);
  if (max_q < 0 || max_kv < 0)
    return fail(FA_ERR_ARG, "max_q=%d and max_kv=%d must be >= 0", (int)max_q, (int)max_kv);
  FA_TRY(check_flag("causal", causal));
  FA_TRY(check_scale(scale));
  if ((int64_t)tokens * heads > kMaxRows)
    return fail(FA_ERR_UNSUPPORTED, "tokens*heads = %lld exceeds 2^31-256", (long long)tokens * heads);
  if ((int64_t)c.batch * c.kv_heads > 0x7fffff)
    return fail(FA_ERR_UNSUPPORTED, "batch*kv_heads = %lld exceeds 2^23-1",
                (long long)c.batch * c.kv_heads);
  return FA_OK;
}

int32_t limit_kv(const fa_paged_cache& c, int32_t max_kv) {
  return std::min(max_kv, c.max_pages * c.page_size);
}

int log2_of(int32_t n) {
  int s = 0;
  while ((1 << s) < n) ++s;
  return s;
}

PageTable page_table(const fa_paged_cache& c, int32_t tokens, int32_t max_kv) {
  PageTable t = {};
  t.table = c.block_table;
  t.cu = c.cu_seqlens;
  t.lens = c.seq_lens;
  t.table_stride = c.table_stride;
  t.batch = c.batch;
  t.num_pages = c.num_pages;
  t.page_shift = log2_of(c.page_size);
  t.tokens = tokens;
  t.max_kv = max_kv;
  return t;
}

// Largest byte offset of a tile's rows from its first (64 tokens, or fewer of a
// group of heads), which the key weights' staging holds in 32 bits.
fa_status check_tile_reach(const int64_t st[2], int32_t group) {
  if (st[0] > kMaxKeyStride || (int64_t)(group - 1) * st[1] > (int64_t(1) << 28))
    return fail(FA_ERR_UNSUPPORTED, "q strides %lld, %lld exceed the kernel's range", (long long)st[0],
                (long long)st[1]);
  return FA_OK;
}

fa_status check_norm(const void* qw, const void* kw, const float* cos, const float* sin, int32_t rot,
                     int32_t rows, int32_t interleaved, int32_t weight_fp32, float eps, int32_t d) {
  if (qw == nullptr || kw == nullptr) return fail(FA_ERR_NULL, "a norm weight is NULL");
  if (cos == nullptr || sin == nullptr) return fail(FA_ERR_NULL, "cos or sin is NULL");
  for (const void* p : {qw, kw, (const void*)cos, (const void*)sin})
    if (!aligned(p, 16))
      return fail(FA_ERR_STRIDE, "norm weights, cos and sin must be 16-byte aligned");
  if (rot < 16 || rot > d || rot % 16 != 0)
    return fail(FA_ERR_ARG, "rot=%d must be a multiple of 16 from 16 to head_dim %d", (int)rot, (int)d);
  if (rows < 1) return fail(FA_ERR_SHAPE, "table_rows=%d must be >= 1", (int)rows);
  FA_TRY(check_flag("interleaved", interleaved));
  FA_TRY(check_flag("weight_fp32", weight_fp32));
  if (!std::isfinite(eps) || eps < 0.0f)
    return fail(FA_ERR_ARG, "eps must be finite and >= 0 (got %g)", (double)eps);
  return FA_OK;
}

NormArgs norm_args(const fa_qk_norm_params& p) {
  NormArgs n = {};
  const void* x[2] = {p.q, p.k};
  void* y[2] = {p.q_out, p.k_out};
  const int64_t* xs[2] = {p.q_stride, p.k_stride};
  const int64_t* ys[2] = {p.q_out_stride, p.k_out_stride};
  for (int i = 0; i < 2; ++i) {
    n.x[i] = static_cast<const char*>(x[i]);
    n.y[i] = static_cast<char*>(y[i]);
    n.x_sb[i] = 2 * xs[i][0];
    n.x_sh[i] = 2 * xs[i][1];
    n.x_st[i] = 2 * xs[i][2];
    n.y_sb[i] = 2 * ys[i][0];
    n.y_sh[i] = 2 * ys[i][1];
    n.y_st[i] = 2 * ys[i][2];
  }
  n.weight[0] = p.q_weight;
  n.weight[1] = p.k_weight;
  n.cos = p.cos;
  n.sin = p.sin;
  n.positions = p.positions;
  n.pos_stride = p.pos_stride;
  n.tokens = (int32_t)((int64_t)p.batch * p.seq_len);
  n.seq_len = p.seq_len;
  n.heads = p.heads;
  n.kv_heads = p.kv_heads;
  n.head_dim = p.head_dim;
  n.rot = p.rot;
  n.table_rows = p.table_rows;
  n.interleaved = p.interleaved;
  n.weight_fp32 = p.weight_fp32;
  n.eps = p.eps;
  n.by_seq = make_fast_div((uint32_t)p.seq_len);
  return n;
}

// The axes of a rotation by `pairs` pairs at `positions`.
fa_status check_axes(const fa_rotary_axes* axes, int pairs, const int32_t* positions) {
  if (axes == nullptr) return fail(FA_ERR_NULL, "axes is NULL");
  if (axes->axes < 1 || axes->axes > 4) return fail(FA_ERR_ARG, "axes must be 1 to 4 (got %d)", (int)axes->axes);
  for (int i = 0; i < pairs; ++i)
    if (axes->axis[i] >= axes->axes)
      return fail(FA_ERR_ARG, "pair %d turns by axis %d of %d", i, (int)axes->axis[i], (int)axes->axes);
  if (axes->axis_stride < 0) return fail(FA_ERR_STRIDE, "axis_stride is negative");
  if (positions == nullptr) return fail(FA_ERR_NULL, "positions is NULL, but a token has several");
  return FA_OK;
}

void set_axes(NormArgs& n, const fa_rotary_axes& axes) {
  n.axes = axes.axes;
  n.axis_stride = axes.axis_stride;
  n.axis_bits[0] = n.axis_bits[1] = 0;
  for (int i = 0; i < n.rot / 2; ++i) n.axis_bits[i / 32] |= (uint64_t)axes.axis[i] << (2 * (i % 32));
}

fa_status check_norm_params(const fa_qk_norm_params* p, bool backward) {
  FA_TRY(check_dtype(p->dtype));
  FA_TRY(check_head_dim(p->head_dim));
  if (p->batch < 1 || p->heads < 1 || p->kv_heads < 1 || p->seq_len < 1)
    return fail(FA_ERR_SHAPE, "batch=%d heads=%d kv_heads=%d seq_len=%d must all be >= 1", (int)p->batch,
                (int)p->heads, (int)p->kv_heads, (int)p->seq_len);
  if ((int64_t)p->batch * p->seq_len > kMaxRows ||
      (int64_t)p->batch * p->seq_len * ((int64_t)p->heads + p->kv_heads) > (int64_t(1) << 36))
    return fail(FA_ERR_UNSUPPORTED, "batch*seq_len and its heads exceed the kernel's range");
  const int64_t qs[3] = {p->batch, p->heads, p->seq_len}, ks[3] = {p->batch, p->kv_heads, p->seq_len};
  FA_TRY(check_rows("q", p->q, p->q_stride, 3));
  FA_TRY(check_rows("k", p->k, p->k_stride, 3));
  FA_TRY(check_rows(backward ? "q's gradient" : "q_out", p->q_out, p->q_out_stride, 3));
  FA_TRY(check_rows(backward ? "k's gradient" : "k_out", p->k_out, p->k_out_stride, 3));
  if (!backward) {
    FA_TRY(check_written("q_out", p->q_out_stride, qs, 3, p->head_dim));
    FA_TRY(check_written("k_out", p->k_out_stride, ks, 3, p->head_dim));
  }
  FA_TRY(check_norm(p->q_weight, p->k_weight, p->cos, p->sin, p->rot, p->table_rows, p->interleaved,
                    p->weight_fp32, p->eps, p->head_dim));
  FA_TRY(check_int32("positions", p->positions, false));
  if (p->pos_stride < 0) return fail(FA_ERR_STRIDE, "positions row stride is negative");
  return FA_OK;
}

}  // namespace
}  // namespace fa

using namespace fa;

extern "C" {

fa_status fa_paged_fwd_validate(const fa_paged_fwd_params* p) {
  clear_error();
  if (p == nullptr) return fail(FA_ERR_NULL, "params is NULL");
  FA_TRY(check_cache(p->cache, true, true, false));
  FA_TRY(check_queries(p->cache, p->tokens, p->heads, p->max_q, p->max_kv, p->softmax_scale, p->causal));
  if (p->tokens == 0) return FA_OK;
  const int64_t size[2] = {p->tokens, p->heads};
  FA_TRY(check_rows("q", p->q, p->q_stride, 2));
  FA_TRY(check_rows("o", p->o, p->o_stride, 2));
  FA_TRY(check_written("o", p->o_stride, size, 2, p->cache.head_dim));
  if (p->lse != nullptr && !aligned(p->lse, 4))
    return fail(FA_ERR_STRIDE, "lse pointer is not 4-byte aligned");
  return FA_OK;
}

fa_status fa_paged_key_weights_validate(const fa_paged_weights_params* p) {
  clear_error();
  if (p == nullptr) return fail(FA_ERR_NULL, "params is NULL");
  FA_TRY(check_cache(p->cache, false, true, false));
  FA_TRY(check_queries(p->cache, p->tokens, p->heads, p->max_q, p->max_kv, p->softmax_scale, p->causal));
  if (p->key_weights == nullptr) return fail(FA_ERR_NULL, "key_weights is NULL");
  if (!aligned(p->key_weights, 4)) return fail(FA_ERR_STRIDE, "key_weights pointer is not 4-byte aligned");
  const int64_t w[2] = {p->cache.num_pages, p->cache.kv_heads};
  FA_TRY(check_written("key_weights", p->w_stride, w, 2, p->cache.page_size));
  if (p->tokens == 0) return FA_OK;
  FA_TRY(check_rows("q", p->q, p->q_stride, 2));
  FA_TRY(check_tile_reach(p->q_stride, p->heads / p->cache.kv_heads));
  if (p->lse == nullptr) return fail(FA_ERR_NULL, "lse is NULL");
  if (!aligned(p->lse, 4)) return fail(FA_ERR_STRIDE, "lse pointer is not 4-byte aligned");
  return FA_OK;
}

fa_status fa_paged_evict_validate(const fa_paged_evict_params* p) {
  clear_error();
  if (p == nullptr) return fail(FA_ERR_NULL, "params is NULL");
  const fa_paged_cache& c = p->cache;
  FA_TRY(check_cache(c, true, false, true));
  if (p->key_weights == nullptr) return fail(FA_ERR_NULL, "key_weights is NULL");
  if (!aligned(p->key_weights, 4)) return fail(FA_ERR_STRIDE, "key_weights pointer is not 4-byte aligned");
  const int64_t w[2] = {c.num_pages, c.kv_heads};
  FA_TRY(check_written("key_weights", p->w_stride, w, 2, c.page_size));
  if (p->keep < 1 || p->recent < 0 || p->recent > p->keep)
    return fail(FA_ERR_ARG, "keep=%d must be >= 1 and recent=%d from 0 to keep", (int)p->keep,
                (int)p->recent);
  if (p->keep > 1 << 30) return fail(FA_ERR_UNSUPPORTED, "keep=%d exceeds 2^30", (int)p->keep);
  if (p->max_kv < 0) return fail(FA_ERR_ARG, "max_kv=%d must be >= 0", (int)p->max_kv);
  if ((int64_t)c.batch * c.kv_heads > 0x7fffff)
    return fail(FA_ERR_UNSUPPORTED, "batch*kv_heads = %lld exceeds 2^23-1", (long long)c.batch * c.kv_heads);
  const int64_t most = std::min<int64_t>(p->keep, (int64_t)c.max_pages * c.page_size);
  if (p->new_pages < 1 || (int64_t)p->new_pages * c.page_size < most)
    return fail(FA_ERR_SHAPE, "new_table's %d pages of %d keys hold fewer than the %lld keys kept",
                (int)p->new_pages, (int)c.page_size, (long long)most);
  if (c.batch == 0) return FA_OK;
  FA_TRY(check_int32("new_table", p->new_table));
  FA_TRY(check_int32("new_lens", p->new_lens));
  FA_TRY(check_int32("kept", p->kept));
  if (c.batch > 1 && p->new_table_stride < p->new_pages)
    return fail(FA_ERR_STRIDE, "new_table row stride %lld is smaller than new_pages %d",
                (long long)p->new_table_stride, (int)p->new_pages);
  if (p->new_table == c.block_table)
    return fail(FA_ERR_ARG, "new_table is block_table: the kept keys go to pages of their own");
  return FA_OK;
}

fa_status fa_qk_norm_rope_validate(const fa_qk_norm_params* p) {
  clear_error();
  if (p == nullptr) return fail(FA_ERR_NULL, "params is NULL");
  return check_norm_params(p, false);
}

fa_status fa_qk_norm_rope_bwd_validate(const fa_qk_norm_bwd_params* p) {
  clear_error();
  if (p == nullptr) return fail(FA_ERR_NULL, "params is NULL");
  const fa_qk_norm_params& f = p->fwd;
  FA_TRY(check_norm_params(&f, true));
  const int64_t qs[3] = {f.batch, f.heads, f.seq_len}, ks[3] = {f.batch, f.kv_heads, f.seq_len};
  FA_TRY(check_rows("dq", p->dq, p->dq_stride, 3));
  FA_TRY(check_written("dq", p->dq_stride, qs, 3, f.head_dim));
  FA_TRY(check_rows("dk", p->dk, p->dk_stride, 3));
  FA_TRY(check_written("dk", p->dk_stride, ks, 3, f.head_dim));
  if (p->dq_weight == nullptr || p->dk_weight == nullptr)
    return fail(FA_ERR_NULL, "a weight's gradient is NULL");
  if (!aligned(p->dq_weight, 4) || !aligned(p->dk_weight, 4))
    return fail(FA_ERR_STRIDE, "weight gradients must be 4-byte aligned");
  return FA_OK;
}

fa_status fa_paged_store_validate(const fa_paged_store_params* p) {
  clear_error();
  if (p == nullptr) return fail(FA_ERR_NULL, "params is NULL");
  const fa_paged_cache& c = p->cache;
  FA_TRY(check_cache(c, true, true, true));
  if (p->tokens < 0 || p->heads < 1)
    return fail(FA_ERR_SHAPE, "tokens=%d must be >= 0 and heads=%d >= 1", (int)p->tokens, (int)p->heads);
  if (p->tokens > kMaxRows ||
      (int64_t)p->tokens * ((int64_t)p->heads + 2 * c.kv_heads) > (int64_t(1) << 36))
    return fail(FA_ERR_UNSUPPORTED, "tokens and heads exceed the kernel's range");
  FA_TRY(check_norm(p->q_weight, p->k_weight, p->cos, p->sin, p->rot, p->table_rows, p->interleaved,
                    p->weight_fp32, p->eps, c.head_dim));
  if (p->tokens == 0) return FA_OK;
  const int64_t qs[2] = {p->tokens, p->heads};
  FA_TRY(check_rows("q", p->q, p->q_stride, 2));
  FA_TRY(check_rows("k", p->k, p->k_stride, 2));
  FA_TRY(check_rows("v", p->v, p->v_stride, 2));
  FA_TRY(check_rows("q_out", p->q_out, p->q_out_stride, 2));
  FA_TRY(check_written("q_out", p->q_out_stride, qs, 2, c.head_dim));
  FA_TRY(check_int32("positions", p->positions));
  return FA_OK;
}

}  // extern "C"

namespace {

// Nothing to compute: no row, or no sequence.
bool idle(const fa_paged_fwd_params& p) { return p.tokens == 0 || p.cache.batch == 0 || p.max_q == 0; }
bool idle(const fa_paged_weights_params& p) {
  return p.tokens == 0 || p.cache.batch == 0 || p.max_q == 0 || p.max_kv == 0;
}

fa_status plan_of(const fa_paged_fwd_params& p, int window, PagedPlan* plan) {
  int cus = 0;
  FA_TRY(current_compute_units(&cus));
  *plan = plan_paged(p.tokens, p.cache.batch, p.cache.kv_heads, p.heads / p.cache.kv_heads,
                     p.cache.head_dim, p.max_q, limit_kv(p.cache, p.max_kv), p.causal != 0, cus, window);
  return FA_OK;
}

uint64_t weights_bytes(const fa_paged_weights_params& p, int splits) {
  if (splits <= 1) return 0;
  const int64_t tiles = (limit_kv(p.cache, p.max_kv) + kWeightKeys - 1) / kWeightKeys;
  return (uint64_t)splits * p.cache.batch * p.cache.kv_heads * tiles * kWeightKeys * 4;
}

fa_status plan_of(const fa_paged_weights_params& p, WeightsPlan* plan) {
  int cus = 0;
  FA_TRY(current_compute_units(&cus));
  *plan = plan_weights(p.tokens, p.cache.batch, p.cache.kv_heads, p.heads / p.cache.kv_heads,
                       p.cache.head_dim, p.max_q, limit_kv(p.cache, p.max_kv), cus);
  return FA_OK;
}

uint64_t norm_bwd_bytes(const fa_qk_norm_params& f, int cus) {
  return (uint64_t)norm_bwd_blocks((int64_t)f.batch * f.seq_len, f.heads + f.kv_heads, f.head_dim, cus) *
         2 * f.head_dim * 4;
}

}  // namespace

namespace {

PagedFwdArgs paged_args(const fa_paged_fwd_params* p) {
  const fa_paged_cache& c = p->cache;
  PagedFwdArgs a = {};
  a.pt = page_table(c, p->tokens, limit_kv(c, p->max_kv));
  a.q = static_cast<const char*>(p->q);
  a.k = static_cast<const char*>(c.k);
  a.v = static_cast<const char*>(c.v);
  a.o = static_cast<char*>(p->o);
  a.lse = p->lse;
  a.q_st = 2 * p->q_stride[0];
  a.q_sh = 2 * p->q_stride[1];
  a.o_st = 2 * p->o_stride[0];
  a.o_sh = 2 * p->o_stride[1];
  a.k_sp = 2 * c.k_stride[0];
  a.k_sh = 2 * c.k_stride[1];
  a.k_ss = (uint32_t)(2 * c.k_stride[2]);
  a.v_sp = 2 * c.v_stride[0];
  a.v_sh = 2 * c.v_stride[1];
  a.v_ss = (uint32_t)(2 * c.v_stride[2]);
  a.heads = p->heads;
  a.kv_heads = c.kv_heads;
  a.group = p->heads / c.kv_heads;
  a.max_q = p->max_q;
  a.causal = p->causal;
  a.scale_log2 = (float)(p->softmax_scale * kLog2e);
  a.by_group = make_fast_div((uint32_t)a.group);
  a.by_kvh = make_fast_div((uint32_t)a.kv_heads);
  return a;
}

}  // namespace

extern "C" {

fa_status fa_paged_fwd_workspace_size(const fa_paged_fwd_params* p, uint64_t* bytes) {
  if (bytes == nullptr) return fail(FA_ERR_NULL, "bytes is NULL");
  *bytes = 0;
  FA_TRY(fa_paged_fwd_validate(p));
  if (idle(*p)) return FA_OK;
  PagedPlan plan;
  FA_TRY(plan_of(*p, 0, &plan));
  *bytes = plan.workspace_bytes;
  return FA_OK;
}

fa_status fa_paged_fwd(const fa_paged_fwd_params* p, void* workspace, uint64_t workspace_bytes,
                       void* stream) {
  FA_TRY(fa_paged_fwd_validate(p));
  if (idle(*p)) return FA_OK;
  PagedPlan plan;
  FA_TRY(plan_of(*p, 0, &plan));
  FA_TRY(check_workspace(workspace, workspace_bytes, plan.workspace_bytes));
  return launched(launch_paged_fwd(paged_args(p), plan, p->cache.head_dim, p->cache.dtype == FA_DTYPE_BF16,
                                   workspace, static_cast<hipStream_t>(stream)));
}

fa_status fa_paged_fwd_scored_validate(const fa_paged_fwd_params* p, const fa_score_params* score) {
  FA_TRY(fa_paged_fwd_validate(p));
  if (score == nullptr) return fail(FA_ERR_NULL, "score is NULL");
  return check_score(*score, p->softmax_scale);
}

fa_status fa_paged_fwd_scored_workspace_size(const fa_paged_fwd_params* p, const fa_score_params* score,
                                             uint64_t* bytes) {
  if (bytes == nullptr) return fail(FA_ERR_NULL, "bytes is NULL");
  *bytes = 0;
  FA_TRY(fa_paged_fwd_scored_validate(p, score));
  if (idle(*p)) return FA_OK;
  PagedPlan plan;
  FA_TRY(plan_of(*p, score_args(*score, p->softmax_scale).window, &plan));
  *bytes = plan.workspace_bytes;
  return FA_OK;
}

fa_status fa_paged_fwd_scored(const fa_paged_fwd_params* p, const fa_score_params* score, void* workspace,
                              uint64_t workspace_bytes, void* stream) {
  FA_TRY(fa_paged_fwd_scored_validate(p, score));
  if (score->softcap == 0.0f && score->slopes == nullptr && score->window == 0)
    return fa_paged_fwd(p, workspace, workspace_bytes, stream);
  if (idle(*p)) return FA_OK;
  PagedFwdArgs a = paged_args(p);
  a.score = score_args(*score, p->softmax_scale);
  PagedPlan plan;
  FA_TRY(plan_of(*p, a.score.window, &plan));
  FA_TRY(check_workspace(workspace, workspace_bytes, plan.workspace_bytes));
  return launched(launch_paged_scored(a, plan, p->cache.head_dim, p->cache.dtype == FA_DTYPE_BF16, workspace,
                                      static_cast<hipStream_t>(stream)));
}

fa_status fa_paged_key_weights_workspace_size(const fa_paged_weights_params* p, uint64_t* bytes) {
  if (bytes == nullptr) return fail(FA_ERR_NULL, "bytes is NULL");
  *bytes = 0;
  FA_TRY(fa_paged_key_weights_validate(p));
  if (idle(*p)) return FA_OK;
  WeightsPlan plan;
  FA_TRY(plan_of(*p, &plan));
  *bytes = weights_bytes(*p, plan.splits);
  return FA_OK;
}

fa_status fa_paged_key_weights(const fa_paged_weights_params* p, void* workspace,
                               uint64_t workspace_bytes, void* stream) {
  FA_TRY(fa_paged_key_weights_validate(p));
  if (idle(*p)) return FA_OK;
  WeightsPlan plan;
  FA_TRY(plan_of(*p, &plan));
  const uint64_t need = weights_bytes(*p, plan.splits);
  FA_TRY(check_workspace(workspace, workspace_bytes, need));
  const fa_paged_cache& c = p->cache;
  PagedWeightsArgs a = {};
  a.pt = page_table(c, p->tokens, limit_kv(c, p->max_kv));
  a.q = static_cast<const char*>(p->q);
  a.k = static_cast<const char*>(c.k);
  a.lse = p->lse;
  a.w = p->key_weights;
  a.q_st = 2 * p->q_stride[0];
  a.q_sh = 2 * p->q_stride[1];
  a.k_sp = 2 * c.k_stride[0];
  a.k_sh = 2 * c.k_stride[1];
  a.k_ss = (uint32_t)(2 * c.k_stride[2]);
  a.w_sp = p->w_stride[0];
  a.w_sh = p->w_stride[1];
  a.heads = p->heads;
  a.kv_heads = c.kv_heads;
  a.group = p->heads / c.kv_heads;
  a.max_q = p->max_q;
  a.causal = p->causal;
  a.scale_log2 = (float)(p->softmax_scale * kLog2e);
  a.key_tiles = (a.pt.max_kv + kWeightKeys - 1) / kWeightKeys;
  a.splits = plan.splits;
  a.by_group = make_fast_div((uint32_t)a.group);
  a.by_kvh = make_fast_div((uint32_t)a.kv_heads);
  a.by_tiles = make_fast_div((uint32_t)a.key_tiles);
  a.by_batch = make_fast_div((uint32_t)c.batch);
  a.by_splits = make_fast_div((uint32_t)plan.splits);
  a.ws = need > 0 ? static_cast<float*>(workspace) : nullptr;
  return launched(launch_paged_weights(a, plan, c.head_dim, c.dtype == FA_DTYPE_BF16,
                                       static_cast<hipStream_t>(stream)));
}

fa_status fa_paged_evict(const fa_paged_evict_params* p, void* stream) {
  FA_TRY(fa_paged_evict_validate(p));
  const fa_paged_cache& c = p->cache;
  if (c.batch == 0) return FA_OK;
  PagedEvictArgs a = {};
  a.pt = page_table(c, 0, limit_kv(c, p->max_kv));
  a.k = static_cast<char*>(c.k);
  a.v = static_cast<char*>(c.v);
  a.w = p->key_weights;
  a.k_sp = 2 * c.k_stride[0];
  a.k_sh = 2 * c.k_stride[1];
  a.k_ss = (uint32_t)(2 * c.k_stride[2]);
  a.v_sp = 2 * c.v_stride[0];
  a.v_sh = 2 * c.v_stride[1];
  a.v_ss = (uint32_t)(2 * c.v_stride[2]);
  a.w_sp = p->w_stride[0];
  a.w_sh = p->w_stride[1];
  a.kv_heads = c.kv_heads;
  a.new_table = p->new_table;
  a.new_table_stride = p->new_table_stride;
  a.new_lens = p->new_lens;
  a.kept = p->kept;
  a.keep = p->keep;
  a.recent = p->recent;
  return launched(launch_paged_evict(a, c.head_dim, static_cast<hipStream_t>(stream)));
}

}  // extern "C"

namespace {

fa_status norm_forward(const fa_qk_norm_params& p, const fa_rotary_axes* axes, void* stream) {
  int cus = 0;
  FA_TRY(current_compute_units(&cus));
  NormArgs n = norm_args(p);
  if (axes != nullptr) set_axes(n, *axes);
  return launched(launch_norm(n, p.dtype == FA_DTYPE_BF16, false, cus, static_cast<hipStream_t>(stream)));
}

fa_status norm_backward(const fa_qk_norm_bwd_params* p, const fa_rotary_axes* axes, void* workspace,
                        uint64_t workspace_bytes, void* stream) {
  int cus = 0;
  FA_TRY(current_compute_units(&cus));
  FA_TRY(check_workspace(workspace, workspace_bytes, norm_bwd_bytes(p->fwd, cus)));
  NormArgs n = norm_args(p->fwd);
  if (axes != nullptr) set_axes(n, *axes);
  void* dx[2] = {p->dq, p->dk};
  const int64_t* ds[2] = {p->dq_stride, p->dk_stride};
  for (int i = 0; i < 2; ++i) {
    n.dx[i] = static_cast<char*>(dx[i]);
    n.dx_sb[i] = 2 * ds[i][0];
    n.dx_sh[i] = 2 * ds[i][1];
    n.dx_st[i] = 2 * ds[i][2];
  }
  n.ws = static_cast<float*>(workspace);
  n.dw[0] = p->dq_weight;
  n.dw[1] = p->dk_weight;
  return launched(launch_norm_bwd(n, p->fwd.dtype == FA_DTYPE_BF16, cus, static_cast<hipStream_t>(stream)));
}

fa_status norm_store(const fa_paged_store_params* p, const fa_rotary_axes* axes, void* stream) {
  const fa_paged_cache& c = p->cache;
  if (p->tokens == 0 || c.batch == 0) return FA_OK;
  int cus = 0;
  FA_TRY(current_compute_units(&cus));
  NormArgs n = {};
  const void* x[3] = {p->q, p->k, p->v};
  const int64_t* xs[3] = {p->q_stride, p->k_stride, p->v_stride};
  for (int i = 0; i < 3; ++i) {
    n.x[i] = static_cast<const char*>(x[i]);
    n.x_st[i] = 2 * xs[i][0];
    n.x_sh[i] = 2 * xs[i][1];
  }
  n.y[0] = static_cast<char*>(p->q_out);
  n.y_st[0] = 2 * p->q_out_stride[0];
  n.y_sh[0] = 2 * p->q_out_stride[1];
  void* y[2] = {c.k, c.v};
  const int64_t* ys[2] = {c.k_stride, c.v_stride};
  for (int i = 0; i < 2; ++i) {
    n.y[1 + i] = static_cast<char*>(y[i]);
    n.y_sb[1 + i] = 2 * ys[i][0];
    n.y_sh[1 + i] = 2 * ys[i][1];
    n.y_st[1 + i] = 2 * ys[i][2];
  }
  n.weight[0] = p->q_weight;
  n.weight[1] = p->k_weight;
  n.cos = p->cos;
  n.sin = p->sin;
  n.positions = p->positions;
  n.pt = page_table(c, p->tokens, c.max_pages * c.page_size);
  n.tokens = p->tokens;
  n.seq_len = p->tokens;
  n.heads = p->heads;
  n.kv_heads = c.kv_heads;
  n.head_dim = c.head_dim;
  n.rot = p->rot;
  n.table_rows = p->table_rows;
  n.interleaved = p->interleaved;
  n.weight_fp32 = p->weight_fp32;
  n.eps = p->eps;
  if (axes != nullptr) set_axes(n, *axes);
  n.by_seq = make_fast_div((uint32_t)p->tokens);
  return launched(launch_norm(n, c.dtype == FA_DTYPE_BF16, true, cus, static_cast<hipStream_t>(stream)));
}

}  // namespace

extern "C" {

fa_status fa_qk_norm_rope(const fa_qk_norm_params* p, void* stream) {
  FA_TRY(fa_qk_norm_rope_validate(p));
  return norm_forward(*p, nullptr, stream);
}

fa_status fa_qk_norm_rope_axes_validate(const fa_qk_norm_params* p, const fa_rotary_axes* axes) {
  FA_TRY(fa_qk_norm_rope_validate(p));
  return check_axes(axes, p->rot / 2, p->positions);
}

fa_status fa_qk_norm_rope_axes(const fa_qk_norm_params* p, const fa_rotary_axes* axes, void* stream) {
  FA_TRY(fa_qk_norm_rope_axes_validate(p, axes));
  return norm_forward(*p, axes, stream);
}

fa_status fa_qk_norm_rope_bwd_workspace_size(const fa_qk_norm_bwd_params* p, uint64_t* bytes) {
  if (bytes == nullptr) return fail(FA_ERR_NULL, "bytes is NULL");
  *bytes = 0;
  FA_TRY(fa_qk_norm_rope_bwd_validate(p));
  int cus = 0;
  FA_TRY(current_compute_units(&cus));
  *bytes = norm_bwd_bytes(p->fwd, cus);
  return FA_OK;
}

fa_status fa_qk_norm_rope_bwd(const fa_qk_norm_bwd_params* p, void* workspace, uint64_t workspace_bytes,
                              void* stream) {
  FA_TRY(fa_qk_norm_rope_bwd_validate(p));
  return norm_backward(p, nullptr, workspace, workspace_bytes, stream);
}

fa_status fa_qk_norm_rope_bwd_axes_validate(const fa_qk_norm_bwd_params* p, const fa_rotary_axes* axes) {
  FA_TRY(fa_qk_norm_rope_bwd_validate(p));
  return check_axes(axes, p->fwd.rot / 2, p->fwd.positions);
}

fa_status fa_qk_norm_rope_bwd_axes(const fa_qk_norm_bwd_params* p, const fa_rotary_axes* axes,
                                   void* workspace, uint64_t workspace_bytes, void* stream) {
  FA_TRY(fa_qk_norm_rope_bwd_axes_validate(p, axes));
  return norm_backward(p, axes, workspace, workspace_bytes, stream);
}

fa_status fa_paged_store(const fa_paged_store_params* p, void* stream) {
  FA_TRY(fa_paged_store_validate(p));
  return norm_store(p, nullptr, stream);
}

fa_status fa_paged_store_axes_validate(const fa_paged_store_params* p, const fa_rotary_axes* axes) {
  FA_TRY(fa_paged_store_validate(p));
  return p->tokens == 0 ? FA_OK : check_axes(axes, p->rot / 2, p->positions);
}

fa_status fa_paged_store_axes(const fa_paged_store_params* p, const fa_rotary_axes* axes, void* stream) {
  FA_TRY(fa_paged_store_axes_validate(p, axes));
  return norm_store(p, axes, stream);
}

}  // extern "C"
