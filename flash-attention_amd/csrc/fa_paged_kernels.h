// Attention of new tokens over a paged key/value cache on gfx950.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i.k_j - m_i),
//   over the keys j that row i sees (causal: j <= L - n + token of i).
//
// One pass over the keys with a running offset m (lazily raised) and sum, fp32
// throughout; P is rounded to the input type for the matrix cores, and o is
// normalised by the sum of the rounded P, the weights it is made of; the
// logsumexp uses the unrounded sum.
//
// A workgroup's rows are tokens times the query heads of one kv head, so a
// key row that is read serves the whole group.  Two kernels:
//  * fa_paged_chunk_kernel: 128 rows, four waves of 32; K/V tiles of 64 keys
//    staged through a two-deep LDS ring by global_load_lds DMA, as
//    fa_fwd16_kernel.  Bound by the matrix cores and the exponentials.
//    4096 tokens over 16384 keys, 32 heads on 8, D = 128, bf16: causal 798 us,
//    1205 TFLOP/s of visible pairs; without the mask 903 us, 1218.  (A matrix
//    product of 8192^3 reaches 1370.)
//  * fa_paged_decode_kernel: at most 16 or 32 rows (a few tokens), the keys of a chunk
//    dealt to two or four waves in tiles of 32, each wave with an LDS ring of its
//    own and no barrier before the end.  Bound by reading the cache: 5.4 TB/s at
//    32 sequences of up to 8192 keys, 8 kv heads, D = 128 (144 us), where a
//    large copy moves 5.0.
// One of them serves a call (plan_paged).  Keys are split over workgroups where
// rows are few (plan_paged, LastRound); fa_paged_merge_kernel joins their
// normalised partials.
//
// Pages are read through their 16-key groups (a page holds whole groups), whose
// page ids a wave holds 64 at a time, one a lane (PageIds).
// Keys past the last visible one re-read that row, absent pages read page 0;
// the scores of both are masked.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "fa_cache_kernels.h"
#include "fa_device_ops.h"
#include "fa_lds_layout.h"
#include "fa_paged_ops.h"
#include "fa_wave_attn.h"

namespace fa {
namespace {

using namespace dev;

// Keys of the tokens' rows: the last key token i of a sequence sees, and the
// end of the keys that tokens up to i see.
template <bool SCORED>
__device__ __forceinline__ int last_key(const PagedFwdArgs& a, const Seq& s, int i) {
  if (SCORED && !a.causal && a.score.window > 0)
    return (int)min((int64_t)s.first + i + a.score.window - 1, (int64_t)s.len - 1);
  return a.causal ? min(s.first + i, s.len - 1) : s.len - 1;
}
// The first key that token i sees, and the tile that keys are read from.
template <bool SCORED>
__device__ __forceinline__ int first_key(const PagedFwdArgs& a, const Seq& s, int i) {
  return SCORED && a.score.window > 0 ? max(0, max(s.first + i, 0) - (a.score.window - 1)) : 0;
}
template <bool SCORED>
__device__ __forceinline__ int first_tile(const PagedFwdArgs& a, const Seq& s, int i) {
  return first_key<SCORED>(a, s, i) & ~63;
}

// What the scores of token i, head h go by.
template <class W>
__device__ __forceinline__ void set_row(const PagedFwdArgs& a, const Seq& s, int i, int h, W& w, int rb) {
  w.first[rb] = first_key<true>(a, s, i);
  w.pos[rb] = s.first + i;
  w.slope[rb] = a.score.slopes != nullptr ? a.score.slopes[h] * a.score.slope_unit : 0.0f;
}

// ---- few rows: decode ----

template <int D, bool BF16, int RB, int NW, bool SCORED>
__global__ void __launch_bounds__(64 * NW) fa_paged_decode_kernel(const PagedFwdArgs a) {
  using W = WaveAttn<D, BF16, 2, RB, SCORED>;
  constexpr int ROWB = 2 * D, TB = 32 * ROWB;   // bytes of a wave's K or V tile
  constexpr int NI = 16 * ROWB / 1024;          // DMA instructions of a 16-key group
  constexpr int BM = 16 * RB;
  __shared__ __attribute__((aligned(1024))) char smem[NW * 4 * TB];  // per wave K0 K1 V0 V1

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int bhs = a.slots * a.kv_heads;
  const int split = fast_div(blockIdx.x, a.by_splits);  // by_splits: by slots * kv heads
  const int bh = blockIdx.x - split * bhs;
  const int b = fast_div(bh, a.by_kvh), kvh = bh - b * a.kv_heads;
  PageIds ids;
  const bool windowed = SCORED && a.score.window > 0;
  if (!windowed) ids.start(a.pt, a.pt.table + b * a.pt.table_stride, split * a.chunk);
  const Seq s = load_seq(a.pt, b, a.max_q);
  const int n_rows = s.nq * a.group;
  if (n_rows <= 0) return;
  const int kv_end = max(0, last_key<SCORED>(a, s, s.nq - 1) + 1);
  const int kv0 = first_tile<SCORED>(a, s, 0);
  const int n_act = max(1, (kv_end - kv0 + a.chunk - 1) / a.chunk);
  if (split >= n_act) return;
  const int c0 = kv0 + split * a.chunk, c1 = min(kv_end, c0 + a.chunk);
  if (windowed) ids.start(a.pt, a.pt.table + b * a.pt.table_stride, c0);
  const int n_tiles = (c1 - c0 + 31) / 32;

  const uint32_t wave_lds = __builtin_amdgcn_readfirstlane(lds_addr(smem)) + wave * 4 * TB;
  W w;
  w.init(wave_lds, wave_lds + 2 * TB, a.scale_log2);
  if constexpr (SCORED) w.init_score(a.score);
  const int l16 = w.l16, g4 = w.g4;
  const int full_end = max(0, last_key<SCORED>(a, s, 0) + 1);  // every row sees the keys before it
  const int full_start = first_key<SCORED>(a, s, s.nq - 1);    // and from there on

  GroupStage<D> stage;
  stage.init(lane, a.k_ss, a.v_ss);
  const char* kbase = a.k + kvh * a.k_sh;
  const char* vbase = a.v + kvh * a.v_sh;
  const int last = c1 - 1;
  // Stages tile t; returns which of its two groups have a page.
  auto issue = [&](int t, int buf) FA_INLINE -> unsigned {
    const int key = c0 + 32 * t;
    ids.reach(key);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int r0 = min(key + 16 * g, last & ~15);
      const int64_t page = ids.page(r0);
      const int in_page = r0 & ((1 << a.pt.page_shift) - 1);
      const uint32_t dst = wave_lds + buf * TB + g * 16 * ROWB;
      stage.copy(kbase + page * a.k_sp + (int64_t)in_page * a.k_ss,
                 vbase + page * a.v_sp + (int64_t)in_page * a.v_ss, dst, dst + 2 * TB, last - r0,
                 a.k_ss, a.v_ss);
    }
    return ids.present(key, 3u);
  };
  unsigned present = 0, present_next = 0;
  if (wave < n_tiles) present = issue(wave, 0);
  // q behind the first tile's DMA: loads return in order, so a wait for all but
  // the next tile's DMA covers q too.
  const char* qh = a.q + s.q0 * a.q_st + (int64_t)kvh * a.group * a.q_sh;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = min(16 * rb + l16, n_rows - 1);
    const int i = fast_div(r, a.by_group), h = r - i * a.group;
    w.last[rb] = last_key<SCORED>(a, s, i);
    if constexpr (SCORED) set_row(a, s, i, kvh * a.group + h, w, rb);
#pragma unroll
    for (int st = 0; st < W::KST; ++st)
      w.qf[rb][st] = *reinterpret_cast<const i16x8*>(qh + i * a.q_st + h * a.q_sh + (32 * st + 8 * g4) * 2);
  }
  auto stage_next = [&](int t, int buf) FA_INLINE {
    if (t + NW < n_tiles) {
      present_next = issue(t + NW, buf ^ 1);
      wait_vmcnt<4 * NI>();
    } else {
      wait_vmcnt<0>();
    }
  };
  // (A chunk's end that is not the end of the keys is a multiple of 64, so no
  // tile reaches past it.)
  auto whole = [&](int t) FA_INLINE {
    return c0 + 32 * t + 32 <= full_end && (!SCORED || c0 + 32 * t >= full_start) && present == 3u;
  };
  if (wave < n_tiles) {
    // Whole tiles, then, from the first tile with a masked key on, the rest:
    // masked tiles are the last ones, or lie on absent pages.  (A window's are
    // the first ones too.)
    int t = wave, buf = 0;
    for (; SCORED && t < n_tiles && !whole(t) && c0 + 32 * t < full_start; t += NW, buf ^= 1) {
      stage_next(t, buf);
      w.template step<0, kMasked>(c0 + 32 * t, present, buf * TB, wave_lds + (2 + buf) * TB);
      present = present_next;
      fence_lds_reads();
    }
    for (; SCORED && t < n_tiles && whole(t); t += NW, buf ^= 1) {
      stage_next(t, buf);
      w.template step<0, kWhole>(c0 + 32 * t, present, buf * TB);
      present = present_next;
      fence_lds_reads();
    }
    for (; !SCORED && t < n_tiles && whole(t); t += NW) {
      stage_next(t, 0);
      w.template step<0, kWhole>(c0 + 32 * t, present, 0);
      present = present_next;
      fence_lds_reads();
      t += NW;
      buf = 1;
      if (t >= n_tiles || !whole(t)) break;
      stage_next(t, 1);
      w.template step<TB, kWhole>(c0 + 32 * t, present, 0);
      present = present_next;
      fence_lds_reads();
      buf = 0;
    }
    for (; t < n_tiles; t += NW, buf ^= 1) {
      stage_next(t, buf);
      w.template step<0, kMasked>(c0 + 32 * t, present, buf * TB, wave_lds + (2 + buf) * TB);
      present = present_next;
      fence_lds_reads();
    }
    if (__builtin_expect(w.odd, false)) {
      w.reset();
      ids.start(a.pt, a.pt.table + b * a.pt.table_stride, c0);
      present = issue(wave, 0);
      buf = 0;
      for (t = wave; t < n_tiles; t += NW, buf ^= 1) {
        stage_next(t, buf);
        w.template step<0, kSafe>(c0 + 32 * t, present, buf * TB);
        present = present_next;
        fence_lds_reads();
      }
    }
  }

  // ---- join the waves: o and sums at the largest offset ----
  constexpr int PITCH = D + 4;  // floats of a row in LDS: rows of 16 lanes on distinct banks
  float* ow = reinterpret_cast<float*>(smem);                 // [NW][BM][PITCH]
  float* mw = ow + NW * BM * PITCH;                           // [NW][BM][3]
  static_assert((BM * PITCH + BM * 3) * 4 <= 4 * TB, "join area");
  __syncthreads();
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = wave * BM + 16 * rb + l16;
#pragma unroll
    for (int db = 0; db < W::DB; ++db)
      *reinterpret_cast<f32x4*>(ow + r * PITCH + 16 * db + 4 * g4) = w.o[db][rb];
    const float lu = W::red_sum(w.lu[rb]);
    if (g4 == 0) {
      mw[r * 3] = w.m[rb];
      mw[r * 3 + 1] = w.ls[rb][0];
      mw[r * 3 + 2] = lu;
    }
  }
  __syncthreads();
  constexpr int TPR = D / 4;  // threads of a row
  const int d = ((int)threadIdx.x % TPR) * 4;
#pragma unroll
  for (int r = (int)threadIdx.x / TPR; r < BM; r += 64 * NW / TPR) {
    if (r >= n_rows) break;
    float mm = -INFINITY;
#pragma unroll
    for (int v = 0; v < NW; ++v) mm = fmaxf(mm, mw[(v * BM + r) * 3]);
    float lr = 0.0f, lu = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    const float base = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float* p = mw + (v * BM + r) * 3;
      // (a wave that saw no key: factor 0 of sums that are 0, or NaN)
      const float f = fast_exp2((p[0] - base) * w.c);
      lr += f * p[1];
      lu += f * p[2];
      acc += f * *reinterpret_cast<const f32x4*>(ow + (v * BM + r) * PITCH + d);
    }
    const bool none = lr == 0.0f;
    const float inv = none ? 0.0f : 1.0f / lr;
    acc *= inv;
    if (n_act == 1) {
      const int i = fast_div(r, a.by_group), h = kvh * a.group + r - i * a.group;
      const int64_t t = s.q0 + i;
      *reinterpret_cast<u32x2*>(a.o + t * a.o_st + h * a.o_sh + d * 2) =
          u32x2{pack2<BF16>(acc[0], acc[1]), pack2<BF16>(acc[2], acc[3])};
      if (a.lse != nullptr && d == 0)
        a.lse[t * a.heads + h] = none ? -INFINITY : w.log2_sum(mm, lu) * kLn2;
    } else {
      const int64_t wr = (((int64_t)b * a.kv_heads + kvh) * a.splits + split) * BM + r;
      *reinterpret_cast<f32x4*>(a.ws_o + wr * D + d) = acc;
      if (d == 0) {
        a.ws_e[wr * 2] = none ? -INFINITY : w.log2_sum(mm, lr);
        a.ws_e[wr * 2 + 1] = none ? -INFINITY : w.log2_sum(mm, lu);
      }
    }
  }
}

// ---- many rows: chunks ----

// Kv head and place (in its list of tiles and pieces) of a workgroup.
// Workgroup w runs on XCD w % 8, in order; the tiles of a head share its keys
// through the XCD's L2, and the longest tiles of all heads should start first:
//  * a multiple of 8 heads: whole heads per XCD, up to four of them interleaved;
//  * 1, 2 or 4: 8 / heads XCDs take turns with a head's places;
//  * else all heads interleaved over all XCDs.
// Workgroups k and k + 32 of an XCD, with its 32 CUs, share a CU.  `turn`, where
// there are so many: the first 32 run backwards, so that the longest of them has
// the shortest neighbour (us without and with: prompts of 4096 and 8192 tokens, 8
// heads on 2, D = 128: 62 and 60, 180 and 167; 2048 tokens, 32 on 8: 57 and 55).
__device__ __forceinline__ bool head_and_place(const PagedFwdArgs& a, bool turn, int& kvh, int& place) {
  const int xcd = blockIdx.x % kNumXcd;
  int i = blockIdx.x / kNumXcd;
  if (turn && i < a.xcd_cus) i = a.xcd_cus - 1 - i;
  if (a.per_xcd > 0) {
    const int grp = fast_div(i, a.by_group_places), w = i - grp * a.unit_group * a.places;
    place = fast_div(w, a.by_unit_group);
    kvh = xcd * a.per_xcd + grp * a.unit_group + (w - place * a.unit_group);
  } else if (a.xcds > 0) {
    kvh = xcd / a.xcds;
    place = i * a.xcds + xcd % a.xcds;
  } else {
    place = fast_div(i * kNumXcd + xcd, a.by_kvh);
    kvh = i * kNumXcd + xcd - place * a.kv_heads;
  }
  return place < a.places;
}

template <int D, bool BF16, bool SCORED>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
    fa_paged_chunk_kernel(const PagedFwdArgs a) {
  using W = WaveAttn<D, BF16, 4, 2, SCORED>;
  constexpr int ROWB = 2 * D, TB = 64 * ROWB, BM = kChunkRows;
  constexpr int DB = D / 16;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB];  // K0 K1 V0 V1
  __shared__ int again;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (threadIdx.x == 0) again = 0;  // ordered by the first barrier
  int kvh, place, b, tile0;
  TileList<BM> list;
  list.init(a);
  LastRound end;
  end.init(a, list.count);
  // (lists of more than 64 sequences are not by length)
  const bool turn = a.pt.batch <= 64 && (end.whole + end.rest * end.pieces) * a.kv_heads > kNumXcd * a.xcd_cus;
  if (!head_and_place(a, turn, kvh, place)) return;
  int pieces = 1, piece = 0, nth = place;
  if (place >= end.whole) {
    pieces = end.pieces;
    // (First pieces of all tiles, second ones, ...: short tiles have no last ones,
    // and gaps leave CUs idle.  128 tokens over 2000 keys, 32 heads on 8: 31 -> 27 us.)
    const int i = place - end.whole;
    if (i >= end.rest * pieces) return;
    piece = i / end.rest;
    nth = i - piece * end.rest + end.whole;
  }
  Seq s;
  if (!list.find(a, nth, b, tile0, s)) return;
  const int n_rows = s.nq * a.group, row0 = tile0 * BM;
  if (row0 >= n_rows) return;
  const int last_row = min(row0 + BM, n_rows) - 1;
  const int kv_end = max(0, last_key<SCORED>(a, s, fast_div(last_row, a.by_group)) + 1);
  const int kv0 = first_tile<SCORED>(a, s, fast_div(row0, a.by_group));
  int n_act = 1, c0 = kv0, c1 = kv_end;
  if (pieces > 1) {
    const int keys = piece_keys(kv_end - kv0, pieces, n_act);
    if (piece >= n_act) return;
    c0 = kv0 + piece * keys;
    c1 = min(kv_end, c0 + keys);
  }
  const int n_tiles = (c1 - c0 + 63) / 64;

  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(smem));
  W w;
  w.init(base, base + 2 * TB, a.scale_log2);
  if constexpr (SCORED) w.init_score(a.score);
  const int l16 = w.l16, g4 = w.g4;
  const int wrow0 = row0 + 32 * wave;

  GroupStage<D> stage;
  stage.init(lane, a.k_ss, a.v_ss);
  const char* kbase = a.k + kvh * a.k_sh;
  const char* vbase = a.v + kvh * a.v_sh;
  const int last = c1 - 1;
  // With a bias by distance from the last tile to the first: a causal row's scores
  // grow towards it, and the first of them would be raised over tile by tile (4096 tokens
  // over 16384 keys, 32 heads on 8, D = 128, bf16, us: 1280 and 868).
  const bool down = SCORED && w.score.biased;
  auto key_of = [&](int t) FA_INLINE { return c0 + 64 * (down ? n_tiles - 1 - t : t); };
  std::conditional_t<SCORED, PageIdsBoth, PageIds> ids;
  auto start_ids = [&]() FA_INLINE {
    const int32_t* row = a.pt.table + b * a.pt.table_stride;
    if constexpr (SCORED)
      ids.start(a.pt, row, c0, n_tiles, down);
    else
      ids.start(a.pt, row, c0);
  };
  // Stages this wave's 16-key group of tile t; returns which of the tile's four
  // groups have a page.
  auto issue = [&](int t, int buf) FA_INLINE -> unsigned {
    const int key = key_of(t);
    ids.reach(key);
    const int r0 = min(key + 16 * wave, last & ~15);
    const int64_t page = ids.page(r0);
    const int in_page = r0 & ((1 << a.pt.page_shift) - 1);
    const uint32_t dst = base + buf * TB + wave * 16 * ROWB;
    stage.copy(kbase + page * a.k_sp + (int64_t)in_page * a.k_ss,
               vbase + page * a.v_sp + (int64_t)in_page * a.v_ss, dst, dst + 2 * TB, last - r0,
               a.k_ss, a.v_ss);
    return ids.present(key, 15u);
  };
  unsigned present = 0, present_next = 0;
  if (n_tiles > 0) {
    start_ids();
    present = issue(0, 0);
  }
  const char* qh = a.q + s.q0 * a.q_st + (int64_t)kvh * a.group * a.q_sh;
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const int r = min(wrow0 + 16 * rb + l16, n_rows - 1);
    const int i = fast_div(r, a.by_group), h = r - i * a.group;
    w.last[rb] = last_key<SCORED>(a, s, i);
    if constexpr (SCORED) set_row(a, s, i, kvh * a.group + h, w, rb);
#pragma unroll
    for (int st = 0; st < W::KST; ++st)
      w.qf[rb][st] = *reinterpret_cast<const i16x8*>(qh + i * a.q_st + h * a.q_sh + (32 * st + 8 * g4) * 2);
  }
  // Keys that every row of the wave sees, and that some row sees.
  const bool rows = wrow0 < n_rows;
  const int full_end = rows ? last_key<SCORED>(a, s, fast_div(wrow0, a.by_group)) + 1 : 0;
  const int wave_end =
      rows ? last_key<SCORED>(a, s, fast_div(min(wrow0 + 31, n_rows - 1), a.by_group)) + 1 : 0;
  const int last_i = rows ? fast_div(min(wrow0 + 31, n_rows - 1), a.by_group) : 0;
  const int full_start = rows ? first_key<SCORED>(a, s, last_i) : 0;
  const int wave_start = rows ? first_key<SCORED>(a, s, fast_div(wrow0, a.by_group)) : 0;
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();

  auto stage_next = [&](int t, int buf) FA_INLINE {
    if (t + 1 < n_tiles) present_next = issue(t + 1, buf ^ 1);
  };
  auto end_tile = [&]() FA_INLINE {
    present = present_next;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };
  // Whole tiles, then, from the wave's first tile with a masked key on, the
  // rest: masked tiles are the last ones, or lie on absent pages.  Every wave
  // passes one barrier per tile, whichever loop it is in.
  auto whole = [&](int t) FA_INLINE {
    return key_of(t) + 64 <= full_end && (!SCORED || key_of(t) >= full_start) && present == 15u;
  };
  int t = 0, buf = 0;
  // (a window's masked tiles are the first ones too)
  auto before_whole = [&](int t) FA_INLINE { return down ? key_of(t) + 64 > full_end : key_of(t) < full_start; };
  auto seen = [&](int t) FA_INLINE { return key_of(t) < wave_end && (!SCORED || key_of(t) + 64 > wave_start); };
  for (; SCORED && t < n_tiles && !whole(t) && before_whole(t); ++t, buf ^= 1) {
    stage_next(t, buf);
    if (seen(t)) w.template step<0, kMasked>(key_of(t), present, buf * TB, base + (2 + buf) * TB);
    end_tile();
  }
  for (; SCORED && t < n_tiles && whole(t); ++t, buf ^= 1) {
    stage_next(t, buf);
    w.template step<0, kWhole>(key_of(t), present, buf * TB);
    end_tile();
  }
  for (; !SCORED && t < n_tiles && whole(t); ++t) {
    stage_next(t, 0);
    w.template step<0, kWhole>(c0 + 64 * t, present, 0);
    end_tile();
    ++t;
    buf = 1;
    if (t >= n_tiles || !whole(t)) break;
    stage_next(t, 1);
    w.template step<TB, kWhole>(c0 + 64 * t, present, 0);
    end_tile();
    buf = 0;
  }
  for (; t < n_tiles; ++t, buf ^= 1) {
    stage_next(t, buf);
    if (seen(t)) w.template step<0, kMasked>(key_of(t), present, buf * TB, base + (2 + buf) * TB);
    end_tile();
  }
  // Infinities or NaN in a masked tile of some wave: all start again (the
  // staging is shared).
  if (w.odd && lane == 0) again = 1;
  __syncthreads();
  if (__builtin_expect(__builtin_amdgcn_readfirstlane(again) != 0, false)) {
    w.reset();
    start_ids();
    present = issue(0, 0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    buf = 0;
    for (t = 0; t < n_tiles; ++t, buf ^= 1) {
      stage_next(t, buf);
      if (seen(t)) w.template step<0, kSafe>(key_of(t), present, buf * TB);
      end_tile();
    }
  }

  float inv[2], lu[2];
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    inv[rb] = w.ls[rb][0] == 0.0f ? 0.0f : 1.0f / w.ls[rb][0];
    lu[rb] = W::red_sum(w.lu[rb]);
  }
  if (n_act > 1) {  // partials: o normalised, sums as log2
    const int64_t wr0 = partial_tile(kvh, a.max_pieces, nth - end.whole, pieces, piece) * BM + 32 * wave;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const int r = 16 * rb + l16;
      if (wrow0 + r >= n_rows) continue;
#pragma unroll
      for (int db = 0; db < DB; ++db)
        *reinterpret_cast<f32x4*>(a.ws_o + (wr0 + r) * D + 16 * db + 4 * g4) = w.o[db][rb] * inv[rb];
      if (g4 == 0) {
        const bool none = w.ls[rb][0] == 0.0f;
        a.ws_e[(wr0 + r) * 2] = none ? -INFINITY : w.log2_sum(w.m[rb], w.ls[rb][0]);
        a.ws_e[(wr0 + r) * 2 + 1] = none ? -INFINITY : w.log2_sum(w.m[rb], lu[rb]);
      }
    }
    return;
  }
  // (the ring is idle)
  write_rows<D, BF16>(smem + wave * 32 * ROWB, w.o, inv, lane, [&](int r) FA_INLINE -> char* {
    if (wrow0 + r >= n_rows) return nullptr;
    const int i = fast_div(wrow0 + r, a.by_group), h = kvh * a.group + wrow0 + r - i * a.group;
    return a.o + (int64_t)(s.q0 + i) * a.o_st + h * a.o_sh;
  });
  if (a.lse != nullptr && g4 < 2) {
    const int r = wrow0 + 16 * g4 + l16;
    // (selects: an index by lane would put the whole state into scratch)
    const float m = g4 == 0 ? w.m[0] : w.m[1], sum = g4 == 0 ? w.ls[0][0] : w.ls[1][0];
    const float l = g4 == 0 ? lu[0] : lu[1];
    if (r < n_rows) {
      const int i = fast_div(r, a.by_group), h = kvh * a.group + r - i * a.group;
      a.lse[(int64_t)(s.q0 + i) * a.heads + h] =
          sum == 0.0f ? -INFINITY : w.log2_sum(m, l) * kLn2;
    }
  }
}

// Joins the partials of split rows: weights 2^(e - max e) of normalised
// partials.  BM: rows of a slot; a decode slot is a sequence.  a.join groups of
// D / 4 lanes share a row, each with every join-th chunk, four in flight, and
// meet in LDS: one group per row left 128 chunks to a loop of dependent loads
// (125 us against 98 for the attention itself at one sequence of 131072 keys).
template <int D, bool BF16, int BM, bool SCORED>
__global__ void __launch_bounds__(256) fa_paged_merge_kernel(const PagedFwdArgs a) {
  const int block = blockIdx.x;
  constexpr int TPR = D / 4, GROUPS = 256 / TPR;
  __shared__ f32x4 part_o[GROUPS][TPR];
  __shared__ float part_e[GROUPS][4];  // top, sum of weights; the same of the plain sums
  const int grp = (int)threadIdx.x / TPR, lane = (int)threadIdx.x % TPR, d = lane * 4;
  constexpr bool kTiles = BM == kChunkRows;
  // Rows of a workgroup: of a tile (join 1) merge_rows, one after another.
  const int rpb = kTiles ? a.merge_rows : GROUPS / a.join;
  const int per = ((kTiles ? BM : a.most_rows) + rpb - 1) / rpb;
  const int sk = block / per, r_first = (block - sk * per) * rpb + grp / a.join;
  const int slot = fast_div(sk, a.by_kvh), kvh = sk - slot * a.kv_heads;
  int b = slot, tile0 = 0, n_act;
  int64_t w0;  // first partial row
  Seq s;
  if constexpr (kTiles) {  // slot: the slot-th tile of the last round
    TileList<BM> list;
    list.init(a);
    LastRound end;
    end.init(a, list.count);
    if (end.pieces <= 1 || slot >= end.rest || !list.find(a, end.whole + slot, b, tile0, s)) return;
    w0 = partial_tile(kvh, a.max_pieces, slot, end.pieces, 0) * BM;
    n_act = end.pieces;
  } else {
    s = load_seq(a.pt, b, a.max_q);
    w0 = (int64_t)sk * a.splits * BM;
    n_act = 0;
  }
  const int n_rows = s.nq * a.group, row0 = tile0 * BM;
  if (row0 >= n_rows) return;
  const int last_row = min(row0 + BM, n_rows) - 1;
  const int kv_end = max(0, last_key<SCORED>(a, s, fast_div(last_row, a.by_group)) + 1);
  const int keys = kv_end - first_tile<SCORED>(a, s, fast_div(row0, a.by_group));
  if constexpr (kTiles)
    piece_keys(keys, n_act, n_act);
  else
    n_act = (keys + a.chunk - 1) / a.chunk;
  if (n_act <= 1) return;
  for (int r0 = 0; r0 < (kTiles ? rpb : 1); r0 += GROUPS) {
    const int r = r_first + r0;
    const bool row = r < BM && row0 + r < n_rows;
    float top = -INFINITY, top_u = -INFINITY, lr = 0.0f, lu = 0.0f;
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row) {
      constexpr int BATCH = 4;
      for (int c = grp & (a.join - 1); c < n_act; c += BATCH * a.join) {
        float e[BATCH], eu[BATCH];
        f32x4 o[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          const int64_t wr = w0 + r + (int64_t)min(c + j * a.join, n_act - 1) * BM;
          e[j] = a.ws_e[wr * 2];
          eu[j] = a.ws_e[wr * 2 + 1];
          o[j] = *reinterpret_cast<const f32x4*>(a.ws_o + wr * D + d);
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          // (e = -inf: its keys are all masked for this row)
          if (c + j * a.join >= n_act || e[j] == -INFINITY) continue;
          const float t = fmaxf(top, e[j]), tu = fmaxf(top_u, eu[j]);
          const float old = fast_exp2(top - t), f = fast_exp2(e[j] - t);
          lr = lr * old + f;
          acc = acc * old + o[j] * f;
          lu = lu * fast_exp2(top_u - tu) + fast_exp2(eu[j] - tu);
          top = t;
          top_u = tu;
        }
      }
    }
    if (a.join > 1) {
      part_o[grp][lane] = acc;
      if (lane == 0) {
        part_e[grp][0] = top;
        part_e[grp][1] = lr;
        part_e[grp][2] = top_u;
        part_e[grp][3] = lu;
      }
      __syncthreads();
      if ((grp & (a.join - 1)) != 0) return;
      for (int g = 0; g < a.join; ++g) {
        top = fmaxf(top, part_e[grp + g][0]);
        top_u = fmaxf(top_u, part_e[grp + g][2]);
      }
      lr = lu = 0.0f;
      acc = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      for (int g = 0; g < a.join; ++g) {
        if (part_e[grp + g][1] == 0.0f) continue;  // no chunk with a visible key
        const float f = fast_exp2(part_e[grp + g][0] - top);
        lr += f * part_e[grp + g][1];
        lu += fast_exp2(part_e[grp + g][2] - top_u) * part_e[grp + g][3];
        acc += part_o[grp + g][lane] * f;
      }
    }
    if (!row) continue;
    const bool none = lr == 0.0f;
    const float inv = none ? 0.0f : 1.0f / lr;
    const int i = fast_div(row0 + r, a.by_group), h = kvh * a.group + row0 + r - i * a.group;
    const int64_t t = s.q0 + i;
    *reinterpret_cast<u32x2*>(a.o + t * a.o_st + h * a.o_sh + d * 2) =
        u32x2{pack2<BF16>(acc[0] * inv, acc[1] * inv), pack2<BF16>(acc[2] * inv, acc[3] * inv)};
    if (a.lse != nullptr && lane == 0)
      a.lse[t * a.heads + h] = none ? -INFINITY : (top_u + __log2f(lu)) * kLn2;
  }
}

template <class F>
hipError_t launch(F* fn, int64_t grid, const PagedFwdArgs& args, hipStream_t stream, int threads = 256) {
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  void* kargs[] = {const_cast<PagedFwdArgs*>(&args)};
  return hipLaunchKernel(reinterpret_cast<const void*>(fn), dim3((unsigned)grid), dim3(threads), kargs,
                         0, stream);
}

// The chunk kernel's grid order (head_and_place) and its workgroups.
int64_t set_order(PagedFwdArgs& a, const PagedPlan& plan) {
  a.per_xcd = a.kv_heads % kNumXcd == 0 ? a.kv_heads / kNumXcd : 0;
  a.unit_group = 1;
  for (int g = 2; g <= 4; ++g)
    if (a.per_xcd % g == 0) a.unit_group = g;
  a.xcd_cus = plan.compute_units / kNumXcd;
  a.xcds = a.per_xcd == 0 && kNumXcd % a.kv_heads == 0 ? kNumXcd / a.kv_heads : 0;
  a.by_group_places = make_fast_div((uint32_t)(a.unit_group * a.places));
  a.by_unit_group = make_fast_div((uint32_t)a.unit_group);
  if (a.xcds > 0) return (int64_t)kNumXcd * ((a.places + a.xcds - 1) / a.xcds);
  return (int64_t)a.kv_heads * a.places;
}

template <int D, bool BF16, bool SCORED>
hipError_t launch_all(const PagedFwdArgs& base, const PagedPlan& plan, void* ws, hipStream_t stream) {
  const PagedGrid& g = plan.grid;
  PagedFwdArgs a = base;
  a.slots = g.slots;
  a.ws_o = g.ws_rows ? static_cast<float*>(ws) : nullptr;
  a.ws_e = g.ws_rows ? a.ws_o + g.ws_rows * D : nullptr;
  a.join = 1;
  constexpr int GROUPS = 256 / (D / 4);  // lane groups of a merge workgroup
  if (g.rows == kChunkRows) {
    a.conc = g.conc;
    a.max_pieces = g.pieces;
    a.by_conc = make_fast_div((uint32_t)g.conc);
    a.piece_cost = piece_cost(g.keys);
    a.places = g.slots + g.pieces;
    const hipError_t e = launch(&fa_paged_chunk_kernel<D, BF16, SCORED>, set_order(a, plan), a, stream);
    if (e != hipSuccess || g.pieces == 0) return e;
    const int64_t tiles = (int64_t)std::min(g.conc - 1, g.slots) * a.kv_heads;
    // Rows of a workgroup: few, unless that makes thousands of workgroups,
    // most of which find no tile.
    a.merge_rows = tiles * (kChunkRows / GROUPS) <= 2048 ? GROUPS : 32;
    return launch(&fa_paged_merge_kernel<D, BF16, kChunkRows, SCORED>, tiles * (kChunkRows / a.merge_rows), a,
                  stream);
  }
  a.splits = g.splits;
  a.chunk = g.chunk;
  const int64_t sk = (int64_t)g.slots * a.kv_heads;
  a.by_splits = make_fast_div((uint32_t)sk);
  // Two waves a workgroup where two workgroups per CU are there to take
  // turns at starting and ending (us, 4 waves -> 2: 32 sequences of 4096 keys,
  // 8 kv heads, D = 128: 105 -> 102; 64 of 1000: 55 -> 50); with fewer, four
  // waves read sooner (4 sequences of 2000: 17 -> 14).
  auto decode = [&](auto rb_c) {
    constexpr int RB = decltype(rb_c)::value;
    return sk * g.splits >= 2 * plan.compute_units
               ? launch(&fa_paged_decode_kernel<D, BF16, RB, 2, SCORED>, sk * g.splits, a, stream, 128)
               : launch(&fa_paged_decode_kernel<D, BF16, RB, 4, SCORED>, sk * g.splits, a, stream, 256);
  };
  const hipError_t e = g.rows == 16 ? decode(std::integral_constant<int, 1>{})
                                    : decode(std::integral_constant<int, 2>{});
  if (e != hipSuccess || g.splits == 1) return e;
  // As many lane groups a row as it has chunks, a power of two.
  while (a.join < g.splits && a.join < GROUPS) a.join *= 2;
  const int rpb = GROUPS / a.join;
  a.most_rows = std::min<int64_t>(g.rows, (int64_t)a.max_q * a.group);
  const int64_t blocks = sk * ((a.most_rows + rpb - 1) / rpb);
  return g.rows == 16 ? launch(&fa_paged_merge_kernel<D, BF16, 16, SCORED>, blocks, a, stream)
                      : launch(&fa_paged_merge_kernel<D, BF16, 32, SCORED>, blocks, a, stream);
}

template <bool SCORED>
hipError_t launch_as(const PagedFwdArgs& args, const PagedPlan& plan, int head_dim, bool bf16, void* workspace,
                     hipStream_t stream) {
  if (head_dim == 128)
    return bf16 ? launch_all<128, true, SCORED>(args, plan, workspace, stream)
                : launch_all<128, false, SCORED>(args, plan, workspace, stream);
  return bf16 ? launch_all<64, true, SCORED>(args, plan, workspace, stream)
              : launch_all<64, false, SCORED>(args, plan, workspace, stream);
}

}  // namespace
}  // namespace fa
