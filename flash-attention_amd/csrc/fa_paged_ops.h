// Device building blocks shared by the kernels over a paged cache: sequences
// and page ids by scalar loads, staging of 16-key groups, LDS reads at
// addresses, explicit waits.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_cache_kernels.h"
#include "fa_device_ops.h"
#include "fa_lds_layout.h"

namespace fa {
namespace {

using namespace dev;


// 16 bytes of LDS at byte address addr + OFF.
template <int OFF>
__device__ __forceinline__ i16x8 lds_read16(uint32_t addr) {
  typedef __attribute__((address_space(3))) const char lds_char_t;
  return *(__attribute__((address_space(3))) const i16x8*)((lds_char_t*)(uintptr_t)addr + OFF);
}

// The debug build -DFA_LDS_POISON fills LDS bytes with NaN before every DMA into
// them, as fa_fwd_kernel.hip's: a read ahead of its wait or barrier shows, and
// with correct synchronisation every result keeps its bits.
#ifdef FA_LDS_POISON
constexpr bool kLdsPoison = true;
#else
constexpr bool kLdsPoison = false;
#endif
__device__ __forceinline__ void poison_1k(uint32_t addr) {
  if constexpr (kLdsPoison) {
    typedef __attribute__((address_space(3))) char lds_char_t;
    *(__attribute__((address_space(3))) u32x4*)((lds_char_t*)(uintptr_t)addr + (threadIdx.x & 63) * 16) =
        u32x4{~0u, ~0u, ~0u, ~0u};
    __builtin_amdgcn_s_waitcnt(0xc07f);
  }
}

// s_waitcnt vmcnt(N), the other counters left alone.
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt is 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70);
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// Ends this wave's LDS reads (lgkmcnt(0)) before what follows, a DMA into the
// bytes they read: no load moves past it.
__device__ __forceinline__ void fence_lds_reads() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_s_waitcnt(0xc07f);
  __builtin_amdgcn_sched_barrier(0);
}

// A scalar load of p[i]: i is the same in every lane, and no kernel writes p.
__device__ __forceinline__ int scalar_load(const int32_t* p, int64_t i) {
  return *(const __attribute__((address_space(4))) int32_t*)(uintptr_t)(p + i);
}

// Sequence b's new tokens and keys, within the limits of the call.
struct Seq {
  int q0;     // packed row of its first new token
  int nq;     // new tokens that are computed (at most max_q)
  int len;    // keys
  int first;  // key index of its first new token (negative: more tokens than keys)
};
__device__ __forceinline__ Seq load_seq(const PageTable& pt, int b, int max_q) {
  const int c0 = min(max(scalar_load(pt.cu, b), 0), pt.tokens);
  const int c1 = min(max(scalar_load(pt.cu, b + 1), c0), pt.tokens);
  Seq s;
  s.q0 = c0;
  s.nq = min(c1 - c0, max_q);
  s.len = min(max(scalar_load(pt.lens, b), 0), pt.max_kv);
  s.first = s.len - (c1 - c0);
  return s;
}

// Page id of key `key` (wave-uniform) in a sequence's table row.
__device__ __forceinline__ int page_id(const PageTable& pt, const int32_t* row, int key) {
  return scalar_load(row, key >> pt.page_shift);
}

// Page ids of 64 16-key groups, 1024 keys, a lane each, and of the 64 behind
// them, on their way.  Read lane by lane: scalar loads inside the tile loop
// would make every LDS wait there a wait for all (they share a counter and
// return out of order).  The ids of the table's row are loaded as far as the
// table may be read, whatever the sequence's length, so that their first load
// need not wait for the length; those past it are not used.
struct PageIds {
  const int32_t* row;
  int limit, shift, base;  // last key of the table; keys base .. base + 1023 are held
  uint32_t pages;
  int cur, next;
  uint64_t there;          // groups with a page
  __device__ __forceinline__ int load(int key0) const {
    return row[min(key0 + 16 * (int)(threadIdx.x & 63), limit) >> shift];
  }
  // Keys from key0, a multiple of 64 below pt.max_kv.
  __device__ __forceinline__ void start(const PageTable& pt, const int32_t* r, int key0) {
    row = r;
    limit = max(pt.max_kv - 1, 0);  // (a table has a page at least)
    shift = pt.page_shift;
    base = key0 - 1024;
    pages = (uint32_t)pt.num_pages;
    next = load(key0);
  }
  __device__ __forceinline__ void advance() {
    base += 1024;
    cur = next;
    there = __ballot((uint32_t)cur < pages);
    next = load(base + 1024);
  }
  // Makes `key` (uniform, ascending) held.
  __device__ __forceinline__ void reach(int key) {
    if (key >= base + 1024) advance();
  }
  // Page of the group of a held key, page 0 for an absent one.
  __device__ __forceinline__ int64_t page(int key) const {
    const int g = (key - base) >> 4;
    return (there >> g) & 1 ? __builtin_amdgcn_readlane(cur, g) : 0;
  }
  // Bit i: whether the i-th group from a held key has a page.
  __device__ __forceinline__ unsigned present(int key, unsigned mask) const {
    return (unsigned)(there >> ((key - base) >> 4)) & mask;
  }
};

// The same in either direction.
struct PageIdsBoth : PageIds {
  int step;  // 1024, or -1024
  __device__ __forceinline__ int load_at(int key0) const {
    return row[max(min(key0 + 16 * (int)(threadIdx.x & 63), limit), 0) >> shift];
  }
  // Of keys c0 .. c0 + 64 tiles - 1, tile by tile from the first, or `down` from the last.
  __device__ __forceinline__ void start(const PageTable& pt, const int32_t* r, int c0, int tiles, bool down) {
    row = r;
    limit = max(pt.max_kv - 1, 0);
    shift = pt.page_shift;
    step = down ? -1024 : 1024;
    const int key0 = down ? c0 + (tiles - 1) / 16 * 1024 : c0;
    base = key0 - step;
    pages = (uint32_t)pt.num_pages;
    next = load_at(key0);
  }
  __device__ __forceinline__ void reach(int key) {
    if ((uint32_t)(key - base) < 1024) return;
    base += step;
    cur = next;
    there = __ballot((uint32_t)cur < pages);
    next = load_at(base + step);
  }
};

// Row tiles of the chunk kernel, the longest first: sequence and tile of the
// n-th one, and how many there are.
//
// Up to 64 sequences: the ones with more keys first, each lane holding one
// sequence's tiles and the number of tiles before them.  More: in their order
// from the last, sequence b's tiles at place f(b) = floor(cu[b] group / BM) + b,
// which leaves room for the last, partial tile of each (places without a tile
// count as tiles); the sequence is then the number of b >= 1 with f(b) <= place,
// counted 64 at a time.
template <int BM>
struct TileList {
  int start, tiles, c0, c1, len;  // this lane's sequence (up to 64)
  int count;

  __device__ __forceinline__ void init(const PagedFwdArgs& a) {
    const int lane = threadIdx.x & 63;
    count = a.slots;
    if (a.pt.batch > 64) return;
    c0 = c1 = tiles = 0;
    len = -1;
    if (lane < a.pt.batch) {
      c0 = min(max(a.pt.cu[lane], 0), a.pt.tokens);
      c1 = min(max(a.pt.cu[lane + 1], c0), a.pt.tokens);
      const int rows = min(c1 - c0, a.max_q) * a.group;
      tiles = (rows + BM - 1) / BM;
      len = min(max(a.pt.lens[lane], 0), a.pt.max_kv);
    }
    start = count = 0;
    for (int i = 0; i < a.pt.batch; ++i) {
      const int l = __builtin_amdgcn_readlane(len, i), t = __builtin_amdgcn_readlane(tiles, i);
      start += l > len || (l == len && i < lane) ? t : 0;
      count += t;
    }
    count = listed_tiles(count, a.slots);
  }
  __device__ __forceinline__ bool find(const PagedFwdArgs& a, int n, int& b, int& tile, Seq& s) const {
    if (a.pt.batch <= 64) {
      const uint64_t has = __ballot(start <= n && n < start + tiles);
      if (has == 0) return false;
      b = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(has));
      tile = __builtin_amdgcn_readlane(start + tiles - 1, b) - n;
      const int nq = __builtin_amdgcn_readlane(c1 - c0, b);
      s.q0 = __builtin_amdgcn_readlane(c0, b);
      s.nq = min(nq, a.max_q);
      s.len = __builtin_amdgcn_readlane(len, b);
      s.first = s.len - nq;
      return true;
    }
    const int lane = threadIdx.x & 63, at = a.slots - 1 - n;
    auto begin = [&](int i, int cu) FA_INLINE {
      return (int)((uint32_t)(min(max(cu, 0), a.pt.tokens) * a.group) / BM) + i;
    };
    int k = 0;
    for (int i0 = 1; i0 <= a.pt.batch; i0 += 64) {
      const int i = i0 + lane;
      const bool before = i <= a.pt.batch && begin(i, a.pt.cu[min(i, a.pt.batch)]) <= at;
      k += __popcll(__ballot(before));
    }
    b = __builtin_amdgcn_readfirstlane(k);
    if (b >= a.pt.batch) return false;
    tile = at - begin(b, scalar_load(a.pt.cu, b));
    s = load_seq(a.pt, b, a.max_q);
    return tile >= 0;
  }
};

// The chunk kernel's last round.  `conc` workgroups of a kv head run at once;
// the tiles that are left after whole rounds of them would keep only some of
// the GPU busy for a whole tile's time, so they are cut into `pieces` of keys:
// the number that finishes them first, at ceil(rest pieces / conc) rounds of
// 1 / pieces of a tile plus a piece's own cost (its join, about the time of 768
// keys), as far as the workspace holds them.  Lane q weighs q + 1 pieces.
struct LastRound {
  int whole, rest, pieces;
  __device__ __forceinline__ void init(const PagedFwdArgs& a, int count) {
    const int rounds = fast_div(count, a.by_conc);
    whole = rounds * a.conc;
    rest = count - whole;
    const int q = (int)(threadIdx.x & 63) + 1;
    const int all = rest * q;
    const float cost = cut_cost(all, fast_div(all + a.conc - 1, a.by_conc), q, a.max_pieces, a.piece_cost);
    float least = cost;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) least = fminf(least, __shfl_xor(least, d));
    pieces = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(__ballot(cost == least)) + 1);
  }
};

// Keys of a piece of a tile that sees keys 0 .. kv_end - 1: whole 64-key
// tiles, 512 keys at least; and the number of pieces that have keys.
__device__ __forceinline__ int piece_keys(int kv_end, int pieces, int& used) {
  const int n = min(pieces, max(1, (kv_end + 511) / 512));
  const int keys = max(64, ((kv_end + n - 1) / n + 63) / 64 * 64);
  used = max(1, (kv_end + keys - 1) / keys);
  return keys;
}

// Staging of 16 consecutive keys of one page: their K rows and V rows to LDS
// in the layouts of the 16x16x32 kernels (lds::Tile16).  The swizzles go by
// key % 16, so one set of lane offsets serves every group.
template <int D>
struct GroupStage {
  static constexpr int ROWB = 2 * D, NI = 16 * ROWB / 1024;  // DMA instructions of K or V
  uint32_t k_src[NI], v_src[NI];
  int r_lane;  // row of this lane in the first instruction
  __device__ __forceinline__ void init(int lane, uint32_t k_ss, uint32_t v_ss) {
    constexpr int LPR = ROWB / 16;  // lanes of a row
    r_lane = lane / LPR;
#pragma unroll
    for (int it = 0; it < NI; ++it) {
      const int r = it * (64 / LPR) + r_lane, pc = lane % LPR;
      k_src[it] = r * k_ss + (pc ^ lds::Tile16<D>::swz_k(r)) * 16;
      v_src[it] = r * v_ss + (pc ^ lds::Tile16<D>::swz_v(r)) * 16;
    }
  }
  // kp, vp: the group's first rows; rows past `lim` re-read row lim.
  __device__ __forceinline__ void copy(const char* kp, const char* vp, uint32_t k_dst, uint32_t v_dst,
                                       int lim, uint32_t k_ss, uint32_t v_ss) const {
#pragma unroll
    for (int it = 0; kLdsPoison && it < NI; ++it) {
      poison_1k(k_dst + it * 1024);
      poison_1k(v_dst + it * 1024);
    }
    if (lim >= 15) {
#pragma unroll
      for (int it = 0; it < NI; ++it) dma_16b(k_src[it], kp, k_dst + it * 1024);
#pragma unroll
      for (int it = 0; it < NI; ++it) dma_16b(v_src[it], vp, v_dst + it * 1024);
    } else {
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        const int over = max(it * (1024 / ROWB) + r_lane - lim, 0);
        dma_16b(k_src[it] - over * k_ss, kp, k_dst + it * 1024);
        dma_16b(v_src[it] - over * v_ss, vp, v_dst + it * 1024);
      }
    }
  }
};

// The same for K alone.
template <int D>
struct KeyStage {
  static constexpr int ROWB = 2 * D, NI = 16 * ROWB / 1024;
  uint32_t src[NI];
  int r_lane;
  __device__ __forceinline__ void init(int lane, uint32_t k_ss) {
    constexpr int LPR = ROWB / 16;
    r_lane = lane / LPR;
#pragma unroll
    for (int it = 0; it < NI; ++it) {
      const int r = it * (64 / LPR) + r_lane;
      src[it] = r * k_ss + ((lane % LPR) ^ lds::Tile16<D>::swz_k(r)) * 16;
    }
  }
  __device__ __forceinline__ void copy(const char* kp, uint32_t dst, int lim, uint32_t k_ss) const {
#pragma unroll
    for (int it = 0; it < NI; ++it) {
      const int over = lim >= 15 ? 0 : max(it * (1024 / ROWB) + r_lane - lim, 0);
      poison_1k(dst + it * 1024);
      dma_16b(src[it] - over * k_ss, kp, dst + it * 1024);
    }
  }
};

}  // namespace
}  // namespace fa
