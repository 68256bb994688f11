// Device building blocks shared by the kernels of attention on whole tensors:
// the keys that a row sees, staging of rows, cleaning of masked rows.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_attention_kernels.h"
#include "fa_device_ops.h"
#include "fa_lds_layout.h"
#include "fa_paged_ops.h"

namespace fa {
namespace {

using namespace dev;

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Keys lo .. hi - 1; a row that sees none has lo = kNoKey, hi = 0.
constexpr int kNoKey = 0x7fffffff;
struct RowKeys {
  int lo, hi;
};
// (hi at or below lo: none)
__device__ __forceinline__ RowKeys limits(const AttnArgs& a, int i, RowKeys k) {
  const int p = i + a.m - a.n;
  if (a.causal) k.hi = min(k.hi, p + 1);
  if (a.score.window > 0) {
    k.lo = max(k.lo, p - (a.score.window - 1));
    if (!a.causal) k.hi = min(k.hi, p + a.score.window);
  }
  return k;
}
__device__ __forceinline__ RowKeys limits(const AttnArgs& a, int i) { return limits(a, i, {0, a.m}); }
__device__ __forceinline__ RowKeys row_keys(const AttnArgs& a, int b, int i) {
  RowKeys k = {0, a.m};
  if (a.ranges != nullptr) {
    const int2 r = *reinterpret_cast<const int2*>(a.ranges + b * a.range_sb + 2 * (int64_t)i);
    k.lo = max(r.x, 0);
    k.hi = min(r.y, a.m);
  }
  k = limits(a, i, k);
  if (k.lo >= k.hi) k = {kNoKey, 0};
  return k;
}

// Keys that some row sees, and that every row sees.
struct TileKeys {
  int lo, hi, all_lo, all_hi;
  __device__ __forceinline__ void start(const RowKeys& k) { *this = {k.lo, k.hi, k.lo, k.hi}; }
  __device__ __forceinline__ void add(const TileKeys& o) {
    lo = min(lo, o.lo);
    hi = max(hi, o.hi);
    all_lo = max(all_lo, o.all_lo);
    all_hi = min(all_hi, o.all_hi);
  }
  template <int WIDTH>
  __device__ __forceinline__ void reduce() {  // over aligned groups of WIDTH lanes
#pragma unroll
    for (int d = 1; d < WIDTH; d <<= 1)
      add({__shfl_xor(lo, d), __shfl_xor(hi, d), __shfl_xor(all_lo, d), __shfl_xor(all_hi, d)});
  }
  __device__ __forceinline__ TileKeys of_lane(int l) const {
    return {__builtin_amdgcn_readlane(lo, l), __builtin_amdgcn_readlane(hi, l), __builtin_amdgcn_readlane(all_lo, l),
            __builtin_amdgcn_readlane(all_hi, l)};
  }
};

// Those of the rows from one with the limits x to one with y.  Without ranges no
// row sees keys before an earlier row's first, nor past a later row's last; rows without
// any come first, and end at or before key 0.
__device__ __forceinline__ TileKeys between(const RowKeys& x, const RowKeys& y) {
  return {x.lo, max(y.hi, 0), y.lo, x.hi};
}

// Those of the 128 rows from row0 on, `all`, and of the 32 of a wave, `own`.
__device__ __forceinline__ void tile_keys(const AttnArgs& a, int b, int row0, int wave, TileKeys& own, TileKeys& all) {
  const int lane = threadIdx.x & 63, end = a.n - 1;
  TileKeys s, t;  // of the first 64 rows, of the others; lanes below 32 and from 32 on
  if (a.ranges != nullptr) {
    s.start(row_keys(a, b, min(row0 + lane, end)));
    t.start(row_keys(a, b, min(row0 + 64 + lane, end)));
    s.reduce<32>();
    t.reduce<32>();
  } else {
    const int i = row0 + (lane & 32);
    s = between(limits(a, min(i, end)), limits(a, min(i + 31, end)));
    t = between(limits(a, min(i + 64, end)), limits(a, min(i + 95, end)));
  }
  all = s.of_lane(0);
  all.add(s.of_lane(32));
  all.add(t.of_lane(0));
  all.add(t.of_lane(32));
  const int at = wave % 2 * 32;
  s = {wave < 2 ? s.lo : t.lo, wave < 2 ? s.hi : t.hi, wave < 2 ? s.all_lo : t.all_lo, wave < 2 ? s.all_hi : t.all_hi};
  own = s.of_lane(at);
}

// Unit and place of a workgroup; false: none.  Workgroup w runs on XCD w % 8, in
// order; the workgroups of a unit share its keys (or rows) through the XCD's L2, and the
// longest ones of all units should start first:
//  * a multiple of 8 units: whole units per XCD, as many of them interleaved as fill
//    it;
//  * 1, 2 or 4: 8 / units XCDs take turns with a unit's places;
//  * else all units interleaved over all XCDs.
// Workgroups k and k + xcd_cus of an XCD share a CU: `turn`, the first xcd_cus run
// backwards, so that the longest of them has the shortest neighbour.
__device__ __forceinline__ bool unit_and_place(const GridOrder& o, int& unit, int& place) {
  const int xcd = blockIdx.x % kNumXcd;
  int i = blockIdx.x / kNumXcd;
  if (o.turn && i < o.xcd_cus) i = o.xcd_cus - 1 - i;
  if (o.per_xcd > 0) {
    const int grp = fast_div(i, o.by_group_places), w = i - grp * o.unit_group * o.places;
    place = fast_div(w, o.by_unit_group);
    unit = xcd * o.per_xcd + grp * o.unit_group + (w - place * o.unit_group);
  } else if (o.xcds > 0) {
    unit = xcd / o.xcds;
    place = i * o.xcds + xcd % o.xcds;
  } else {
    place = fast_div(i * kNumXcd + xcd, o.by_units);
    unit = i * kNumXcd + xcd - place * o.units;
  }
  return place < o.places;
}

// The lane, computed anew: a register less along the loop.
__device__ __forceinline__ int lane_now() {
  int l;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(l));
  return l;
}

// x of lane l.  (__shfl_xor keeps the lane in a register.)
__device__ __forceinline__ float from_lane(float x, int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * l, __builtin_bit_cast(int, x)));
}

// x of the lane that is N ahead in the same 16 (DPP row_ror), around their end.
template <int N>
__device__ __forceinline__ float turned_row(float x) {
  const int w = __builtin_bit_cast(int, x);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(w, w, 0x120 + N, 0xf, 0xf, false));
}

// Staging of 16 rows of a tensor into LDS in the layout of lds::TileBoth.
template <int D>
struct RowStage {
  static constexpr int ROWB = 2 * D, NI = 16 * ROWB / 1024, LPR = ROWB / 16;
  uint32_t src[NI];
  __device__ __forceinline__ void init(int lane, uint32_t st) {
#pragma unroll
    for (int it = 0; it < NI; ++it) {
      const int r = it * (64 / LPR) + lane / LPR;
      src[it] = r * st + ((lane % LPR) ^ lds::TileBoth<D>::swz(r)) * 16;
    }
  }
  // p: the first row; rows past `lim` re-read row lim.
  __device__ __forceinline__ void copy(const char* p, uint32_t dst, int lim, uint32_t st) const {
#pragma unroll
    for (int it = 0; it < NI; ++it) {
      poison_1k(dst + it * 1024);
      const int r = it * (64 / LPR) + (int)(threadIdx.x & 63) / LPR;
      const uint32_t over = lim >= 15 ? 0u : (uint32_t)max(r - lim, 0);
      dma_16b(src[it] - over * st, p, dst + it * 1024);
    }
  }
};

template <int OFF>
__device__ __forceinline__ u32x2 lds_read8(uint32_t addr) {
  return *(__attribute__((address_space(3))) const u32x2*)(uintptr_t)(addr + OFF);
}
template <int OFF>
__device__ __forceinline__ void lds_write8(uint32_t addr, u32x2 w) {
  *(__attribute__((address_space(3))) u32x2*)(uintptr_t)(addr + OFF) = w;
}
__device__ __forceinline__ f32x4 lds_quad(uint32_t addr) {
  return __builtin_bit_cast(f32x4, lds_read16<0>(addr));
}
__device__ __forceinline__ float lds_read4(uint32_t addr) {
  return *(__attribute__((address_space(3))) const float*)(uintptr_t)addr;
}
__device__ __forceinline__ void lds_write4(uint32_t addr, float x) {
  *(__attribute__((address_space(3))) float*)(uintptr_t)addr = x;
}
__device__ __forceinline__ void lds_write16(uint32_t addr, u32x4 w) {
  *(__attribute__((address_space(3))) u32x4*)(uintptr_t)addr = w;
}

template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t u, float* f) {
  if constexpr (BF16) {
    f[0] = __builtin_bit_cast(float, u << 16);
    f[1] = __builtin_bit_cast(float, u & 0xffff0000u);
  } else {
    const f16x2 x = __builtin_bit_cast(f16x2, u);
    f[0] = (float)x[0];
    f[1] = (float)x[1];
  }
}
template <bool BF16>
__device__ __forceinline__ void unpack8(u32x4 w, float* f) {
#pragma unroll
  for (int j = 0; j < 4; ++j) unpack2<BF16>(w[j], f + 2 * j);
}

// A tile that some row or key does not see whole: 0 times an infinity or NaN of a
// masked row would be NaN in the products that sum over these rows.  Clears the
// infinities and NaN among the ROWS rows at LDS address `at`, which this wave has
// staged, and returns the rows (bit r) that held any.
template <int D, bool BF16, int ROWS>
__device__ __forceinline__ unsigned clean_rows(uint32_t at) {
  constexpr int ROWB = 2 * D, NI = ROWS * ROWB / 1024, LPR = ROWB / 16;
  constexpr uint32_t E = BF16 ? 0x7F807F80u : 0x7C007C00u, L = BF16 ? 0x00800080u : 0x04000400u;
  const int lane = lane_now();
  unsigned rows = 0;
#pragma unroll
  for (int it = 0; it < NI; ++it) {
    const uint32_t addr = at + it * 1024 + lane * 16;
    u32x4 w = __builtin_bit_cast(u32x4, lds_read16<0>(addr));
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) any |= (w[j] & E) + L;  // an exponent of all ones carries
    uint64_t bad = __ballot((any & 0x80008000u) != 0);
    if (__builtin_expect(bad == 0, true)) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t half = ((w[j] & E) + L) & 0x80008000u;
      w[j] &= ~(((half >> 15) << 16) - (half >> 15));
    }
    lds_write16(addr, w);
    for (int r = 0; r < 64 / LPR; ++r)
      if ((bad >> (r * LPR)) & ((1ull << LPR) - 1)) rows |= 1u << (it * (64 / LPR) + r);
  }
  return rows;
}

}  // namespace
}  // namespace fa
