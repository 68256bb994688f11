// Attention of a wave's rows over tiles of keys in LDS, on v_mfma_f32_16x16x32:
// products, scores, the running softmax and the handling of masked keys.  Shared
// by the kernels over a paged cache and by attention on whole tensors.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_device_ops.h"
#include "fa_lds_layout.h"
#include "fa_paged_ops.h"
#include "fa_score.h"

namespace fa {
namespace {

using namespace dev;

// Offset and limit of the lazy softmax, as in fa_fwd_kernel.hip: the offset is
// raised, to kHeadroom above the row max, only when a tile's sum of p reaches
// kSumLimit, so every P is finite in fp16 and the largest stays normal.
constexpr float kSumLimit = 61440.0f;
template <bool BF16>
constexpr float kHeadroom = BF16 ? 4.0f : 1.0f;

constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

// kTrusting: kMasked, but for its look for infinities and NaN.
enum StepMode { kWhole, kMasked, kTrusting, kSafe };

// The state of a wave's RB blocks of 16 rows over tiles of 16 NKB keys, on
// v_mfma_f32_16x16x32 with the layouts of fa_fwd16_kernel: S^T = K Q^T (lane
// l: keys 16kb + 4 (l / 16) + i of row 16rb + l % 16), O^T += V^T P^T.
// SCORED: scores may be capped and biased, and a row's keys begin at first[rb].
template <int D, bool BF16, int NKB, int RB, bool SCORED = false>
struct WaveAttn {
  static constexpr int KST = D / 32, DB = D / 16, ROWB = 2 * D, NCH = NKB / 2;
  i16x8 qf[RB][KST];
  f32x4 o[DB][RB];
  f32x4 ls[RB];             // row sums of the rounded P (every element)
  float lu[RB];             // this lane's sums of the unrounded p
  float m[RB], nmc[RB];     // offset (raw scores) and -m c, +inf while m = -inf
  int last[RB];             // last key this lane's row sees
  uint32_t k_addr[KST], v_addr[DB];  // LDS operand addresses in tile 0
  float c;
  int lane, l16, g4;
  bool odd;                 // a masked tile held an infinity or NaN (uniform)
  // SCORED
  int first[RB];            // first key this lane's row sees
  int pos[RB];              // the row's place among the keys
  float slope[RB];          // slope of its bias, in units of the scores
  Score score;

  __device__ __forceinline__ void init(uint32_t k_lds, uint32_t v_lds, float scale_log2) {
    lane = threadIdx.x & 63;
    l16 = lane & 15;
    g4 = lane >> 4;
    c = scale_log2;
#pragma unroll
    for (int st = 0; st < KST; ++st) k_addr[st] = k_lds + lds::k16_read_offset<D>(0, st, lane);
#pragma unroll
    for (int db = 0; db < DB; ++db) v_addr[db] = v_lds + lds::v16_read_offset<D>(0, 0, db, lane);
    reset();
  }
  __device__ __forceinline__ void reset() {
    odd = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db][rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      ls[rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      lu[rb] = 0.0f;
      m[rb] = -INFINITY;
      nmc[rb] = INFINITY;
    }
  }

  // Behind init.
  __device__ __forceinline__ void init_score(const ScoreArgs& a) {
    score.init(a);
    if (score.capped) c = score.twice;
  }

  // log2 of the sum of exponentials, from the offset and the sum by it.
  __device__ __forceinline__ float log2_sum(float offset, float sum) const {
    const float x = offset * c + __log2f(sum);
    return SCORED ? x + score.left_out() : x;
  }

  static __device__ __forceinline__ float red_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
  }
  static __device__ __forceinline__ float red_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
  }

  // One tile of keys kt0.. in LDS, OFF + off bytes behind the tile-0 addresses.
  // MODE kWhole: every row sees all of it.  Else some row sees only part of it,
  // or a group is absent (bit kb of `present` clear), and 0 times an infinity or
  // NaN of a masked key must not reach o: kMasked notes such elements in the V
  // tile (at v_tile) in `odd`, and the caller starts again with kSafe, which
  // takes care of them.  (One step that does either spilled 32 registers.)
  template <int OFF, int MODE>
  __device__ __forceinline__ void step(int kt0, unsigned present, uint32_t off, uint32_t v_tile = 0) {
    constexpr bool MASKED = MODE != kWhole;
    f32x4 s[NKB][RB];
    {
      constexpr int NK = NKB * KST, KW = NK < 3 ? NK : 3;
      i16x8 ka[KW];
      static_for<0, KW>([&](auto i_c) FA_INLINE {
        constexpr int i = decltype(i_c)::value;
        ka[i] = lds_read16<OFF + (i % NKB) * 16 * ROWB>(k_addr[i / NKB] + off);
      });
      __builtin_amdgcn_sched_barrier(0);
      static_for<0, NK>([&](auto i_c) FA_INLINE {
        constexpr int i = decltype(i_c)::value;
        constexpr int st = i / NKB, kb = i % NKB;
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
          s[kb][rb] = mfma16<BF16>(ka[i % KW], qf[rb][st], st == 0 ? zero : s[kb][rb]);
        if constexpr (i + KW < NK) {
          constexpr int n = i + KW;
          ka[i % KW] = lds_read16<OFF + (n % NKB) * 16 * ROWB>(k_addr[n / NKB] + off);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    }
    constexpr int NPV = NCH * DB, VD = NPV < 4 ? NPV : 4;
    i16x8 va[VD];
    auto read_v = [&](auto i_c) FA_INLINE {
      constexpr int i = decltype(i_c)::value;
      constexpr int at = OFF + (i / DB) * 32 * ROWB;
      va[i % VD] = ds_read_tr_pair<at, at + 16 * ROWB>(v_addr[i % DB] + off);
    };
    if constexpr (!MASKED) static_for<0, VD>(read_v);
    __builtin_amdgcn_sched_barrier(0);

    if constexpr (SCORED) {
      if (score.capped)
        each(s, [&](float x, int, int, int) FA_INLINE { return score.minus_tail(x); });
      if (score.biased) {
        float at[RB];  // the lane's first key as seen from its row
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) at[rb] = (float)(kt0 + 4 * g4 - pos[rb]);
        each(s, [&](float x, int kb, int rb, int i) FA_INLINE {
          return fmaf(-slope[rb], fabsf(at[rb] + (float)(16 * kb + i)), x);
        });
      }
    }
    if constexpr (MASKED) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int rel = last[rb] - kt0 - 4 * g4;
        const int rel_first = SCORED ? first[rb] - kt0 - 4 * g4 : 0;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
          const int lim = (present >> kb) & 1u ? rel - 16 * kb : -1;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i > lim || (SCORED && i < rel_first - 16 * kb)) s[kb][rb][i] = -INFINITY;
        }
      }
    }

    // P = exp2(s c - m c), packed as P^T: chunk ch, word j of key block
    // 2ch + j / 2, scores 2 (j % 2) and the next.
    i16x8 pf[NCH][RB];
    float tsum[RB];
    auto pack_p = [&]() FA_INLINE {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        tsum[rb] = 0.0f;
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
          u32x4 w;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int kb = 2 * ch + (j >> 1), i = 2 * (j & 1);
            const float p0 = fast_exp2(fmaf(s[kb][rb][i], c, nmc[rb]));
            const float p1 = fast_exp2(fmaf(s[kb][rb][i + 1], c, nmc[rb]));
            w[j] = pack2<BF16>(p0, p1);
            tsum[rb] += p0 + p1;
          }
          pf[ch][rb] = __builtin_bit_cast(i16x8, w);
        }
      }
    };
    pack_p();
    bool over = !(tsum[0] < kSumLimit);
#pragma unroll
    for (int rb = 1; rb < RB; ++rb) over = over || !(tsum[rb] < kSumLimit);
    if (__any(over)) {
      // The offset of every row whose max exceeds it moves to kHeadroom above
      // that max; rows without a visible key so far keep m = -inf and P = 0.
      float keep[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
          mx = max3(mx, max3(s[kb][rb][0], s[kb][rb][1], s[kb][rb][2]), s[kb][rb][3]);
        mx = red_max(mx);
        bool grow = mx > m[rb];
        if constexpr (SCORED) {
          // (only a row's own sums: no bit of it goes by the rows beside it)
          const int own = !(tsum[rb] < kSumLimit);
          const int pair = own | __shfl_xor(own, 16);
          grow = grow && (pair | __shfl_xor(pair, 32)) != 0;
        }
        const float m_new = grow ? mx + kHeadroom<BF16> / c : m[rb];
        const float alpha = fast_exp2(grow ? (m[rb] - m_new) * c : 0.0f);
        m[rb] = m_new;
        lu[rb] *= alpha;
        ls[rb] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db][rb] *= alpha;
        keep[rb] = m_new == -INFINITY ? INFINITY : -m_new * c;
        nmc[rb] = m_new == -INFINITY ? 0.0f : keep[rb];
      }
      pack_p();
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) nmc[rb] = keep[rb];
    }
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) lu[rb] += tsum[rb];
    const short one = BF16 ? (short)0x3F80 : (short)0x3C00;
    const i16x8 ones = {one, one, one, one, one, one, one, one};

    if constexpr (MODE == kSafe) {
      pv_safe(kt0, present, off, pf);
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) ls[rb] = mfma16<BF16>(ones, pf[ch][rb], ls[rb]);
      return;
    }
    if constexpr (MODE == kMasked) odd = odd || any_non_finite(v_tile);
    if constexpr (MODE == kMasked || MODE == kTrusting) static_for<0, VD>(read_v);
    // With two waves on a SIMD unit, the one in its products goes first: the
    // other's exponentials fill the gaps.  4096 tokens over 16384 keys, bf16, 32
    // heads on 8, us without and with: D = 128 causal 827 and 798, without the
    // mask 948 and 903, there 939 with Q K^T as well; D = 64 530 and 527, and 603
    // and 601, so not there.
    constexpr bool FIRST = NKB == 4 && D == 128;
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(1);
    __builtin_amdgcn_sched_barrier(0);
    static_for<0, NPV>([&](auto j_c) FA_INLINE {
      constexpr int j = decltype(j_c)::value;
      constexpr int ch = j / DB, db = j % DB;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        o[db][rb] = mfma16<BF16>(va[j % VD], pf[ch][rb], o[db][rb]);
        if constexpr (db == DB - 1) ls[rb] = mfma16<BF16>(ones, pf[ch][rb], ls[rb]);
      }
      if constexpr (j + VD < NPV) read_v(std::integral_constant<int, j + VD>{});
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (FIRST) __builtin_amdgcn_s_setprio(0);
  }

  template <class F>
  static __device__ __forceinline__ void each(f32x4 (&s)[NKB][RB], F&& f) {
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[kb][rb][i] = f(s[kb][rb][i], kb, rb, i);
  }

  // Whether some sum is NaN.  It stays so, once it is.
  __device__ __forceinline__ bool any_nan() const {
    bool nan = false;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = 0; i < 4; ++i) nan = nan || o[db][rb][i] != o[db][rb][i];
    return __any(nan);
  }

  // Whether the V tile at LDS address v_tile holds an infinity or a NaN.
  __device__ __forceinline__ bool any_non_finite(uint32_t v_tile) {
    constexpr uint32_t E = BF16 ? 0x7F807F80u : 0x7C007C00u, L = BF16 ? 0x00800080u : 0x04000400u;
    uint32_t any = 0;
#pragma unroll
    for (int it = 0; it < 16 * NKB * ROWB / 1024; ++it) {
      const u32x4 w = __builtin_bit_cast(u32x4, lds_read16<0>(v_tile + it * 1024 + lane * 16));
#pragma unroll
      for (int j = 0; j < 4; ++j) any |= (w[j] & E) + L;  // an exponent of all ones carries
    }
    return __any((any & 0x80008000u) != 0);
  }

  // O += P V of a masked tile with infinities or NaN in V:
  // the product with infinities and NaN as 0, and per (row, dim) a count of
  // those among the keys that the row sees, on the matrix core with weights 1
  // (+inf), 2^7 (-inf) and 2^14 (NaN), at most 64 of each: sums that fp32
  // holds exactly.
  __device__ __forceinline__ void pv_safe(int kt0, unsigned present, uint32_t off,
                                          const i16x8 (&pf)[NCH][RB]) {
    constexpr uint32_t E = BF16 ? 0x7F807F80u : 0x7C007C00u, L = BF16 ? 0x00800080u : 0x04000400u;
    constexpr uint32_t M = BF16 ? 0x007F007Fu : 0x03FF03FFu, H = 0x80008000u;
    constexpr uint32_t kOne = BF16 ? 0x3F80u : 0x3C00u;
    constexpr uint32_t kPos = kOne * 0x10001u, kNeg = (BF16 ? 0x4300u : 0x5800u) * 0x10001u;
    constexpr uint32_t kNan = (BF16 ? 0x4680u : 0x7400u) * 0x10001u;
    i16x8 see[NCH][RB];  // 1 for a visible key, laid out as P
#pragma unroll
    for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        u32x4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int kb = 2 * ch + (j >> 1), key = kt0 + 16 * kb + 4 * g4 + 2 * (j & 1);
          const bool there = (present >> kb) & 1u;
          const int lo = SCORED ? first[rb] : 0;
          w[j] = (there && key <= last[rb] && key >= lo ? kOne : 0u) |
                 (there && key + 1 <= last[rb] && key + 1 >= lo ? kOne << 16 : 0u);
        }
        see[ch][rb] = __builtin_bit_cast(i16x8, w);
      }
    static_for<0, DB>([&](auto db_c) FA_INLINE {
      constexpr int db = decltype(db_c)::value;
      f32x4 n[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) n[rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      static_for<0, NCH>([&](auto ch_c) FA_INLINE {
        constexpr int ch = decltype(ch_c)::value, at = ch * 32 * ROWB;
        const u32x4 v =
            __builtin_bit_cast(u32x4, ds_read_tr_pair<at, at + 16 * ROWB>(v_addr[db] + off));
        u32x4 fin, ind;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          auto spread = [](uint32_t x) FA_INLINE { return ((x >> 15) << 16) - (x >> 15); };  // bit 15 -> half
          const uint32_t bad = spread(((v[j] & E) + L) & H);
          const uint32_t nan = bad & spread(((v[j] & M) + 0x7FFF7FFFu) & H);
          const uint32_t neg = spread(v[j] & H);
          fin[j] = v[j] & ~bad;
          ind[j] = (nan & kNan) | (bad & ~nan & ((neg & kNeg) | (~neg & kPos)));
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          o[db][rb] = mfma16<BF16>(__builtin_bit_cast(i16x8, fin), pf[ch][rb], o[db][rb]);
          n[rb] = mfma16<BF16>(__builtin_bit_cast(i16x8, ind), see[ch][rb], n[rb]);
        }
      });
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int x = (int)n[rb][e];
          if (x & 127) o[db][rb][e] += INFINITY;
          if ((x >> 7) & 127) o[db][rb][e] -= INFINITY;
          if (x >> 14) o[db][rb][e] = NAN;
        }
      __builtin_amdgcn_sched_barrier(0);
    });
  }
};

// Writes a wave's 32 rows, o[db][rb] as WaveAttn holds them times f[rb], to
// row(r) (NULL: none).  Lanes l and l ^ 16 swap halves so each holds a 16-byte
// piece of a row; whole rows leave through an LDS row tile of the wave, `ot`.
template <int D, bool BF16, class Row>
__device__ __forceinline__ void write_rows(char* ot, const f32x4 (&o)[D / 16][2], const float (&f)[2],
                                           int lane, Row&& row) {
  constexpr int ROWB = 2 * D, DB = D / 16;
  const int l16 = lane & 15, g4 = lane >> 4, my_rb = g4 & 1;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    u32x2 own[2];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
      own[rb] = u32x2{pack2<BF16>(o[db][rb][0] * f[rb], o[db][rb][1] * f[rb]),
                      pack2<BF16>(o[db][rb][2] * f[rb], o[db][rb][3] * f[rb])};
    const u32x2 send = my_rb == 0 ? own[1] : own[0];
    const u32x2 recv = {(uint32_t)__shfl_xor((int)send[0], 16), (uint32_t)__shfl_xor((int)send[1], 16)};
    const u32x2 mine = my_rb == 0 ? own[0] : own[1];
    const u32x4 x = my_rb == 0 ? u32x4{mine[0], mine[1], recv[0], recv[1]}
                               : u32x4{recv[0], recv[1], mine[0], mine[1]};
    *reinterpret_cast<u32x4*>(ot + lds::row_tile_offset(16 * my_rb + l16, 2 * db + (g4 >> 1), ROWB)) = x;
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  constexpr int NC = ROWB / 16, RPI = 64 / NC;
  const int rr = lane / NC, cc = lane & (NC - 1);
#pragma unroll
  for (int j = 0; j < 32 / RPI; ++j) {
    const int r = j * RPI + rr;
    const u32x4 x = *reinterpret_cast<const u32x4*>(ot + lds::row_tile_offset(r, cc, ROWB));
    char* to = row(r);
    if (to != nullptr) *reinterpret_cast<u32x4*>(to + cc * 16) = x;
  }
}

}  // namespace
}  // namespace fa
