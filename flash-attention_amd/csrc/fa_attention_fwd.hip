// Attention of whole tensors with capped, biased and masked scores, on gfx950.
//
//   z = scale q_i.k_j;  c = cap tanh(z / cap);  x = c - slope |p_i - j|
//   o_i = sum_j P v_j, P = exp(x - lse_i), over the keys lo_i <= j < hi_i
//
// A workgroup has 128 rows of a head and passes once over the keys that any of them
// sees, 64 at a time through a two-deep LDS ring: one team of four waves of 32 rows
// (WaveAttn), or two that take turns with the tiles and join their sums (plan:
// attn_args).  Its keys start at the first one that a row sees, so that the tiles
// of a document begin with it.
//
// Bound by the matrix cores at the power limit where rows are long: 2 x 8192 causal tokens,
// 32 heads on 8, D = 128, bf16, 1040 us, 1060 TFLOP/s of visible pairs (busy 57 % of the cycles, at
// 1.9 GHz); a matrix product of 8192^3 reaches 1245.  With capped scores by the vector
// units, 1310 us.  Short rows: the chain of the longest tile, about 1.5 us a tile.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_attention_ops.h"
#include "fa_wave_attn.h"

namespace fa {
namespace {

using namespace dev;

// Team by team of four waves, TEAMS of them.
template <int D, bool BF16, int TEAMS>
__global__ void __launch_bounds__(256 * TEAMS) __attribute__((amdgpu_waves_per_eu(2, 2)))
    fa_attn_fwd_kernel(const AttnArgs a) {
  using W = WaveAttn<D, BF16, 4, 2, true>;
  constexpr int ROWB = 2 * D, TB = 64 * ROWB;
  __shared__ __attribute__((aligned(1024))) char smem[TEAMS * 4 * TB];  // of each team K0 K1 V0 V1
  __shared__ int again;

  const int lane = threadIdx.x & 63;
  const int team = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;  // of its team
  if (threadIdx.x == 0) again = 0;  // ordered by the first barrier
  int unit, within;  // (the last tiles first, which are the longest of a causal mask)
  if (!unit_and_place(a.rows, unit, within)) return;
  const int back = fast_div(within, a.by_group);
  const int b = fast_div(unit, a.by_kvh), kvh = unit - b * a.kv_heads;
  const int h = kvh * a.group + within - back * a.group;
  const int row0 = (a.tiles - 1 - back) * kAttnRows, wrow0 = row0 + 32 * wave;

  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(smem)) + team * 4 * TB;
  W w;
  w.init(base, base + 2 * TB, a.scale_log2);
  w.init_score(a.score);
  const int l16 = w.l16, g4 = w.g4;
  const float slope = w.score.biased ? a.score.slopes[h] * a.score.slope_unit : 0.0f;
  TileKeys keys, all;  // of the wave's rows, of the workgroup's
  tile_keys(a, b, row0, wave, keys, all);
  const int c0 = all.lo, c1 = all.hi;  // (no key: kNoKey and 0)
  const int n_tiles = c0 < c1 ? (c1 - c0 + 63) / 64 : 0;
  // Tile t TEAMS + team is the team's in turn t.  With a bias by distance the last one comes
  // first: a causal row's scores grow towards it, and its offset would be raised tile by tile
  // (us, 2 x 8192 causal rows, 32 heads on 8, D = 128: 1380 and 1095; a window of 1024 without a
  // bias, 16384 rows, 16 heads: 184 from the first, 190 from the last).
  const int turns = (n_tiles + TEAMS - 1) / TEAMS;
  const bool down = w.score.biased;
  const int first_key = down ? c0 + 64 * (n_tiles - 1) : c0, tile_step = down ? -64 : 64;
  auto key_of = [&](int t) FA_INLINE { return first_key + tile_step * (t * TEAMS + team); };
  const char* kh = a.k.p + b * a.k.sb + kvh * a.k.sh;
  const char* vh = a.v.p + b * a.v.sb + kvh * a.v.sh;
  GroupStage<D> stage;
  stage.init(lane, (uint32_t)a.k.st, (uint32_t)a.v.st);
  auto issue = [&](int t, int buf) FA_INLINE {
    if (t * TEAMS + team >= n_tiles) return;
    const int r0 = min(key_of(t) + 16 * wave, c1 - 1);
    const uint32_t dst = base + buf * TB + wave * 16 * ROWB;
    stage.copy(kh + r0 * a.k.st, vh + r0 * a.v.st, dst, dst + 2 * TB, c1 - 1 - r0, (uint32_t)a.k.st,
               (uint32_t)a.v.st);
  };
  issue(0, 0);
  // (behind the first copies: one wait for all)
  const char* qh = a.q.p + b * a.q.sb + h * a.q.sh;
  RowKeys see[2];
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) see[rb] = row_keys(a, b, min(wrow0 + 16 * rb + l16, a.n - 1));
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const int i = min(wrow0 + 16 * rb + l16, a.n - 1);
    w.first[rb] = see[rb].lo;
    w.last[rb] = see[rb].hi - 1;
    w.pos[rb] = i + a.m - a.n;
    w.slope[rb] = slope;
#pragma unroll
    for (int st = 0; st < W::KST; ++st)
      w.qf[rb][st] = *reinterpret_cast<const i16x8*>(qh + i * a.q.st + (32 * st + 8 * g4) * 2);
  }
  auto end_tile = [&]() FA_INLINE {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
  };
  end_tile();
  // Tiles with a masked key, those that every row of the wave sees whole, and the
  // rest.  Every wave passes one barrier a tile, whichever loop it is in.
  int t = 0, buf = 0;
  auto masked = [&](int end) FA_INLINE {
    for (; t < end; ++t, buf ^= 1) {
      const int k0 = key_of(t);
      issue(t + 1, buf ^ 1);
      if (k0 < keys.hi && k0 + 64 > keys.lo)
        w.template step<0, kTrusting>(k0, 15u, buf * TB);
      end_tile();
    }
  };
  const int whole0 = keys.all_lo <= c0 ? 0 : (int)min((uint32_t)n_tiles, ((uint32_t)(keys.all_lo - c0) + 63) / 64);
  const int whole1 = min(n_tiles, max(keys.all_hi - c0, 0) / 64);
  auto turns_to = [&](int tiles) FA_INLINE { return (max(tiles - team, 0) + TEAMS - 1) / TEAMS; };
  const int turn1 = turns_to(down ? n_tiles - whole0 : whole1);
  masked(turns_to(down ? n_tiles - whole1 : whole0));
  for (; t < turn1; ++t, buf ^= 1) {
    issue(t + 1, buf ^ 1);
    w.template step<0, kWhole>(key_of(t), 15u, buf * TB);
    end_tile();
  }
  masked(turns);
  // 0 times an infinity or NaN of a masked key: the sum is NaN.  Then all start again
  // (the staging is shared) with steps that take care of them.  (In place of a look at V in
  // each masked tile: 16384 rows in a window of 1024, 16 heads, D = 128, fp16, 187 us before,
  // 181 now; documents in 16384 rows, 32 heads on 8, bf16, 461 and 434.)
  if (whole0 > 0 || whole1 < n_tiles)
    if (w.any_nan() && lane == 0) again = 1;
  __syncthreads();
  if (__builtin_expect(__builtin_amdgcn_readfirstlane(again) != 0, false)) {
    w.reset();
    issue(0, 0);
    end_tile();
    buf = 0;
    for (t = 0; t < turns; ++t, buf ^= 1) {
      const int k0 = key_of(t);
      issue(t + 1, buf ^ 1);
      if (k0 < keys.hi && k0 + 64 > keys.lo) w.template step<0, kSafe>(k0, 15u, buf * TB);
      end_tile();
    }
  }

  // The second team hands its sums to the first, by wave and lane.
  if constexpr (TEAMS == 2) {
    constexpr int PART = (D / 16 * 2 + 2) * 1024;
    const uint32_t at = lds_addr(smem) + wave * PART + lane * 16;
    if (team == 1) {
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
#pragma unroll
        for (int db = 0; db < W::DB; ++db)
          lds_write16(at + (2 * db + rb) * 1024, __builtin_bit_cast(u32x4, w.o[db][rb]));
        lds_write16(at + (2 * W::DB + rb) * 1024, __builtin_bit_cast(u32x4, f32x4{w.m[rb], w.ls[rb][0], w.lu[rb], 0.0f}));
      }
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __syncthreads();
    if (team == 1) return;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const f32x4 x = lds_quad(at + (2 * W::DB + rb) * 1024);
      const float m = fmaxf(w.m[rb], x[0]);
      const float own = w.m[rb] == m ? 1.0f : fast_exp2((w.m[rb] - m) * w.c);
      const float other = x[0] == m ? 1.0f : fast_exp2((x[0] - m) * w.c);
      w.m[rb] = m;
      w.ls[rb][0] = w.ls[rb][0] * own + x[1] * other;
      w.lu[rb] = w.lu[rb] * own + x[2] * other;
#pragma unroll
      for (int db = 0; db < W::DB; ++db)
        w.o[db][rb] = w.o[db][rb] * own + lds_quad(at + (2 * db + rb) * 1024) * other;
    }
  }

  float inv[2], lu[2];
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    inv[rb] = w.ls[rb][0] == 0.0f ? 0.0f : 1.0f / w.ls[rb][0];
    lu[rb] = W::red_sum(w.lu[rb]);
  }
  char* oh = a.o.p + b * a.o.sb + h * a.o.sh;
  char* ot = smem + wave * (TEAMS == 1 ? 32 * ROWB : (D / 16 * 2 + 2) * 1024);
  write_rows<D, BF16>(ot, w.o, inv, lane, [&](int r) FA_INLINE -> char* {
    return wrow0 + r < a.n ? oh + (wrow0 + r) * a.o.st : nullptr;
  });
  if (a.o_low != nullptr) {  // (nothing of what is no number, or rounds to none)
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
      for (int db = 0; db < W::DB; ++db) {
        const f32x4 x = w.o[db][rb] * inv[rb];
        float r[4];
        unpack2<BF16>(pack2<BF16>(x[0], x[1]), r);
        unpack2<BF16>(pack2<BF16>(x[2], x[3]), r + 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) w.o[db][rb][i] = fabsf(r[i]) < INFINITY ? x[i] - r[i] : 0.0f;
      }
    const float one[2] = {1.0f, 1.0f};
    char* lh = a.o_low + ((int64_t)b * a.heads + h) * a.n * ROWB;
    write_rows<D, BF16>(ot, w.o, one, lane, [&](int r) FA_INLINE -> char* {
      return wrow0 + r < a.n ? lh + (int64_t)(wrow0 + r) * ROWB : nullptr;
    });
  }
  if (a.lse != nullptr && g4 < 2) {
    const int r = wrow0 + 16 * g4 + l16;
    const float m = g4 == 0 ? w.m[0] : w.m[1], sum = g4 == 0 ? w.ls[0][0] : w.ls[1][0];
    const float l = g4 == 0 ? lu[0] : lu[1];
    if (r < a.n)
      a.lse[((int64_t)b * a.heads + h) * a.n + r] = sum == 0.0f ? -INFINITY : w.log2_sum(m, l) * kLn2;
  }
}

template <int D, bool BF16>
hipError_t launch_as(const AttnArgs& a, hipStream_t stream) {
  const int64_t grid = grid_size(a.rows);
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  void* kargs[] = {const_cast<AttnArgs*>(&a)};
  const void* fn = a.row_teams == 1 ? reinterpret_cast<const void*>(&fa_attn_fwd_kernel<D, BF16, 1>)
                                    : reinterpret_cast<const void*>(&fa_attn_fwd_kernel<D, BF16, 2>);
  return hipLaunchKernel(fn, dim3((unsigned)grid), dim3(256 * a.row_teams), kargs, 0, stream);
}

}  // namespace

hipError_t launch_attn_fwd(const AttnArgs& a, int head_dim, bool bf16, hipStream_t stream) {
  if (head_dim == 128) return bf16 ? launch_as<128, true>(a, stream) : launch_as<128, false>(a, stream);
  return bf16 ? launch_as<64, true>(a, stream) : launch_as<64, false>(a, stream);
}

}  // namespace fa
