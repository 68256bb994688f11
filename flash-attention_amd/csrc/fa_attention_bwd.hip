// Gradients of attention with capped, biased and masked scores, on gfx950.
//
//   delta_i = go_i.(o_i + o_low_i) - glse_i;  dS = P (go_i.v_j - delta_i) (1 - (c / cap)^2)
//   gv_j = sum_i P go_i;  gk_j = scale sum_i dS q_i;  gq_i = scale sum_j dS k_j
//
// P is computed again from the logsumexp.  No atomics on results: sums run in a fixed
// order, at the price of computing scores and go.v twice (7 products of the size of
// q.k in place of 5):
//  * fa_attn_rows_kernel: delta, the keys that each row sees, and, for every span
//    of 32 rows, their limits.
//  * fa_attn_order_kernel, with key ranges: which tiles of keys have most rows.
//  * fa_attn_dkv_kernel: 128 keys of a kv head, four waves of 32, whose K and V
//    stay in registers; passes over the spans of 32 rows that see any of them, of all query
//    heads of the group, staged through a ring.  S = Q K^T and go V^T come out with
//    lanes along the keys, as P and dS have to go into gv^T += go^T P and
//    gk^T += Q^T dS.  Few keys and many rows are split over workgroups, whose parts
//    fa_attn_join_kernel adds.
//  * fa_attn_dq_kernel: 128 rows of a head, as the forward pass.
// Where workgroups are few, teams of four waves share one's spans or tiles (plan_attn_bwd).
//
// 2 x 8192 causal tokens, 32 heads on 8, D = 128, bf16, us: rows 47 (75 with o_low, 5.3 TB/s), dk and
// dv 2170 (1010 TFLOP/s of their four products), dq 1480 (1120 of three); a matrix product
// of 8192^3 reaches 1245.  The matrix cores are busy 49 and 55 % of the cycles, at 1.9 GHz (the power
// limit); capped scores add vector work, 2430 and 1790.  fp16, on a box that takes 1930 and 1357 for these:
// 2135 and 1466; D = 64 1460 and 820, vector units (the look at dS's factors is 85 of each dk, dv).
//
// Rounding: P and dS are rounded to the input type for the matrix cores (as P of
// the forward pass); all sums are fp32.  fp16 has few exponents: P is scaled by
// 2^12, so that it keeps its 11 bits down to 2^-26, and dS by a power of two, by what bounds it:
//   |dS_ij| <= |go_i| |v_j| + |delta_i|   (P and the derivative are at most 1; |.|: 2-norms)
//  * dk: a key's rows so far that see it; the bound goes to 2^12 .. 2^13 and may grow to 2^15
//    before the factor and the sum so far are lowered.  (Of all rows of the head: a row that does
//    not see the key, of another document or before it, would decide what is left of its sums.)
//  * dq: a row's bound for |v| up to 64, at 2^12 .. 2^13 too.  Should a sum be no number all the
//    same, the rows start again with that for the largest |v| that there is, 2^20.  (The largest
//    dS is then above 2: what is lost is below 2^-26 of it.)
// What dS loses to the type's least step, 2^-25, is below 2^-37 of the bound.
//
// Masked keys and rows contribute nothing whatever they hold: their P and dS are
// 0, and infinities and NaN among the staged rows of a tile that is not seen
// whole are cleared (clean_rows); rows and keys that do see one get NaN, also those
// of a wave whose own part of the tile is seen whole.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "fa_attention_ops.h"
#include "fa_wave_attn.h"

namespace fa {
namespace {

using namespace dev;

template <bool BF16>
constexpr float kShift = BF16 ? 0.0f : 12.0f;  // log2 of P's factor

// The record of a span, [2][4 fields][16 rows] floats: for each 16 rows
enum RecordField { kLse, kDelta, kLo, kHi };  // (lse in log2, less kShift and the cap; minus delta)
// fp16: then |go| of each row, and the largest |go| and |delta| of all; 0 in place of infinities and NaN,
// for whose rows and keys no factor helps.
constexpr int kRowNorms = 4 * kSpan, kSpanMost = kRowNorms + kSpan;
template <bool BF16>
constexpr int kRecord = record_floats(BF16);
// dS is made with a quarter of capped scores' derivative, 1 - tanh^2 = 4 tail (1 - tail).
template <bool CAP>
constexpr float kQuarters = CAP ? 4.0f : 1.0f;
// The largest product of a factor (which holds these, and P's 2^-12) with the bound of dS.
template <bool CAP>
constexpr float kBoundMost = 8.0f * kQuarters<CAP>;
// dS's factor for a bound in [2^e, 2^(e + 1)).
template <bool CAP>
__device__ __forceinline__ float grad_factor(float bound) {
  const int e = (int)((__builtin_bit_cast(uint32_t, bound) >> 23) & 255) - 127;
  return kQuarters<CAP> * __builtin_bit_cast(float, (uint32_t)(127 - min(max(e, -60), 100)) << 23);
}

// ---- rows ----

// 64 rows of one head a workgroup, D / 8 lanes a row.  Bound by reading go and o.
constexpr int kRowsBlock = 64;
template <int D, bool BF16>
__global__ void __launch_bounds__(256) fa_attn_rows_kernel(const AttnArgs a) {
  constexpr int LPR = D / 8, RPP = 256 / LPR;  // rows of a pass
  __shared__ float delta[kRowsBlock], squares[kRowsBlock];
  const int blocks = (a.n + kRowsBlock - 1) / kRowsBlock;
  const int bh = blockIdx.x / blocks, block = blockIdx.x - bh * blocks;
  const int b = bh / a.heads, h = bh - b * a.heads;
  const char* gh = a.go.p + b * a.go.sb + h * a.go.sh;
  const char* oh = a.o.p + b * a.o.sb + h * a.o.sh;
#pragma unroll
  for (int r0 = 0; r0 < kRowsBlock; r0 += RPP) {
    const int r = r0 + (int)threadIdx.x / LPR;
    const int64_t i = min(block * kRowsBlock + r, a.n - 1);
    const int at = (int)threadIdx.x % LPR * 16;
    float g[8], o[8], sum = 0.0f, square = 0.0f;
    unpack8<BF16>(*reinterpret_cast<const u32x4*>(gh + i * a.go.st + at), g);
    unpack8<BF16>(*reinterpret_cast<const u32x4*>(oh + i * a.o.st + at), o);
    if (a.o_low != nullptr) {
      float low[8];
      unpack8<BF16>(*reinterpret_cast<const u32x4*>(a.o_low + ((int64_t)bh * a.n + i) * 2 * D + at), low);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] += low[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sum = fmaf(g[j], o[j], sum);
      if constexpr (!BF16) square = fmaf(g[j], g[j], square);
    }
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) {
      sum += __shfl_xor(sum, d);
      if constexpr (!BF16) square += __shfl_xor(square, d);
    }
    if (threadIdx.x % LPR == 0) {
      delta[r] = sum;
      squares[r] = square;
    }
  }
  __syncthreads();
  if (threadIdx.x >= kRowsBlock) return;
  const int r = threadIdx.x, i = block * kRowsBlock + r, span = i / kSpan;
  RowKeys k = {kNoKey, 0};
  float lse = INFINITY, d = 0.0f, norm = 0.0f;  // P = 0
  if (i < a.n) {
    k = row_keys(a, b, i);
    if (k.hi > 0) {
      const int64_t at = (int64_t)bh * a.n + i;
      lse = a.lse[at] * kLog2e - kShift<BF16> - a.score.cap;  // (the cap that scores leave out)
      d = (a.glse != nullptr ? a.glse[at] : 0.0f) - delta[r];
      norm = sqrtf(squares[r]);
    }
  }
  TileKeys t;
  t.start(k);
  t.reduce<kSpan>();
  float most[2] = {norm < INFINITY ? norm : 0.0f, fabsf(d) < INFINITY ? fabsf(d) : 0.0f};
  norm = most[0];
  if constexpr (!BF16) {
#pragma unroll
    for (int w = 1; w < kSpan; w <<= 1)
#pragma unroll
      for (int i = 0; i < 2; ++i) most[i] = fmaxf(most[i], __shfl_xor(most[i], w));
  }
  if (span >= a.spans) return;
  float* record = a.records + ((int64_t)bh * a.spans + span) * kRecord<BF16>;
  if constexpr (!BF16) record[kRowNorms + r % kSpan] = norm;
  float* rec = record + (r % kSpan >> 4) * 64 + (r & 15);
  rec[16 * kLse] = lse;
  rec[16 * kDelta] = d;
  rec[16 * kLo] = __builtin_bit_cast(float, k.lo);
  rec[16 * kHi] = __builtin_bit_cast(float, k.hi);
  if (r % kSpan != 0) return;
  if (h == 0)
    reinterpret_cast<int4*>(a.bounds)[(int64_t)b * a.spans + span] = int4{t.lo, t.hi, t.all_lo, t.all_hi};
  if constexpr (!BF16) *reinterpret_cast<float2*>(record + kSpanMost) = float2{most[0], most[1]};
}

// ---- the order of the tiles of keys ----

// Ranks them by the spans of rows that see a key of them: one workgroup a batch entry.
// Each span adds one where its keys begin and takes it off behind their end (sums of
// integers: their order does not matter), and the running sum is the tiles' work.
constexpr int kOrderThreads = 1024;
__global__ void __launch_bounds__(kOrderThreads) fa_attn_order_kernel(const AttnArgs a) {
  static_assert(kMaxOrdered == kOrderThreads, "a thread per tile");
  __shared__ __attribute__((aligned(16))) int work[kMaxOrdered + 1];
  __shared__ int sums[kOrderThreads / 64];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int4* bounds = reinterpret_cast<const int4*>(a.bounds) + (int64_t)b * a.spans;
  work[tid] = 0;
  if (tid == 0) work[kMaxOrdered] = 0;
  __syncthreads();
  for (int s = tid; s < a.spans; s += kOrderThreads) {
    const int2 k = *reinterpret_cast<const int2*>(bounds + s);
    if (k.x >= k.y) continue;
    atomicAdd(&work[k.x / kAttnKeys], 1);
    atomicAdd(&work[(k.y - 1) / kAttnKeys + 1], -1);
  }
  __syncthreads();
  int mine = work[tid];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int x = __shfl_up(mine, d);
    if (lane >= d) mine += x;
  }
  if (lane == 63) sums[tid / 64] = mine;
  __syncthreads();
  for (int i = 0; i < tid / 64; ++i) mine += sums[i];
  work[tid] = tid < a.key_tiles ? mine : -1;
  __syncthreads();
  // A tile's place: behind those with more work and the earlier ones with as much.
  if (tid >= a.key_tiles) return;
  int place = 0;
#pragma unroll 4
  for (int u = 0; u < a.key_tiles; u += 4) {
    const int4 w = *reinterpret_cast<const int4*>(work + u);
    place += (w.x > mine || (w.x == mine && u < tid)) + (w.y > mine || (w.y == mine && u + 1 < tid)) +
             (w.z > mine || (w.z == mine && u + 2 < tid)) + (w.w > mine || (w.w == mine && u + 3 < tid));
  }
  a.key_order[(int64_t)b * a.key_tiles + place] = tid;
}

// ---- scores and their gradients, four at a time ----

// A value that is the same in every lane, in a scalar register.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
// The compiler takes x as new here: it is computed before, and what is computed from
// it after, not kept in registers from outside of a loop.
template <class T>
__device__ __forceinline__ T fresh(T x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <bool CAP>
struct Grads {
  Score score;
  float slope, unit;  // slope: in units of what it is added to; unit: the factor of products
  __device__ __forceinline__ void init(const AttnArgs& a, int h) {
    score.init(a.score);
    slope = uniform(score.biased ? a.score.slopes[h] * (CAP ? kLog2e : a.score.slope_unit) : 0.0f);
    unit = uniform(a.scale_log2);
  }
  // away: from a score's row to its key.
  __device__ __forceinline__ float biased(float x, float away) const {
    return fmaf(-slope, fabsf(away), x);
  }
};

template <bool BF16>
__device__ __forceinline__ i16x8 pack8(const f32x4& x, const f32x4& y) {
  return __builtin_bit_cast(i16x8, u32x4{pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]),
                                         pack2<BF16>(y[0], y[1]), pack2<BF16>(y[2], y[3])});
}

// c[cb] = init + sum over D of the 16 rows at LDS address `at` (a lane's offset in
// it) times the 16 NCB columns held in f.
// beside(i): vector work that goes between the products, in D / 32 parts.
template <int D, bool BF16, int NCB, class Beside>
__device__ __forceinline__ void row_product(uint32_t at, const i16x8 (&f)[NCB][D / 32], const f32x4& init,
                                            f32x4 (&c)[NCB], Beside&& beside) {
  constexpr int KST = D / 32, AHEAD = KST < 3 ? KST : 3;
  i16x8 x[AHEAD];
  auto read = [&](auto i_c) FA_INLINE {
    constexpr int st = decltype(i_c)::value;
    x[st % AHEAD] = lds_read16<0>(at ^ lds::TileBoth<D>::row_step(st));
  };
  static_for<0, AHEAD>(read);
  __builtin_amdgcn_sched_barrier(0);
  static_for<0, KST>([&](auto i_c) FA_INLINE {
    constexpr int st = decltype(i_c)::value;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) c[cb] = mfma16<BF16>(x[st % AHEAD], f[cb][st], st == 0 ? init : c[cb]);
    if constexpr (st + AHEAD < KST) read(std::integral_constant<int, st + AHEAD>{});
    beside(i_c);
    __builtin_amdgcn_sched_barrier(0);
  });
}

// acc[db][cb] += the 32 rows at LDS address `at`, turned, times f[cb].
template <int D, bool BF16, int NCB>
__device__ __forceinline__ void turned_product(uint32_t at, const i16x8 (&f)[NCB], f32x4 (&acc)[D / 16][NCB]) {
  constexpr int DB = D / 16, AHEAD = 3, ROWB = 2 * D;
  i16x8 x[AHEAD];
  auto read = [&](auto i_c) FA_INLINE {
    constexpr int db = decltype(i_c)::value;
    x[db % AHEAD] = ds_read_tr_pair<0, 16 * ROWB>(at ^ lds::TileBoth<D>::turned_block(db));
  };
  static_for<0, AHEAD>(read);
  // The wave that is in these products goes first, so that the other wave's
  // exponentials fill the gaps (dk, dv of 2 x 8192 tokens, 32 heads on 8, causal, us without
  // and with: D = 128 2288 and 2214; D = 64 1652 and 1670).
  if constexpr (D == 128) __builtin_amdgcn_s_setprio(1);
  __builtin_amdgcn_sched_barrier(0);
  static_for<0, DB>([&](auto i_c) FA_INLINE {
    constexpr int db = decltype(i_c)::value;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) acc[db][cb] = mfma16<BF16>(x[db % AHEAD], f[cb], acc[db][cb]);
    if constexpr (db + AHEAD < DB) read(std::integral_constant<int, db + AHEAD>{});
    __builtin_amdgcn_sched_barrier(0);
  });
  if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
}

// A wave's sums at a lane's place in LDS, 1 KiB a register quad.
template <int DB>
__device__ __forceinline__ void put_sums(uint32_t at, const f32x4 (&x)[DB][2]) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) lds_write16(at + (2 * db + cb) * 1024, __builtin_bit_cast(u32x4, x[db][cb]));
}
template <int DB>
__device__ __forceinline__ void add_sums(uint32_t at, f32x4 (&x)[DB][2]) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) x[db][cb] += lds_quad(at + (2 * db + cb) * 1024);
}

// ---- gradients of k and v ----

// A span of rows of a head, below 0: none; `code`: the span, and whether the wave's
// keys are seen by some row, by all, and the workgroup's by all.
struct Span {
  int head;
  uint32_t code;
  __device__ __forceinline__ bool is() const { return head >= 0; }
  __device__ __forceinline__ int at() const { return (int)(code & 0x1fffffffu); }
  __device__ __forceinline__ bool seen() const { return (code >> 29) & 1; }
  __device__ __forceinline__ bool whole() const { return (code >> 30) & 1; }
  __device__ __forceinline__ bool all() const { return code >> 31; }
};

// The kernel's arguments, read where they are used: what only the ends of a loop need
// would take scalar registers all along it.
__device__ __forceinline__ const __attribute__((address_space(4))) AttnArgs& late_args() {
  auto* p = (const __attribute__((address_space(4))) AttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *p;
}

template <int D, bool BF16, bool CAP, int TEAMS>
__global__ void __launch_bounds__(256 * TEAMS) __attribute__((amdgpu_waves_per_eu(D == 128 ? 2 : 3, D == 128 ? 2 : 3)))
    fa_attn_dkv_kernel(const AttnArgs a) {
  constexpr int ROWB = 2 * D, KST = D / 32, DB = D / 16;
  constexpr int TB = kSpan * ROWB, SLOT = 2 * TB + 1024, SLOTS = 4;  // bytes: Q, go, record
  constexpr int NI = 16 * ROWB / 1024, LPR = ROWB / 16, RPI = 64 / LPR;  // copies of 16 rows
  constexpr int PART = 2 * DB * 1024;  // bytes of a wave's sums
  constexpr int RINGS = TEAMS * SLOTS * SLOT, SUMS = (TEAMS - 1) * 2 * 4 * PART;
  __shared__ __attribute__((aligned(1024))) char smem[RINGS > SUMS ? RINGS : SUMS];
  __shared__ __attribute__((aligned(16))) struct {
    float spoiled[SLOTS][2][kSpan];  // NaN for rows of Q, of go with an infinity or NaN, else 0
    // of a wave's keys: dS's factors, |v|; the largest of their products, of the factors
    float factor[BF16 ? 0 : 4][2][32], largest[BF16 ? 0 : 4][2];
  } aside[TEAMS];

  const int lane = threadIdx.x & 63;
  const int team = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;  // of its team
  // The first keys first: a causal mask's longest.
  int unit, within;
  if (!unit_and_place(a.cols, unit, within)) return;
  const int place = fast_div(within, a.by_splits), split = within - place * a.splits;
  const int b = fast_div(unit, a.by_kvh), kvh = unit - b * a.kv_heads, h0 = kvh * a.group;
  const int tile = a.key_order != nullptr ? uniform(a.key_order[(int64_t)b * a.key_tiles + place]) : place;
  const int j0 = tile * kAttnKeys, w0 = j0 + 32 * wave;

  f32x4 gk[DB][2], gv[DB][2];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) gk[db][cb] = gv[db][cb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // The spans with a row that sees a key of the workgroup, of the split's (every
  // splits-th, so that the splits of a causal mask are alike), head after head, the
  // last ones first: those are a causal mask's that all tiles of keys have, and are
  // read from L2 by all but one.  Bit i of `hit` is span at0 + i.  Each turn takes one for
  // each team; `any`: there was one for the first.
  const int spans = a.spans, group = a.group, last0 = (spans - 1) & ~63;
  uint64_t hit = 0, seen = 0, whole = 0, all = 0;
  int h = 0, at0 = last0 + 64;
  auto next = [&](bool& any) FA_INLINE -> Span {
    Span mine = {-1, 0};
    any = false;
#pragma unroll 1
    for (int e = 0; e < TEAMS; ++e) {
      while (hit == 0) {
        at0 -= 64;
        if (at0 < 0) {
          if (h + 1 >= group) {
            at0 = 0;  // (and none next time)
            return mine;
          }
          ++h;
          at0 = last0;
        }
        const auto& x = late_args();
        const int s = at0 + lane_now();
        int4 k = {kNoKey, 0, kNoKey, 0};
        if (s < spans) k = reinterpret_cast<const int4*>(x.bounds)[(int64_t)b * spans + s];
        const bool of_split = s - fast_div(s, FastDiv{x.by_splits.mul, x.by_splits.shift}) * x.splits == split;
        hit = __ballot(of_split && k.x < j0 + kAttnKeys && k.y > j0);
        seen = __ballot(k.x < w0 + 32 && k.y > w0);
        whole = __ballot(k.z <= w0 && k.w >= w0 + 32);
        all = __ballot(k.z <= j0 && k.w >= j0 + kAttnKeys);
      }
      const int i = 63 - __builtin_clzll(hit);
      hit ^= 1ull << i;
      any = true;
      if (e == team)
        mine = Span{h, (uint32_t)(at0 + i) | (uint32_t)((seen >> i) & 1) << 29 | (uint32_t)((whole >> i) & 1) << 30 |
                           (uint32_t)((all >> i) & 1) << 31};
    }
    return mine;
  };

  // Staging: waves 0 and 1 copy 16 rows of Q each, 2 and 3 of go; wave 0 the record.
  // (The swizzle of row i + r is that of i, exclusive or that of r.)
  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(smem)) + team * SLOTS * SLOT;
  const bool of_go = wave >= 2;
  const int sr = (wave & 1) * 16;  // this wave's first row
  const Rows3& sx = of_go ? a.go : a.q;
  const uint32_t sst = (uint32_t)sx.st, sto = (of_go ? TB : 0) + sr * ROWB;
  const char* sp = sx.p + b * sx.sb + h0 * sx.sh + sr * (int64_t)sst;  // of the head to come
  const char* records = reinterpret_cast<const char*>(a.records + ((int64_t)b * a.heads + h0) * spans * kRecord<BF16>);
  const int64_t head_step = sx.sh;
  const int row_end = a.n - 1 - sr;
  int staged_head = 0;
  const uint32_t src_row = (lane / LPR) * sst, src_chunk = ((lane % LPR) ^ lds::TileBoth<D>::swz(lane / LPR)) * 16;
  auto issue = [&](const Span& x, uint32_t slot) FA_INLINE {
    for (; staged_head < x.head; ++staged_head) {
      sp += head_step;
      records += (int64_t)spans * (kRecord<BF16> * 4);
    }
    const int row = x.at() * kSpan;  // (less sr)
    const uint32_t dst = base + slot * SLOT + sto;
    const char* from = sp + (int64_t)row * sst;
    if (row + 15 <= row_end) {
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        poison_1k(dst + it * 1024);
        dma_16b(src_row + it * RPI * sst + (src_chunk ^ (lds::TileBoth<D>::swz(it * RPI) * 16)), from, dst + it * 1024);
      }
    } else {  // rows past the last one re-read it
      const int l = lane_now(), back = max(0, row - row_end);
#pragma unroll
      for (int it = 0; it < NI; ++it) {
        poison_1k(dst + it * 1024);
        const int r = it * RPI + l / LPR, c = (l % LPR) ^ lds::TileBoth<D>::swz(r);
        dma_16b(min(r, row_end - row + back) * sst + c * 16, from - (int64_t)back * sst, dst + it * 1024);
      }
    }
    if (wave == 0) {  // (1 KiB: the next record too, or what is behind the last one)
      poison_1k(base + slot * SLOT + 2 * TB);
      dma_16b(lane_now() * 16, records + (int64_t)x.at() * (kRecord<BF16> * 4), base + slot * SLOT + 2 * TB);
    }
  };
  // The copies of a span are there, `later`: but for those of one issued after it.
  // If the span is not seen whole, this wave cleans the rows that it has copied.
  const uint32_t spoiled_at = __builtin_amdgcn_readfirstlane(lds_addr(aside)) + team * (int)sizeof(aside[0]);
  auto finish = [&](const Span& x, uint32_t slot, bool later) FA_INLINE {
    if (!later)
      wait_vmcnt<0>();
    else if (wave == 0)
      wait_vmcnt<NI + 1>();
    else
      wait_vmcnt<NI>();
    if (x.is() && !x.all()) {
      const unsigned bad = clean_rows<D, BF16, 16>(base + slot * SLOT + sto);
      const int l = lane_now();
      if (l < 16)
        lds_write4(spoiled_at + (slot * 2 + (of_go ? 1 : 0)) * kSpan * 4 + (sr + l) * 4, (bad >> l) & 1 ? NAN : 0.0f);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __syncthreads();
  };

  // Two spans are on their way while one is computed.
  bool now_any, then_any = false;
  Span now = next(now_any), then = {-1, 0};
  uint32_t slot = 0;
  int head = -1;
  if (now_any) {
    if (now.is()) issue(now, 0);
    then = next(then_any);
    if (then.is()) issue(then, 1);
  }
  i16x8 kf[2][KST], vf[2][KST];
#pragma unroll
  for (int cb = 0; cb < 2; ++cb) {
    const int64_t j = min(w0 + 16 * cb + (lane & 15), a.m - 1);
    const char* kp = a.k.p + b * a.k.sb + kvh * a.k.sh + j * a.k.st + (lane >> 4) * 16;
    const char* vp = a.v.p + b * a.v.sb + kvh * a.v.sh + j * a.v.st + (lane >> 4) * 16;
#pragma unroll
    for (int st = 0; st < KST; ++st) {
      kf[cb][st] = *reinterpret_cast<const i16x8*>(kp + 64 * st);
      vf[cb][st] = *reinterpret_cast<const i16x8*>(vp + 64 * st);
    }
  }
  // (each wave its own keys', in its order: no barrier)
  auto factor_at = [&](int l) FA_INLINE { return spoiled_at + SLOTS * 2 * kSpan * 4 + (w0 & 96) * 8 + l * 4; };
  auto largest_at = [&]() FA_INLINE { return spoiled_at + (SLOTS * 2 * kSpan + 4 * 64) * 4 + (w0 & 96) / 4; };
  if constexpr (!BF16) {
    // (more than any bound above 2^-57 takes; behind the last key one that every bound fits)
    constexpr float first = kBoundMost<CAP> * 0x1p57f;
    if (lane < 32) lds_write4(factor_at(lane), w0 + lane < a.m ? first : 0x1p-60f);
    lds_write8<0>(largest_at(), u32x2{__builtin_bit_cast(uint32_t, first), __builtin_bit_cast(uint32_t, first)});
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      float square = 0.0f;
#pragma unroll
      for (int st = 0; st < KST; ++st) {
        const u32x4 x = __builtin_bit_cast(u32x4, vf[cb][st]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t word = x[j];  // (bit_cast of an element itself takes the first one)
          const auto pair = __builtin_bit_cast(f16x2, word);
          square = __builtin_amdgcn_fdot2(pair, pair, square, false);
        }
      }
      square += from_lane(square, lane ^ 16);
      square += from_lane(square, lane ^ 32);
      if (lane < 16) lds_write4(factor_at(32 + 16 * cb + lane), square < INFINITY ? sqrtf(square) : 0.0f);
    }
  }
  finish(now, 0, false);  // (what was loaded so far: no wait for it later, which would be one for copies too)

  Grads<CAP> grads;
  // fp16: new factors of dS, also for what its sum holds, where rows that see a key take its bound
  // further than those before.  (2 x 8192 causal rows, 32 heads on 8, us without any look and with one at each
  // span: D = 64 1362 and 1445, D = 128 1997 and 2077; one at 64 spans where their limits are read costs
  // as much.)
  auto fit = [&](uint32_t record, bool masked) FA_INLINE {
    const int l = lane_now(), key0 = w0 + (l & 15);
    const uint32_t at = factor_at(l & 15);
    const float v[2] = {lds_read4(at + 128), lds_read4(at + 192)};
    float bound[2] = {0.0f, 0.0f}, largest[2] = {0.0f, 0.0f};
    if (masked) {
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        const uint32_t quad = record + rb * 256 + (l >> 4) * 16;
        const i32x4 lo = __builtin_bit_cast(i32x4, lds_quad(quad + 64 * kLo)) - key0;
        const i32x4 hi = __builtin_bit_cast(i32x4, lds_quad(quad + 64 * kHi)) - key0;
        const f32x4 go = lds_quad(record + 4 * kRowNorms + rb * 64 + (l >> 4) * 16), delta = lds_quad(quad + 64 * kDelta);
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            bound[cb] =
                fmaxf(bound[cb], 16 * cb >= lo[i] && 16 * cb < hi[i] ? fmaf(go[i], v[cb], fabsf(delta[i])) : 0.0f);
      }
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) {
        bound[cb] = fmaxf(bound[cb], from_lane(bound[cb], lane_now() ^ 16));
        bound[cb] = fmaxf(bound[cb], from_lane(bound[cb], lane_now() ^ 32));
      }
    } else {
      const float go = lds_read4(record + 4 * kSpanMost), delta = lds_read4(record + 4 * kSpanMost + 4);
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) bound[cb] = fmaf(go, v[cb], delta);
    }
    const float factors[2] = {lds_read4(at), lds_read4(at + 64)};
    // (that keys which no row has seen yet have the first factor made it look)
    if (!__any(bound[0] * factors[0] > kBoundMost<CAP> || bound[1] * factors[1] > kBoundMost<CAP>)) return;
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      const float factor = factors[cb];
      const float to = bound[cb] * factor > kBoundMost<CAP> ? grad_factor<CAP>(bound[cb]) : factor;
      // (their ratio: powers of two; 0 if it is less than there is)
      const float change =
          __builtin_bit_cast(float, max(__builtin_bit_cast(int, to) - __builtin_bit_cast(int, factor) + 0x3f800000, 0));
#pragma unroll
      for (int db = 0; db < DB; ++db) gk[db][cb] *= change;
      lds_write4(at + 64 * cb, to);
      largest[0] = fmaxf(largest[0], v[cb] * to);
      largest[1] = fmaxf(largest[1], to);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      static_for<0, 4>([&](auto d_c) FA_INLINE {
        largest[i] = fmaxf(largest[i], turned_row<1 << decltype(d_c)::value>(largest[i]));
      });
      lds_write4(largest_at() + 4 * i, largest[i]);
    }
  };
  // A span in `slot`; `masked`: some row does not see all of the wave's keys, `cleaned`: of
  // the workgroup's (finish).  (Scores become P in place, dS takes the place of go V^T: the
  // accumulators leave few registers, none to keep addresses across spans.)
  auto step = [&](int row0, uint32_t slot, bool masked, bool cleaned) FA_INLINE {
    const int l = lane_now();
    const int key0 = w0 + (l & 15);
    const uint32_t tile = base + slot * SLOT;
    u32x4 pw[2], dw[2];  // P and dS as packed pairs: words 0, 1 of rows 4 (l / 16) .., 2, 3 of those 16 on
    u32x2 most, largest;  // (read ahead of the first product)
    if constexpr (!BF16) {
      most = lds_read8<4 * kSpanMost>(tile + 2 * TB);
      largest = lds_read8<0>(largest_at());
    }
    static_for<0, 2>([&](auto rb_c) FA_INLINE {
      constexpr int rb = decltype(rb_c)::value;
      const uint32_t rows = tile + rb * 16 * ROWB + lds::TileBoth<D>::row_offset(l);
      const uint32_t quad = tile + 2 * TB + rb * 256 + (l >> 4) * 16;
      f32x4 c[2], e[2];
      const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
      row_product<D, BF16, 2>(rows, kf, zero, c, [](auto) FA_INLINE {});
      if constexpr (!BF16 && rb == 0) {
        auto f = [](uint32_t x) FA_INLINE { return __builtin_bit_cast(float, x); };
        if (__builtin_expect(__any(fmaf(f(most[0]), f(largest[0]), f(most[1]) * f(largest[1])) > kBoundMost<CAP>), false))
          fit(tile + 2 * TB, masked);
      }
      const int away = row0 + 16 * rb + 4 * (l >> 4) + a.m - a.n - key0;  // of key block 0
      auto away_of = [&](int cb, int i) FA_INLINE { return (float)(away - 16 * cb) + (float)i; };
      f32x4 lse = lds_quad(quad + 64 * kLse);
      if (cleaned) {
        const uint32_t bad = spoiled_at + slot * 2 * kSpan * 4 + rb * 64 + (l >> 4) * 16;
        lse += lds_quad(bad) + lds_quad(bad + kSpan * 4);
      }
      if (!CAP && grads.score.biased)
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
#pragma unroll
          for (int i = 0; i < 4; ++i) c[cb][i] = grads.biased(c[cb][i], away_of(cb, i));
      // The exponentials, or the first ones of capped scores, beside go V^T.
      float factor[2];  // (read late: registers)
      auto read_factor = [&]() FA_INLINE {
        if constexpr (BF16) return;
        const uint32_t at = factor_at(lane_now() & 15);
        factor[0] = lds_read4(at);
        factor[1] = lds_read4(at + 64);
      };
      row_product<D, BF16, 2>(rows + TB, vf, lds_quad(quad + 64 * kDelta), e, [&](auto i_c) FA_INLINE {
        constexpr int PART = 8 / KST;
        if constexpr (!CAP && decltype(i_c)::value == KST - 1) read_factor();
#pragma unroll
        for (int j = 0; j < PART; ++j) {
          const int at = decltype(i_c)::value * PART + j;
          const float x = c[at / 4][at % 4];
          c[at / 4][at % 4] = CAP ? grads.score.tail(x) : fast_exp2(fmaf(x, grads.unit, -lse[at % 4]));
        }
      });
      if constexpr (CAP) {
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float t = c[cb][i];
            e[cb][i] *= fmaf(-t, t, t);
            c[cb][i] = fmaf(-grads.score.twice, t, -lse[i]);
          }
        if (grads.score.biased)
#pragma unroll
          for (int cb = 0; cb < 2; ++cb)
#pragma unroll
            for (int i = 0; i < 4; ++i) c[cb][i] = grads.biased(c[cb][i], away_of(cb, i));
        read_factor();
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
#pragma unroll
          for (int i = 0; i < 4; ++i) c[cb][i] = fast_exp2(c[cb][i]);
      }
#pragma unroll
      for (int cb = 0; cb < 2; ++cb)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[cb][i] *= BF16 ? c[cb][i] : c[cb][i] * factor[cb];
      if (masked) {
        const i32x4 lo = __builtin_bit_cast(i32x4, lds_quad(quad + 64 * kLo)) - key0;
        const i32x4 hi = __builtin_bit_cast(i32x4, lds_quad(quad + 64 * kHi)) - key0;
#pragma unroll
        for (int cb = 0; cb < 2; ++cb)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * cb < lo[i] || 16 * cb >= hi[i]) c[cb][i] = e[cb][i] = 0.0f;
      }
#pragma unroll
      for (int cb = 0; cb < 2; ++cb) {
        // (kept: the compiler would pack at the end and hold all until then)
        pw[cb][2 * rb] = fresh(pack2<BF16>(c[cb][0], c[cb][1]));
        pw[cb][2 * rb + 1] = fresh(pack2<BF16>(c[cb][2], c[cb][3]));
        dw[cb][2 * rb] = fresh(pack2<BF16>(e[cb][0], e[cb][1]));
        dw[cb][2 * rb + 1] = fresh(pack2<BF16>(e[cb][2], e[cb][3]));
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    const uint32_t turned = tile + lds::TileBoth<D>::turned_offset(lane_now());
    const i16x8 pf[2] = {__builtin_bit_cast(i16x8, pw[0]), __builtin_bit_cast(i16x8, pw[1])};
    const i16x8 df[2] = {__builtin_bit_cast(i16x8, dw[0]), __builtin_bit_cast(i16x8, dw[1])};
    turned_product<D, BF16, 2>(turned + TB, pf, gv);
    turned_product<D, BF16, 2>(turned, df, gk);
  };

  while (now_any) {
    Span last = {-1, 0};
    bool last_any = false;
    if (then_any) last = next(last_any);
    if (last.is()) issue(last, (slot + 2) % SLOTS);
    if (now.is() && now.seen()) {
      if (now.head != head) {
        head = now.head;
        grads.init(a, h0 + head);
      }
      step(now.at() * kSpan, slot, !now.whole(), !now.all());
    }
    slot = (slot + 1) % SLOTS;
    finish(then, slot, last.is());
    now = then;
    then = last;
    now_any = then_any;
    then_any = last_any;
  }

  // (powers of two but for the scale)
  if constexpr (!BF16) {
    const uint32_t at = factor_at(lane_now() & 15);
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      const float back = 1.0f / lds_read4(at + cb * 64);
#pragma unroll
      for (int db = 0; db < DB; ++db) gk[db][cb] *= back;
    }
  }
  // The first team takes all of gk, the second all of gv, by wave and lane.
  if constexpr (TEAMS > 1) {
    const uint32_t at = lds_addr(smem) + wave * PART + lane_now() * 16;
    if (team != 0) put_sums<DB>(at + (team - 1) * 4 * PART, gk);
    if (team != 1) put_sums<DB>(at + (TEAMS - 1 + (team == 0 ? 0 : team - 1)) * 4 * PART, gv);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __syncthreads();
    if (team > 1) return;
#pragma unroll
    for (int i = 0; i < TEAMS - 1; ++i) {
      if (team == 0) add_sums<DB>(at + i * 4 * PART, gk);
      if (team == 1) add_sums<DB>(at + (TEAMS - 1 + i) * 4 * PART, gv);
    }
  }
  const bool has_k = TEAMS == 1 || team == 0, has_v = TEAMS == 1 || team == 1;

  const auto& x = late_args();
  const float fv[2] = {fast_exp2(-kShift<BF16>), fast_exp2(-kShift<BF16>)};
  const float scale = kQuarters<CAP> * x.scale * fv[0], fk[2] = {scale, scale};
  const int l = lane_now(), m = x.m;
  if (x.parts != nullptr) {
    const int64_t rows = (int64_t)x.batch * x.kv_heads * m;
    float* to = x.parts + ((int64_t)split * rows + (int64_t)unit * m) * 2 * D + 4 * (l >> 4);
#pragma unroll
    for (int cb = 0; cb < 2; ++cb) {
      const int j = w0 + 16 * cb + (l & 15);
      if (j >= m) continue;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        if (has_k) *reinterpret_cast<f32x4*>(to + (int64_t)j * 2 * D + 16 * db) = gk[db][cb] * fk[0];
        if (has_v) *reinterpret_cast<f32x4*>(to + (int64_t)j * 2 * D + D + 16 * db) = gv[db][cb] * fv[0];
      }
    }
    return;
  }
  // (of the sums, what this wave has read)
  char* ot = smem + wave * PART + (TEAMS > 1 && team == 1 ? (TEAMS - 1) * 4 * PART : 0);
  char* kp = x.gk.p + b * x.gk.sb + kvh * x.gk.sh;
  char* vp = x.gv.p + b * x.gv.sb + kvh * x.gv.sh;
  const int64_t k_st = x.gk.st, v_st = x.gv.st;
  if (has_k) write_rows<D, BF16>(ot, gk, fk, l, [&](int r) FA_INLINE -> char* { return w0 + r < m ? kp + (w0 + r) * k_st : nullptr; });
  if (has_v) write_rows<D, BF16>(ot, gv, fv, l, [&](int r) FA_INLINE -> char* { return w0 + r < m ? vp + (w0 + r) * v_st : nullptr; });
}

// Adds the splits' parts in their order: 8 elements a thread.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) fa_attn_join_kernel(const AttnArgs a) {
  constexpr int TPR = 2 * D / 8;  // threads of a key
  const int64_t rows = (int64_t)a.batch * a.kv_heads * a.m;
  const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;
  const int d = (int)threadIdx.x % TPR * 8;
  f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x;
  for (int s = 0; s < a.splits; ++s) {
    const float* from = a.parts + (s * rows + row) * 2 * D + d;
    x += *reinterpret_cast<const f32x4*>(from);
    y += *reinterpret_cast<const f32x4*>(from + 4);
  }
  const int64_t unit = row / a.m, j = row - unit * a.m;
  const int64_t b = unit / a.kv_heads, kvh = unit - b * a.kv_heads;
  const Rows3& to = d < D ? a.gk : a.gv;
  *reinterpret_cast<i16x8*>(to.p + b * to.sb + kvh * to.sh + j * to.st + (d % D) * 2) = pack8<BF16>(x, y);
}

// ---- gradients of q ----

// D = 64 has registers for three waves of a SIMD unit: 2 x 8192 rows, 32 heads on 8, causal,
// fp16, 1060 us with two and 930 with three.
template <int D, bool BF16, bool CAP, int TEAMS>
__global__ void __launch_bounds__(256 * TEAMS)
    __attribute__((amdgpu_waves_per_eu(D == 64 && TEAMS == 1 ? 3 : 2, D == 64 && TEAMS == 1 ? 3 : 2)))
    fa_attn_dq_kernel(const AttnArgs a) {
  constexpr int ROWB = 2 * D, TB = 64 * ROWB, KST = D / 32, DB = D / 16;
  __shared__ __attribute__((aligned(1024))) char smem[TEAMS * 4 * TB];  // of each team K0 V0 K1 V1
  // fp16: some row's sum is no number, which rows', the rows' factors then
  __shared__ int again, odd[BF16 ? 1 : kAttnRows];
  __shared__ float least[BF16 ? 1 : kAttnRows];

  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = lane >> 4;
  const int team = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;  // of its team
  int unit, within;
  if (!unit_and_place(a.rows, unit, within)) return;
  const int back = fast_div(within, a.by_group);
  const int b = fast_div(unit, a.by_kvh), kvh = unit - b * a.kv_heads;
  const int h = kvh * a.group + within - back * a.group;
  const int row0 = (a.tiles - 1 - back) * kAttnRows, wrow0 = row0 + 32 * wave;

  TileKeys keys, all;  // of the wave's rows, of the workgroup's
  tile_keys(a, b, row0, wave, keys, all);
  const int c0 = all.lo, c1 = all.hi;
  // (tile t TEAMS + team is the team's in turn t)
  const int turns = c0 < c1 ? ((c1 - c0 + 63) / 64 + TEAMS - 1) / TEAMS : 0;
  auto key_of = [&](int t) FA_INLINE { return c0 + 64 * (t * TEAMS + team); };
  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(smem)) + team * 4 * TB;
  const char* kh = a.k.p + b * a.k.sb + kvh * a.k.sh;
  const char* vh = a.v.p + b * a.v.sb + kvh * a.v.sh;
  RowStage<D> stage_k;
  RowStage<D> stage_v;
  stage_k.init(lane, (uint32_t)a.k.st);
  stage_v.init(lane, (uint32_t)a.v.st);
  auto issue = [&](int t, int buf) FA_INLINE {
    if (t >= turns || key_of(t) >= c1) return;
    const int r0 = min(key_of(t) + 16 * wave, c1 - 1);
    const uint32_t dst = base + buf * 2 * TB + wave * 16 * ROWB;
    stage_k.copy(kh + r0 * a.k.st, dst, c1 - 1 - r0, (uint32_t)a.k.st);
    stage_v.copy(vh + r0 * a.v.st, dst + TB, c1 - 1 - r0, (uint32_t)a.v.st);
  };
  issue(0, 0);
  if constexpr (!BF16) {  // (ordered by the first barrier)
    if (threadIdx.x == 0) again = 0;
    if (threadIdx.x < kAttnRows) odd[threadIdx.x] = 0;
  }
  // (behind the first copies: one wait for all)
  i16x8 qf[2][KST], gf[2][KST];
  float lse[2], delta[2], factor[2];  // (minus delta)
  RowKeys see[2];
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const int r = min(wrow0 + 16 * rb + l16, a.n - 1);
    const int64_t i = r;
    const char* qp = a.q.p + b * a.q.sb + h * a.q.sh + i * a.q.st + 16 * g4;
    const char* gp = a.go.p + b * a.go.sb + h * a.go.sh + i * a.go.st + 16 * g4;
#pragma unroll
    for (int st = 0; st < KST; ++st) {
      qf[rb][st] = *reinterpret_cast<const i16x8*>(qp + 64 * st);
      gf[rb][st] = *reinterpret_cast<const i16x8*>(gp + 64 * st);
    }
    const float* record = a.records + (((int64_t)b * a.heads + h) * a.spans + r / kSpan) * kRecord<BF16>;
    const float* rec = record + r % kSpan / 16 * 64 + r % 16;
    lse[rb] = rec[16 * kLse];
    delta[rb] = rec[16 * kDelta];
    see[rb].lo = __builtin_bit_cast(int, rec[16 * kLo]);
    see[rb].hi = __builtin_bit_cast(int, rec[16 * kHi]);
    factor[rb] = 1.0f;
    if constexpr (!BF16) {
      const float norm = record[kRowNorms + r % kSpan];
      factor[rb] = grad_factor<CAP>(fmaf(norm, 0x1p6f, fabsf(delta[rb])));
      least[32 * wave + 16 * rb + l16] = grad_factor<CAP>(fmaf(norm, 0x1p20f, fabsf(delta[rb])));
    }
  }
  // The staged keys of tile t are there: cleaned if some row does not see all of
  // them, with V's rows set to NaN for the ones that do.
  auto finish = [&](int t, int buf) FA_INLINE {
    __builtin_amdgcn_s_waitcnt(0);
    const int k0 = key_of(t);
    if (t < turns && k0 < c1 && !(k0 >= all.all_lo && k0 + 64 <= all.all_hi)) {
      const uint32_t rows = base + buf * 2 * TB + wave * 16 * ROWB;
      const unsigned bad = clean_rows<D, BF16, 16>(rows);
      if (__builtin_expect(bad != 0, false)) {
        constexpr int LPR = ROWB / 16;
        const int l = lane_now();
        for (int r = l / LPR; r < 16; r += 64 / LPR)
          if ((bad >> r) & 1) lds_write16(rows + TB + r * ROWB + l % LPR * 16, u32x4{~0u, ~0u, ~0u, ~0u});
      }
      __builtin_amdgcn_s_waitcnt(0);
    }
    __syncthreads();
  };

  f32x4 gq[DB][2];
  const uint32_t row_at = base + lds::TileBoth<D>::row_offset(lane);
  const uint32_t turned_at = base + lds::TileBoth<D>::turned_offset(lane);
  Grads<CAP> grads;
  grads.init(a, h);
  const int ahead = a.m - a.n;

  // 32 keys from k0, in half `half` of the tile.
  auto step = [&](int k0, int off, int half, bool masked) FA_INLINE {
    const uint32_t rows = row_at + off + half * 32 * ROWB;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 s[2][2], dp[2][2];
    const int key0 = k0 + 4 * g4;
    auto away_of = [&](int rb, int kb, int i) FA_INLINE {
      return (float)(key0 + 16 * kb - (min(wrow0 + 16 * rb + l16, a.n - 1) + ahead)) + (float)i;
    };
    // The exponentials of a product, or the first ones of capped scores, beside the next.
    auto none = [](auto) FA_INLINE {};
    auto bias = [&](int kb) FA_INLINE {
      if (!CAP && grads.score.biased)
#pragma unroll
        for (int rb = 0; rb < 2; ++rb)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kb][rb][i] = grads.biased(s[kb][rb][i], away_of(rb, kb, i));
    };
    auto part = [&](auto kb_c) FA_INLINE {
      return [&](auto i_c) FA_INLINE {
        constexpr int PART = 8 / KST, kb = decltype(kb_c)::value;
#pragma unroll
        for (int j = 0; j < PART; ++j) {
          const int at = decltype(i_c)::value * PART + j;
          const float x = s[kb][at / 4][at % 4];
          s[kb][at / 4][at % 4] = CAP ? grads.score.tail(x) : fast_exp2(fmaf(x, grads.unit, -lse[at / 4]));
        }
      };
    };
    row_product<D, BF16, 2>(rows, qf, zero, s[0], none);
    bias(0);
    row_product<D, BF16, 2>(rows + 16 * ROWB, qf, zero, s[1], part(std::integral_constant<int, 0>{}));
    bias(1);
    row_product<D, BF16, 2>(rows + TB, gf, zero, dp[0], part(std::integral_constant<int, 1>{}));
    row_product<D, BF16, 2>(rows + TB + 16 * ROWB, gf, zero, dp[1], none);
    i16x8 df[2];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      auto each = [&](auto&& fn) FA_INLINE {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[kb][rb][i] = fn(s[kb][rb][i], kb, i);
      };
      if constexpr (CAP) {
        each([&](float x, int kb, int i) FA_INLINE {
          dp[kb][rb][i] = (dp[kb][rb][i] + delta[rb]) * fmaf(-x, x, x);
          return fmaf(-grads.score.twice, x, -lse[rb]);
        });
        if (grads.score.biased)
          each([&](float x, int kb, int i) FA_INLINE { return grads.biased(x, away_of(rb, kb, i)); });
      }
      each([&](float x, int kb, int i) FA_INLINE {
        float p = x;
        if constexpr (CAP)
          p = fast_exp2(x);
        else
          dp[kb][rb][i] += delta[rb];
        if constexpr (!BF16) p *= factor[rb];
        return p * dp[kb][rb][i];
      });
      if (masked)
        each([&](float x, int kb, int i) FA_INLINE {
          const int key = key0 + 16 * kb + i;
          return key >= see[rb].lo && key < see[rb].hi ? x : 0.0f;
        });
      df[rb] = pack8<BF16>(s[0][rb], s[1][rb]);
    }
    turned_product<D, BF16, 2>(turned_at + off + half * 32 * ROWB, df, gq);
  };

#pragma unroll 1
  for (bool last = BF16;;) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) gq[db][rb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    finish(0, 0);
    int buf = 0;
    for (int t = 0; t < turns; ++t, buf ^= 1) {
      const int k0 = key_of(t);
      issue(t + 1, buf ^ 1);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = k0 + 32 * half;
        if (k >= keys.all_lo && k + 32 <= keys.all_hi)
          step(k, buf * 2 * TB, half, false);
        else if (k < keys.hi && k + 32 > keys.lo)
          step(k, buf * 2 * TB, half, true);
      }
      finish(t + 1, buf ^ 1);
    }
    if (last) break;
    // (all start again: the staging is shared, and teams have the same factors)
    last = true;
    const int at = 32 * wave + (lane_now() & 15);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      bool no = false;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) no = no || !(fabsf(gq[db][rb][i]) < INFINITY);
      if (no) again = odd[at + 16 * rb] = 1;
    }
    __syncthreads();
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(again) == 0, true)) break;
    issue(0, 0);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
      if (odd[at + 16 * rb] != 0) factor[rb] = least[at + 16 * rb];
  }

  // The second team hands its sums to the first, by wave and lane.
  constexpr int PART = 2 * DB * 1024;
  if constexpr (TEAMS == 2) {
    const uint32_t at = lds_addr(smem) + wave * PART + lane_now() * 16;
    if (team == 1) put_sums<DB>(at, gq);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __syncthreads();
    if (team == 1) return;
    add_sums<DB>(at, gq);
  }
  float f[2];
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) f[rb] = kQuarters<CAP> * a.scale * fast_exp2(-kShift<BF16>) / factor[rb];
  char* qh = a.gq.p + b * a.gq.sb + h * a.gq.sh;
  write_rows<D, BF16>(smem + wave * PART, gq, f, lane_now(), [&](int r) FA_INLINE -> char* {
    return wrow0 + r < a.n ? qh + (wrow0 + r) * a.gq.st : nullptr;
  });
}

template <class F>
hipError_t launch(F* fn, int64_t grid, int threads, const AttnArgs& a, hipStream_t stream) {
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  void* kargs[] = {const_cast<AttnArgs*>(&a)};
  return hipLaunchKernel(reinterpret_cast<const void*>(fn), dim3((unsigned)grid), dim3(threads), kargs, 0, stream);
}

template <int D, bool BF16, bool CAP>
hipError_t launch_dkv(const AttnArgs& a, hipStream_t stream) {
  constexpr int TEAMS = key_teams(D);
  const int64_t grid = grid_size(a.cols);
  return a.key_teams == 1 ? launch(&fa_attn_dkv_kernel<D, BF16, CAP, 1>, grid, 256, a, stream)
                          : launch(&fa_attn_dkv_kernel<D, BF16, CAP, TEAMS>, grid, 256 * TEAMS, a, stream);
}
template <int D, bool BF16, bool CAP>
hipError_t launch_dq(const AttnArgs& a, hipStream_t stream) {
  const int64_t grid = grid_size(a.rows);
  return a.row_teams == 1 ? launch(&fa_attn_dq_kernel<D, BF16, CAP, 1>, grid, 256, a, stream)
                          : launch(&fa_attn_dq_kernel<D, BF16, CAP, 2>, grid, 512, a, stream);
}

template <int D, bool BF16>
hipError_t launch_as(const AttnArgs& a, hipStream_t stream) {
  hipError_t e = launch(&fa_attn_rows_kernel<D, BF16>, (int64_t)a.batch * a.heads * ((a.n + kRowsBlock - 1) / kRowsBlock),
                        256, a, stream);
  if (e != hipSuccess) return e;
  if (a.key_order != nullptr) {
    e = launch(&fa_attn_order_kernel, a.batch, kOrderThreads, a, stream);
    if (e != hipSuccess) return e;
  }
  const bool cap = a.score.cap > 0.0f;
  e = cap ? launch_dkv<D, BF16, true>(a, stream) : launch_dkv<D, BF16, false>(a, stream);
  if (e != hipSuccess) return e;
  if (a.parts != nullptr) {
    const int64_t rows = (int64_t)a.batch * a.kv_heads * a.m;
    e = launch(&fa_attn_join_kernel<D, BF16>, (rows * (2 * D / 8) + 255) / 256, 256, a, stream);
    if (e != hipSuccess) return e;
  }
  return cap ? launch_dq<D, BF16, true>(a, stream) : launch_dq<D, BF16, false>(a, stream);
}

}  // namespace

hipError_t launch_attn_bwd(const AttnArgs& a, int head_dim, bool bf16, hipStream_t stream) {
  if (head_dim == 128) return bf16 ? launch_as<128, true>(a, stream) : launch_as<128, false>(a, stream);
  return bf16 ? launch_as<64, true>(a, stream) : launch_as<64, false>(a, stream);
}

}  // namespace fa
