// Key weights and eviction of a paged key/value cache on gfx950.
//
// Key weights: add_j = sum over rows i that see key j of
// exp(scale q_i.k_j - lse_i), one pass over K.  fa_weights_few_kernel takes the
// sequences of at most 32 rows and is bound by reading K.  fa_weights_kernel:
// a wave keeps 64 keys in registers as the B operand of v_mfma_f32_16x16x32 and
// the workgroup's four waves (256 keys) walk over the rows together, 64 at a
// time through LDS; a lane holds one key of each 16-key block and 4 rows, so
// its sums stay in registers and meet once at the end.  It is bound by the
// vector unit: per row and key one exponential (a quarter of the rate), one
// multiply-add and one add, 24 cycles of a SIMD per 64 of them, beside half
// the matrix work of attention.  4096 tokens over 32768 keys, fp16, 32 heads on
// 8, D = 128: 1078 us, 956 TFLOP/s; 1000 tokens over 8192 keys, 16 heads on 4:
// 43 us, of which a third are launches and the start of three workgroups per CU.
//
// fa_select_kernel: the keep - recent heaviest of a head's keys by a radix
// search for their least weight (digits of 11, 11 and 10 bits), and the list of
// the kept keys in order.  fa_move_kernel copies their rows, and counts them
// for the new lengths: bound by memory.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "fa_cache_kernels.h"
#include "fa_device_ops.h"
#include "fa_lds_layout.h"
#include "fa_paged_ops.h"

namespace fa {
namespace {

using namespace dev;

constexpr float kLog2e = 1.4426950408889634f;

template <int D, bool BF16>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3)))
    fa_weights_kernel(const PagedWeightsArgs a) {
  constexpr int ROWB = 2 * D, KST = D / 32, KB = 4, RT = 64;  // 64 keys of a wave, rows of a tile
  constexpr int TB = RT * ROWB, NI = TB / 4 / 1024;           // bytes of a row tile, DMAs of a wave
  constexpr int LPR = ROWB / 16;
  __shared__ __attribute__((aligned(1024))) char smem[2 * TB];
  __shared__ float neg_lse[4][RT];  // of each wave's current row tile

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  // (sequence, kv head, key tile or pair of them, row split): the splits slowest
  const int rest = fast_div(blockIdx.x, a.by_places), place = blockIdx.x - rest * a.places;
  const int bk = fast_div(rest, a.by_kvh), kvh = rest - bk * a.kv_heads;
  const int split = fast_div(bk, a.by_batch), b = bk - split * a.pt.batch;
  const Seq s = load_seq(a.pt, b, a.max_q);
  const int n_rows = s.nq * a.group;
  const int n_tiles = (s.len + kWeightKeys - 1) / kWeightKeys;
  if (n_rows < a.min_rows || n_rows <= 0 || place >= (a.pairs ? (n_tiles + 1) / 2 : n_tiles)) return;
  const int32_t* row = a.pt.table + b * a.pt.table_stride;

  const char* qh = a.q + s.q0 * a.q_st + (int64_t)kvh * a.group * a.q_sh;
  const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(smem));
  auto issue = [&](int t, int buf) FA_INLINE {
    const int i0 = fast_div(min(t * RT, n_rows - 1), a.by_group);  // first token: the DMA's base
    const char* src = qh + i0 * a.q_st;
#pragma unroll
    for (int it = 0; it < NI; ++it) {
      const int rt = (wave * NI + it) * (1024 / ROWB) + lane / LPR;
      const int r = min(t * RT + rt, n_rows - 1);
      const int i = fast_div(r, a.by_group), h = r - i * a.group;
      const int c = (lane % LPR) ^ lds::Tile16<D>::swz_k(rt);
      poison_1k(base + buf * TB + (wave * NI + it) * 1024);
      dma_16b((uint32_t)((i - i0) * (int)a.q_st + h * (int)a.q_sh + c * 16), src,
              base + buf * TB + (wave * NI + it) * 1024);
    }
  };
  // lse (log2) and last visible key of row t * RT + lane, for all lanes;
  // rows that do not exist or have no weights see nothing.
  float lse_n = 0.0f;
  int last_n = -1;
  auto fetch_row = [&](int t) FA_INLINE {
    const int r = t * RT + lane, rc = min(r, n_rows - 1);
    const int i = fast_div(rc, a.by_group), h = rc - i * a.group;
    const float l = a.lse[(int64_t)(s.q0 + i) * a.heads + kvh * a.group + h];
    last_n = r < n_rows && l != -INFINITY ? (a.causal ? min(s.first + i, s.len - 1) : s.len - 1) : -1;
    lse_n = l * kLog2e;
  };
  int k_off[KST];
#pragma unroll
  for (int st = 0; st < KST; ++st) k_off[st] = lds::k16_read_offset<D>(0, st, lane);

  for (int sub = 0; sub < 2; ++sub) {
    const int tile = sub == 0 ? place : n_tiles - 1 - place;
    if (sub == 1 && (!a.pairs || tile == place)) break;
    const int key0 = tile * kWeightKeys, wkey0 = key0 + 64 * wave;

    // This lane's keys wkey0 + 16kb + l16: rows of K past the end re-read the
    // last key, absent pages page 0; their sums are not used.
    i16x8 kf[KB][KST];
    unsigned there = 0;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int r0 = min(wkey0 + 16 * kb, (s.len - 1) & ~15);
      const int id = page_id(a.pt, row, r0);
      const bool ok = (uint32_t)id < (uint32_t)a.pt.num_pages;
      if (ok) there |= 1u << kb;
      const int in_page = (r0 & ((1 << a.pt.page_shift) - 1)) + min(l16, s.len - 1 - r0);
      const char* kp = a.k + (int64_t)(ok ? id : 0) * a.k_sp + kvh * a.k_sh + (int64_t)in_page * a.k_ss;
#pragma unroll
      for (int st = 0; st < KST; ++st)
        kf[kb][st] = *reinterpret_cast<const i16x8*>(kp + (32 * st + 8 * g4) * 2);
    }

    // Row tiles: from the first token that sees the first key, cut into the
    // grid's splits.
    const int i_first = a.causal ? max(0, key0 - s.first) : 0;
    const int t_begin = (int)min((int64_t)i_first * a.group, (int64_t)n_rows) / RT;
    const int t_all = (n_rows + RT - 1) / RT - t_begin;
    const int each = fast_div(t_all, a.by_splits), more = t_all - each * a.splits;
    const int t0 = t_begin + split * each + min(split, more);
    const int t1 = t0 + each + (split < more ? 1 : 0);

    float acc[KB] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (t0 < t1) {
      fetch_row(t0);
      issue(t0, 0);
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    // One row tile from LDS.  MASKED: some row does not see some of the wave's keys.
    auto compute = [&](auto masked_c, int buf, float lse, int last) FA_INLINE {
      constexpr bool MASKED = decltype(masked_c)::value;
      neg_lse[wave][lane] = -lse;
      f32x4 sc[2][KB];  // the next 16 rows' products run beside this one's exponentials
      auto products = [&](int rb) FA_INLINE {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) sc[rb & 1][kb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < KST; ++st) {
          const i16x8 qa = *reinterpret_cast<const i16x8*>(smem + buf * TB + rb * 16 * ROWB + k_off[st]);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) sc[rb & 1][kb] = mfma16<BF16>(qa, kf[kb][st], sc[rb & 1][kb]);
        }
      };
      products(0);
#pragma unroll
      for (int rb = 0; rb < RT / 16; ++rb) {
        if (rb + 1 < RT / 16) products(rb + 1);
        // rows 16rb + 4g4 + i, keys wkey0 + 16kb + l16
        const f32x4 nl = *reinterpret_cast<const f32x4*>(&neg_lse[wave][16 * rb + 4 * g4]);
        int rel[4];
        if constexpr (MASKED) {
#pragma unroll
          for (int i = 0; i < 4; ++i) rel[i] = __shfl(last, 16 * rb + 4 * g4 + i) - wkey0 - l16;
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = fast_exp2(fmaf(sc[rb & 1][kb][i], a.scale_log2, nl[i]));
            if constexpr (MASKED)
              acc[kb] += 16 * kb <= rel[i] ? p : 0.0f;
            else
              acc[kb] += p;
          }
      }
    };
    // Rows ascend, and with them the keys they see: masked tiles (or ones that
    // see none of the wave's keys) first, whole ones, and a last one whose rows
    // end inside it.  Loops of their own, so that the whole ones carry no masks;
    // every wave passes one barrier a tile, whichever loop it is in.
    int t = t0;
    auto step = [&](auto masked_c) FA_INLINE {
      const float lse = lse_n;
      const int last = last_n, buf = (t - t0) & 1;
      if (t + 1 < t1) {
        issue(t + 1, buf ^ 1);
        fetch_row(t + 1);
      }
      if (!decltype(masked_c)::value || (__any(last >= wkey0) && wkey0 < s.len)) compute(masked_c, buf, lse, last);
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      ++t;
    };
    auto whole = [&]() FA_INLINE { return __all(last_n >= wkey0 + 63); };
    while (t < t1 && !whole()) step(std::true_type{});
    while (t < t1 && whole()) step(std::false_type{});
    while (t < t1) step(std::true_type{});

    // Lane group g4 finishes key block g4, so a lane the key of its number.  (The
    // lane is asked for again: kept from the start, it was spilled.)
    const int me = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    float mine = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      float x = acc[kb];
      x += __shfl_xor(x, 16);
      x += __shfl_xor(x, 32);
      if (me >> 4 == kb) mine = x;
    }
    const int key = wkey0 + me;
    if (a.ws != nullptr) {
      a.ws[((((int64_t)split * a.pt.batch + b) * a.kv_heads + kvh) * a.key_tiles + tile) * kWeightKeys +
           64 * wave + me] = mine;
    } else if (key < s.len && ((there >> (me >> 4)) & 1u)) {
      const int id = row[key >> a.pt.page_shift];
      float* w = a.w + (int64_t)id * a.w_sp + kvh * a.w_sh + (key & ((1 << a.pt.page_shift) - 1));
      *w = key >= s.first ? mine : *w + mine;
    }
  }
}

// Few rows (a few tokens): q stays in registers as the A operand, K streams
// through two LDS tiles of 32 keys that each wave has to itself, and the keys'
// sums gather in LDS.  Bound by reading K.  32 sequences of up to 8192 keys, 8
// kv heads, D = 128: 93 us with loads straight to registers, one 256-key tile a
// workgroup; 78 so, with four workgroups of 2048 keys per CU (5.1 TB/s); 82
// with four LDS tiles a wave and two workgroups per CU; 88 with 1024 keys.
template <int D, bool BF16, int RB>
__global__ void __launch_bounds__(128) fa_weights_few_kernel(const PagedWeightsArgs a) {
  constexpr int NW = 2, ST = 2, kDepth = ST - 1;             // waves, ring tiles
  constexpr int ROWB = 2 * D, KST = D / 32, TB = 32 * ROWB, NI = 16 * ROWB / 1024;
  __shared__ __attribute__((aligned(1024))) char smem[NW * ST * TB];
  __shared__ float sums[kWeightChunk];  // of a.few_keys keys

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int rest = fast_div(blockIdx.x, a.by_few), chunk = blockIdx.x - rest * a.few_chunks;
  const int b = fast_div(rest, a.by_kvh), kvh = rest - b * a.kv_heads;
  const int c0 = chunk * a.few_keys;
  const int32_t* row = a.pt.table + b * a.pt.table_stride;
  PageIds ids;
  ids.start(a.pt, row, c0);
  const Seq s = load_seq(a.pt, b, a.max_q);
  const int n_rows = s.nq * a.group;
  if (n_rows <= 0 || n_rows > a.max_rows || c0 >= s.len) return;
  const int c1 = min(s.len, c0 + a.few_keys), last = c1 - 1;
  const int n_tiles = (c1 - c0 + 31) / 32;

  const uint32_t wave_lds = __builtin_amdgcn_readfirstlane(lds_addr(smem)) + wave * ST * TB;
  KeyStage<D> stage;
  stage.init(lane, a.k_ss);
  const char* kbase = a.k + kvh * a.k_sh;
  auto issue = [&](int t, int slot) FA_INLINE {
    const int key = c0 + 32 * t;
    ids.reach(key);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int r0 = min(key + 16 * g, last & ~15);
      const int in_page = r0 & ((1 << a.pt.page_shift) - 1);
      stage.copy(kbase + ids.page(r0) * a.k_sp + (int64_t)in_page * a.k_ss,
                 wave_lds + slot * TB + g * 16 * ROWB, last - r0, a.k_ss);
    }
  };
  // This wave's tiles: wave, wave + NW, ...
  const int mine = (n_tiles - wave + NW - 1) / NW;
#pragma unroll
  for (int i = 0; i < kDepth; ++i)
    if (i < mine) issue(wave + i * NW, i);

  // q, and lse (log2) and last visible key of rows 16rb + 4g4 + i.
  const char* qh = a.q + s.q0 * a.q_st + (int64_t)kvh * a.group * a.q_sh;
  i16x8 qf[RB][KST];
  float lse[RB][4];
  int see[RB][4];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = min(16 * rb + l16, n_rows - 1);
    const int i = fast_div(r, a.by_group), h = r - i * a.group;
#pragma unroll
    for (int st = 0; st < KST; ++st)
      qf[rb][st] = *reinterpret_cast<const i16x8*>(qh + i * a.q_st + h * a.q_sh + (32 * st + 8 * g4) * 2);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int rr = 16 * rb + 4 * g4 + e, rc = min(rr, n_rows - 1);
      const int ii = fast_div(rc, a.by_group), hh = rc - ii * a.group;
      const float l = a.lse[(int64_t)(s.q0 + ii) * a.heads + kvh * a.group + hh];
      see[rb][e] = rr < n_rows && l != -INFINITY ? (a.causal ? min(s.first + ii, s.len - 1) : s.len - 1) : -1;
      lse[rb][e] = l * kLog2e;
    }
  }
  uint32_t k_addr[KST];
#pragma unroll
  for (int st = 0; st < KST; ++st) k_addr[st] = wave_lds + lds::k16_read_offset<D>(0, st, lane);

  auto tile = [&](auto slot_c, int i) FA_INLINE {
    constexpr int SLOT = decltype(slot_c)::value;
    const int t = wave + i * NW;
    if (i + kDepth < mine) {
      issue(t + kDepth * NW, (SLOT + kDepth) % ST);
      wait_vmcnt<2 * NI * kDepth>();
    } else {
      wait_vmcnt<0>();
    }
    f32x4 sc[2][RB];
#pragma unroll
    for (int st = 0; st < KST; ++st)
      static_for<0, 2>([&](auto kb_c) FA_INLINE {
        constexpr int kb = decltype(kb_c)::value;
        const i16x8 kf = lds_read16<SLOT * TB + kb * 16 * ROWB>(k_addr[st]);
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) sc[kb][rb] = mfma16<BF16>(qf[rb][st], kf, st == 0 ? zero : sc[kb][rb]);
      });
    float x[2] = {0.0f, 0.0f};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const int key = c0 + 32 * t + 16 * kb + l16;
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = fast_exp2(fmaf(sc[kb][rb][e], a.scale_log2, -lse[rb][e]));
          x[kb] += key <= see[rb][e] ? p : 0.0f;
        }
      x[kb] += __shfl_xor(x[kb], 16);
      x[kb] += __shfl_xor(x[kb], 32);
    }
    if (g4 < 2) sums[32 * t + lane] = g4 == 0 ? x[0] : x[1];
    fence_lds_reads();
  };
  for (int i = 0; i < mine; i += ST) {
    static_for<0, ST>([&](auto slot_c) FA_INLINE {
      if (i + decltype(slot_c)::value < mine) tile(slot_c, i + decltype(slot_c)::value);
    });
  }
  __syncthreads();
  // Eight keys a thread in flight: one after another cost as much as the sums.
  constexpr int PER = 8, STEP = PER * 64 * NW;
  for (int k0 = c0; k0 < c1; k0 += STEP) {
    int id[PER];
    float* w[PER];
    float old[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int key = k0 + j * 64 * NW + (int)threadIdx.x;
      id[j] = key < c1 ? row[key >> a.pt.page_shift] : -1;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int key = k0 + j * 64 * NW + (int)threadIdx.x;
      w[j] = a.w + (int64_t)id[j] * a.w_sp + kvh * a.w_sh + (key & ((1 << a.pt.page_shift) - 1));
      old[j] = 0.0f;
      if ((uint32_t)id[j] < (uint32_t)a.pt.num_pages && key < s.first) old[j] = *w[j];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if ((uint32_t)id[j] < (uint32_t)a.pt.num_pages)
        *w[j] = old[j] + sums[k0 - c0 + j * 64 * NW + threadIdx.x];
  }
}

// Adds the row splits' sums, in their order, to the weights.
__global__ void __launch_bounds__(256) fa_weights_sum_kernel(const PagedWeightsArgs a) {
  const int rest = fast_div(blockIdx.x, a.by_tiles), tile = blockIdx.x - rest * a.key_tiles;
  const int b = fast_div(rest, a.by_kvh), kvh = rest - b * a.kv_heads;
  const Seq s = load_seq(a.pt, b, a.max_q);
  const int key = tile * kWeightKeys + threadIdx.x;
  if (s.nq * a.group < a.min_rows || s.nq <= 0 || key >= s.len) return;
  const int id = a.pt.table[b * a.pt.table_stride + (key >> a.pt.page_shift)];
  const float* part = a.ws + (((int64_t)b * a.kv_heads + kvh) * a.key_tiles + tile) * kWeightKeys + threadIdx.x;
  const int64_t step = (int64_t)a.pt.batch * a.kv_heads * a.key_tiles * kWeightKeys;
  constexpr int BATCH = 8;  // loads in flight
  float sum = 0.0f;
  for (int c = 0; c < a.splits; c += BATCH) {
    float x[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) x[j] = c + j < a.splits ? part[(c + j) * step] : 0.0f;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) sum += x[j];
  }
  if ((uint32_t)id >= (uint32_t)a.pt.num_pages) return;
  float* w = a.w + (int64_t)id * a.w_sp + kvh * a.w_sh + (key & ((1 << a.pt.page_shift) - 1));
  *w = key >= s.first ? sum : *w + sum;
}

// ---- eviction ----

// Bits of a weight in an order: larger weights, larger numbers; both zeros
// alike, NaN above all.
__device__ __forceinline__ uint32_t weight_order(float x) {
  if (x != x) return ~0u;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 + 0 = +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / 64;
constexpr int kSelBins = 2048, kSelCopies = 4;

// One workgroup per sequence and kv head.  A thread owns K consecutive keys of
// a segment of 1024 K, in one page (a page holds whole groups of 16): one page
// lookup, vector loads, and index order is thread order, so the places of the
// kept keys are one prefix sum per segment.  Weights of the first segment stay
// in registers; longer sequences read the others again in each of the three
// passes.  The histogram has copies by lane, as near weights share their top
// bits and LDS atomics on one word queue up.  Bound by its few steps one after
// another, not by memory: 8 sequences x 8 heads of 16384 keys take 15.5 us; 40
// with one key a thread and eight-bit digits, 19 with 8 copies (clearing and
// adding them up), 16.4 with the kept keys put in order in LDS first.
template <int K>
__global__ void __launch_bounds__(kSelThreads) fa_select_kernel(const PagedEvictArgs a) {
  __shared__ int hist[kSelCopies][kSelBins];
  __shared__ int wave_n[kSelWaves];
  __shared__ int pick[3];
  __shared__ int bad;
  typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));  // any key weight's address
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / a.kv_heads, kvh = blockIdx.x - b * a.kv_heads;
  const int len = min(max(a.pt.lens[b], 0), a.pt.max_kv);
  const int n = min(len, a.keep);
  const int32_t* row = a.pt.table + b * a.pt.table_stride;
  const int32_t* new_row = a.new_table + b * a.new_table_stride;
  int32_t* kept = a.kept + ((int64_t)b * a.kv_heads + kvh) * a.keep;
  const int shift_p = a.pt.page_shift, page = 1 << shift_p;

  if (tid == 0) bad = 0;
  __syncthreads();
  bool miss = false;
  for (int i = tid; i * (int64_t)page < len; i += kSelThreads)
    miss = miss || (uint32_t)row[i] >= (uint32_t)a.pt.num_pages;
  for (int i = tid; i * (int64_t)page < n; i += kSelThreads)
    miss = miss || (uint32_t)new_row[i] >= (uint32_t)a.pt.num_pages;
  if (__any(miss) && lane == 0) bad = 1;
  __syncthreads();
  // (The new length is not written here: it may be the old one's place, which
  // the other heads still read.)
  const int count = bad ? 0 : n;
  for (int t = count + tid; t < a.keep; t += kSelThreads) kept[t] = -1;
  if (bad) return;
  if (len <= a.keep) {
    for (int t = tid; t < n; t += kSelThreads) kept[t] = t;
    return;
  }

  // The want heaviest of the keys before the recent ones.
  const int old = len - a.recent, want = a.keep - a.recent;
  constexpr int kSeg = kSelThreads * K;
  uint32_t u[K];
  auto load = [&](int seg) FA_INLINE {
    const int i0 = seg + tid * K;
    if (i0 >= old) return;
    const float* w = a.w + (int64_t)row[i0 >> shift_p] * a.w_sp + kvh * a.w_sh + (i0 & (page - 1));
#pragma unroll
    for (int j = 0; j < K; j += 4) {
      const f32x4_u x = *reinterpret_cast<const f32x4_u*>(w + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) u[j + e] = weight_order(x[e]);
    }
  };
  load(0);
  uint32_t prefix = 0, mask = 0;  // the top bits of the want-th largest
  int left = want;                // its rank among the keys with that prefix
#pragma unroll 1
  for (int pass = 0; pass < 3 && want > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kSelCopies * kSelBins; i += kSelThreads) (&hist[0][0])[i] = 0;
    __syncthreads();
#pragma unroll 1
    for (int seg = 0; seg < old; seg += kSeg) {
      if (old > kSeg) load(seg);
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (seg + tid * K + j < old && (u[j] & mask) == prefix)
          atomicAdd(&hist[lane & (kSelCopies - 1)][(u[j] >> shift) & digit], 1);
    }
    __syncthreads();
    // Two bins a thread; counts of the keys above them by a suffix sum.
    int c[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      c[j] = 0;
#pragma unroll
      for (int q = 0; q < kSelCopies; ++q) c[j] += hist[q][2 * tid + j];
    }
    int above = c[0] + c[1];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_down(above, d);
      above += lane + d < 64 ? x : 0;
    }
    if (lane == 0) wave_n[wave] = above;
    __syncthreads();
    above -= c[0] + c[1];
#pragma unroll
    for (int w = 1; w < kSelWaves; ++w) above += w > wave ? wave_n[w] : 0;
#pragma unroll
    for (int j = 1; j >= 0; --j) {
      if (above < left && left <= above + c[j]) {
        pick[0] = 2 * tid + j;
        pick[1] = left - above;
        pick[2] = c[j];
      }
      above += c[j];
    }
    __syncthreads();
    prefix |= (uint32_t)pick[0] << shift;
    mask |= digit << shift;
    left = pick[1];
    if (pick[2] == left) break;  // every key with this prefix is kept
  }

  // Kept: keys above the threshold, the first `left` that equal it (in the bits
  // that were looked at), and the recent ones: key i goes to place (larger
  // before i) + (equal before i, at most left).  Both counts in one prefix sum,
  // 16 bits each (a segment has at most 2^14 keys).
  int gt_before = 0, eq_before = 0;
#pragma unroll 1
  for (int seg = 0; seg < old && want > 0; seg += kSeg) {
    if (old > kSeg) load(seg);
    int mine = 0;
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (seg + tid * K + j < old) mine += (u[j] & mask) > prefix ? 1 : (u[j] & mask) == prefix ? 1 << 16 : 0;
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int x = __shfl_up(sum, d);
      sum += lane >= d ? x : 0;
    }
    if (lane == 63) wave_n[wave] = sum;
    __syncthreads();
    int before = sum - mine, all = 0;
#pragma unroll
    for (int w = 0; w < kSelWaves; ++w) {
      before += w < wave ? wave_n[w] : 0;
      all += wave_n[w];
    }
    int g = gt_before + (before & 0xffff), e = eq_before + (before >> 16);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const int i = seg + tid * K + j;
      const bool gt = i < old && (u[j] & mask) > prefix, eq = i < old && (u[j] & mask) == prefix;
      if (gt || (eq && e < left)) kept[g + min(e, left)] = i;
      g += gt;
      e += eq;
    }
    gt_before += all & 0xffff;
    eq_before += all >> 16;
    __syncthreads();
  }
  for (int t = tid; t < a.recent; t += kSelThreads) kept[want + t] = old + t;
}

// Copies the kept keys' rows of K and V, and their weights.  LPR lanes move a
// row, kMoveRows rows apart per lane in flight.  The number of kept keys, the
// same for every head of a sequence, ends at the first place that holds -1.
constexpr int kMoveRows = 2;  // (of 64 heads of 4096 keys, D = 128, 55 us: 4 rows 2 us more, 8 rows 7)
template <int D>
__global__ void __launch_bounds__(256) fa_move_kernel(const PagedEvictArgs a, int blocks, int most) {
  constexpr int LPR = 2 * D / 16, RPB = 256 / LPR;
  const int bk = blockIdx.x / blocks, b = bk / a.kv_heads, kvh = bk - b * a.kv_heads;
  const int t0 = (blockIdx.x - bk * blocks) * RPB * kMoveRows + (int)threadIdx.x / LPR;
  const int c = ((int)threadIdx.x % LPR) * 16;
  const int32_t* row = a.pt.table + b * a.pt.table_stride;
  const int32_t* new_row = a.new_table + b * a.new_table_stride;
  const int32_t* kept = a.kept + (int64_t)bk * a.keep;
  const int shift = a.pt.page_shift, mask = (1 << shift) - 1;
  int src[kMoveRows];
  u32x4 k[kMoveRows], v[kMoveRows];
  float w[kMoveRows];
#pragma unroll
  for (int j = 0; j < kMoveRows; ++j) src[j] = t0 + j * RPB < most ? kept[t0 + j * RPB] : -1;
  if (kvh == 0 && c == 0) {
#pragma unroll
    for (int j = 0; j < kMoveRows; ++j) {
      const int t = t0 + j * RPB;
      if (src[j] >= 0 && (t + 1 == most || kept[t + 1] < 0)) a.new_lens[b] = t + 1;
      if (t == 0 && src[j] < 0) a.new_lens[b] = 0;
    }
  }
#pragma unroll
  for (int j = 0; j < kMoveRows; ++j)
    if (src[j] >= 0) {
      const int64_t id = row[src[j] >> shift];
      const int at = src[j] & mask;
      k[j] = *reinterpret_cast<const u32x4*>(a.k + id * a.k_sp + kvh * a.k_sh + (int64_t)at * a.k_ss + c);
      v[j] = *reinterpret_cast<const u32x4*>(a.v + id * a.v_sp + kvh * a.v_sh + (int64_t)at * a.v_ss + c);
      if (c == 0) w[j] = a.w[id * a.w_sp + kvh * a.w_sh + at];
    }
#pragma unroll
  for (int j = 0; j < kMoveRows; ++j)
    if (src[j] >= 0) {
      const int t = t0 + j * RPB, at = t & mask;
      const int64_t id = new_row[t >> shift];
      *reinterpret_cast<u32x4*>(a.k + id * a.k_sp + kvh * a.k_sh + (int64_t)at * a.k_ss + c) = k[j];
      *reinterpret_cast<u32x4*>(a.v + id * a.v_sp + kvh * a.v_sh + (int64_t)at * a.v_ss + c) = v[j];
      if (c == 0) a.w[id * a.w_sp + kvh * a.w_sh + at] = w[j];
    }
}

}  // namespace

hipError_t launch_paged_weights(const PagedWeightsArgs& args, const WeightsPlan& plan, int head_dim,
                                bool bf16, hipStream_t stream) {
  PagedWeightsArgs a = args;
  a.min_rows = plan.few_rows > 0 ? plan.few_rows + 1 : 1;
  a.max_rows = plan.few_rows;
  void* kargs[] = {&a};
  const int64_t bk = (int64_t)a.pt.batch * a.kv_heads;
  if (plan.few_rows > 0) {
    a.few_keys = plan.few_keys;
    a.few_chunks = (a.pt.max_kv + a.few_keys - 1) / a.few_keys;
    a.by_few = make_fast_div((uint32_t)a.few_chunks);
    const int64_t grid = bk * a.few_chunks;
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    auto few = [&](auto rb_c) -> const void* {
      constexpr int RB = decltype(rb_c)::value;
      if (head_dim == 128)
        return bf16 ? reinterpret_cast<const void*>(&fa_weights_few_kernel<128, true, RB>)
                    : reinterpret_cast<const void*>(&fa_weights_few_kernel<128, false, RB>);
      return bf16 ? reinterpret_cast<const void*>(&fa_weights_few_kernel<64, true, RB>)
                  : reinterpret_cast<const void*>(&fa_weights_few_kernel<64, false, RB>);
    };
    const void* fn = plan.few_rows <= 16 ? few(std::integral_constant<int, 1>{})
                                         : few(std::integral_constant<int, 2>{});
    const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)grid), dim3(128), kargs, 0, stream);
    if (e != hipSuccess) return e;
  }
  if (plan.splits == 0) return hipSuccess;
  const int64_t tiles = bk * a.key_tiles;
  a.pairs = plan.pairs;
  a.places = a.pairs ? (a.key_tiles + 1) / 2 : a.key_tiles;
  a.by_places = make_fast_div((uint32_t)a.places);
  const int64_t grid = bk * a.places * a.splits;
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  const void* fn;
  if (head_dim == 128)
    fn = bf16 ? reinterpret_cast<const void*>(&fa_weights_kernel<128, true>)
              : reinterpret_cast<const void*>(&fa_weights_kernel<128, false>);
  else
    fn = bf16 ? reinterpret_cast<const void*>(&fa_weights_kernel<64, true>)
              : reinterpret_cast<const void*>(&fa_weights_kernel<64, false>);
  const hipError_t e = hipLaunchKernel(fn, dim3((unsigned)grid), dim3(256), kargs, 0, stream);
  if (e != hipSuccess || a.ws == nullptr) return e;
  return hipLaunchKernel(reinterpret_cast<const void*>(&fa_weights_sum_kernel), dim3((unsigned)tiles),
                         dim3(256), kargs, 0, stream);
}

hipError_t launch_paged_evict(const PagedEvictArgs& args, int head_dim, hipStream_t stream) {
  PagedEvictArgs a = args;
  const int64_t bk = (int64_t)a.pt.batch * a.kv_heads;
  int most = std::min(a.keep, a.pt.max_kv);
  const int per = 256 / (2 * head_dim / 16) * kMoveRows;
  int blocks = std::max(1, (most + per - 1) / per);  // (no keys: the new lengths)
  if (bk * blocks > 0x7fffffff) return hipErrorInvalidValue;
  void* sargs[] = {&a};
  // Four keys a thread where they hold all of a sequence: less work in a row.
  const void* select = a.pt.max_kv <= 4 * kSelThreads
                           ? reinterpret_cast<const void*>(&fa_select_kernel<4>)
                           : reinterpret_cast<const void*>(&fa_select_kernel<16>);
  hipError_t e = hipLaunchKernel(select, dim3((unsigned)bk),
                                 dim3(kSelThreads), sargs, 0, stream);
  if (e != hipSuccess) return e;
  void* margs[] = {&a, &blocks, &most};
  const void* fn = head_dim == 128 ? reinterpret_cast<const void*>(&fa_move_kernel<128>)
                                   : reinterpret_cast<const void*>(&fa_move_kernel<64>);
  return hipLaunchKernel(fn, dim3((unsigned)(bk * blocks)), dim3(256), margs, 0, stream);
}

}  // namespace fa
