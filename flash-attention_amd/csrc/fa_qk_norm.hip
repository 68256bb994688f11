// Per-head RMS norm of q and k with the position rotation, forward and
// backward, and the store of new tokens into a paged cache, on gfx950.
//
//   xh = x rstd, rstd = (mean(x^2) + eps)^(-1/2);  y = R(pos) (xh w)
//   g = R(pos)^T dy;  dx = rstd (g w - xh mean(g w xh));  dw = sum_rows g xh
//
// One pass: a row is read, normed, turned and written, in fp32 with one
// rounding at the end.  The backward pass computes rstd again from x, which it
// reads anyway, so the forward keeps nothing.  All of it is bound by memory:
// 2 x 8192 tokens, 32 + 8 heads of 128, bf16: 61 us forward (5.5 TB/s), 104
// backward (4.8) and 5 for the join of dw; the store of 8 prompts of 3000
// tokens, 16 heads of 64: 36 us.
//
// D / 8 lanes share a row.  A lane owns 8 elements so that the pairs of the
// rotation lie within a lane: 4 from each half of the rotated dims (two 8-byte
// loads), or 8 neighbours (interleaved pairs, and the dims past the rotation).
// It reads and writes the same elements, so outputs may be the inputs.  A lane
// group keeps one token and walks over its heads, so the token's cosines,
// sines and place in the cache are looked up once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "fa_cache_kernels.h"
#include "fa_device_ops.h"

namespace fa {
namespace {

using namespace dev;

template <bool BF16>
__device__ __forceinline__ void unpack4(u32x2 w, float* f) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t u = w[j];  // (a bit_cast of w[j] itself reads element 0)
    if constexpr (BF16) {
      f[2 * j] = __builtin_bit_cast(float, u << 16);
      f[2 * j + 1] = __builtin_bit_cast(float, u & 0xffff0000u);
    } else {
      const f16x2 h = __builtin_bit_cast(f16x2, u);
      f[2 * j] = (float)h[0];
      f[2 * j + 1] = (float)h[1];
    }
  }
}

// A lane's 8 elements of a row: 4 at byte `a`, 4 at byte `b` (b = a + 8 where
// they are neighbours).
struct Raw {
  u32x2 a, b;
};
template <bool INTER>
__device__ __forceinline__ Raw load_raw(const char* row, int a, int b) {
  if constexpr (INTER) {
    const u32x4 w = *reinterpret_cast<const u32x4*>(row + a);
    return Raw{u32x2{w[0], w[1]}, u32x2{w[2], w[3]}};
  } else {
    return Raw{*reinterpret_cast<const u32x2*>(row + a), *reinterpret_cast<const u32x2*>(row + b)};
  }
}
template <bool BF16, bool INTER>
__device__ __forceinline__ void store8(char* row, int a, int b, const float* f) {
  const u32x2 lo = {pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3])};
  const u32x2 hi = {pack2<BF16>(f[4], f[5]), pack2<BF16>(f[6], f[7])};
  if constexpr (INTER) {
    *reinterpret_cast<u32x4*>(row + a) = u32x4{lo[0], lo[1], hi[0], hi[1]};
  } else {
    *reinterpret_cast<u32x2*>(row + a) = lo;
    *reinterpret_cast<u32x2*>(row + b) = hi;
  }
}

// Sum over the LPR lanes of a row (aligned groups).
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int d = 1; d < LPR; d <<= 1) x += __shfl_xor(x, d);
  return x;
}

// The rotation of a lane's 8 elements: pairs (j, 4 + j), or interleaved
// (2j, 2j + 1), j = 0..3.  SIGN -1: the inverse.
template <bool INTER, int SIGN>
__device__ __forceinline__ void rotate(float* f, const float* c, const float* s) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int p = INTER ? 2 * j : j, q = INTER ? 2 * j + 1 : 4 + j;
    const float x = f[p], y = f[q], sn = SIGN * s[j];
    f[p] = x * c[j] - y * sn;
    f[q] = y * c[j] + x * sn;
  }
}

template <int D, bool BF16, bool INTER>
struct Lane {
  static constexpr int LPR = D / 8;
  int a, b;        // byte offsets of the lane's elements in a row
  float c[4], s[4];
  __device__ __forceinline__ void place(const NormArgs& n) {
    const int j = threadIdx.x % LPR;
    const bool turned = 8 * j < n.rot;
    const int ea = INTER ? 8 * j : turned ? 4 * j : n.rot + 8 * (j - n.rot / 8);
    a = 2 * ea;
    b = INTER || !turned ? a + 8 : 2 * (n.rot / 2 + 4 * j);
  }
  // The token's cosines and sines: 1 and 0 past the rotation, NaN for a
  // position outside the tables.
  __device__ __forceinline__ void angles(const NormArgs& n, int pos) {
    const int j = threadIdx.x % LPR;
    const bool turned = 8 * j < n.rot, known = (uint32_t)pos < (uint32_t)n.table_rows;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = known ? 1.0f : NAN;
      s[i] = known ? 0.0f : NAN;
    }
    if (turned && known) {
      const int64_t at = (int64_t)pos * (n.rot / 2) + 4 * j;
      const f32x4 cv = *reinterpret_cast<const f32x4*>(n.cos + at);
      const f32x4 sv = *reinterpret_cast<const f32x4*>(n.sin + at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = cv[i];
        s[i] = sv[i];
      }
    }
  }
  __device__ __forceinline__ void weights(const NormArgs& n, int which, float* w) const {
    const char* p = static_cast<const char*>(n.weight[which]);
    if (n.weight_fp32) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(p + 2 * a);
      const f32x4 y = *reinterpret_cast<const f32x4*>(p + 2 * b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = x[i];
        w[4 + i] = y[i];
      }
    } else {
      unpack4<BF16>(*reinterpret_cast<const u32x2*>(p + a), w);
      unpack4<BF16>(*reinterpret_cast<const u32x2*>(p + b), w + 4);
    }
  }
};

constexpr int kRows = 4;      // rows a lane group has in flight
constexpr int kBwdHeads = 4;  // heads of a block of the backward pass

// Tokens x heads.  STORE: packed new tokens, heads H .. H + KH - 1 are k's and
// the next KH are v's, both to the cache.
template <int D, bool BF16, bool INTER, bool STORE>
__global__ void __launch_bounds__(256) fa_norm_kernel(const NormArgs n) {
  using L = Lane<D, BF16, INTER>;
  constexpr int LPR = L::LPR, TPW = 256 / LPR, TPV = 64 / LPR;  // tokens of a workgroup, a wave
  const int token = blockIdx.x % n.blocks_x * TPW + (int)threadIdx.x / LPR;
  const int h0 = blockIdx.x / n.blocks_x * n.head_chunk;
  const int heads = n.heads + (STORE ? 2 : 1) * n.kv_heads, h1 = min(heads, h0 + n.head_chunk);

  bool mine = token < n.tokens;
  const int tok = min(token, n.tokens - 1);
  const int b = STORE ? 0 : fast_div(tok, n.by_seq), t = STORE ? tok : tok - b * n.seq_len;
  // What needs no place in the cache is asked for first: the loads below wait
  // for one another.
  const int pos = n.positions == nullptr ? t : n.positions[b * n.pos_stride + t];
  L l;
  l.place(n);
  float w[2][8];
  if (h0 < n.heads) l.weights(n, 0, w[0]);
  if (h1 > n.heads && h0 < n.heads + n.kv_heads) l.weights(n, 1, w[1]);

  // Place in the cache, from the number of sequences that end before the
  // token (counted by the whole wave, 64 sequences at a time).
  int64_t page = -1;
  int at = 0;
  if constexpr (STORE) {
    const int lane = threadIdx.x & 63;
    const int wave_token = blockIdx.x % n.blocks_x * TPW + ((int)threadIdx.x >> 6) * TPV;
    const int first = n.pt.cu[0];
    int seq = 0;
    for (int i0 = 1; i0 <= n.pt.batch; i0 += 64) {
      const int i = i0 + lane;
      const int end = i <= n.pt.batch ? n.pt.cu[i] : 0x7fffffff;
#pragma unroll
      for (int g = 0; g < TPV; ++g) {
        const int ended = __popcll(__ballot(end <= wave_token + g));
        if (lane / LPR == g) seq += ended;
      }
    }
    mine = mine && seq < n.pt.batch && token >= first;
    if (mine && h1 > n.heads) {
      // (the limits of load_seq: the token's key is the one its query ends at)
      const int c0 = min(max(n.pt.cu[seq], 0), n.tokens);
      const int c1 = min(max(n.pt.cu[seq + 1], c0), n.tokens);
      const int key = min(max(n.pt.lens[seq], 0), n.pt.max_kv) - c1 + token;
      if (key >= 0 && token >= c0 && token < c1) {
        const int id = n.pt.table[seq * n.pt.table_stride + (key >> n.pt.page_shift)];
        if ((uint32_t)id < (uint32_t)n.pt.num_pages) page = id;
        at = key & ((1 << n.pt.page_shift) - 1);
      }
    }
  }
  l.angles(n, pos);
  if (!mine) return;

  auto range = [&](auto x_c, int lo, int hi, const float* wt) FA_INLINE {
    constexpr int X = decltype(x_c)::value;
    const char* src = n.x[X] + b * n.x_sb[X] + t * n.x_st[X];
    char* dst = n.y[X];
    if (STORE && X > 0) {
      if (page < 0) return;
      dst += page * n.y_sb[X] + at * n.y_st[X];
    } else {
      dst += b * n.y_sb[X] + t * n.y_st[X];
    }
    for (int h = lo; h < hi; h += kRows) {
      Raw raw[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (h + r < hi) raw[r] = load_raw<INTER>(src + (h + r) * n.x_sh[X], l.a, l.b);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (h + r >= hi) break;
        char* out = dst + (h + r) * n.y_sh[X];
        float f[8];
        if constexpr (X == 2) {  // v is copied
          if constexpr (INTER) {
            *reinterpret_cast<u32x4*>(out + l.a) = u32x4{raw[r].a[0], raw[r].a[1], raw[r].b[0], raw[r].b[1]};
          } else {
            *reinterpret_cast<u32x2*>(out + l.a) = raw[r].a;
            *reinterpret_cast<u32x2*>(out + l.b) = raw[r].b;
          }
          continue;
        }
        unpack4<BF16>(raw[r].a, f);
        unpack4<BF16>(raw[r].b, f + 4);
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
        const float rstd = rsqrtf(row_sum<LPR>(ss) * (1.0f / D) + n.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = f[i] * rstd * wt[i];
        rotate<INTER, 1>(f, l.c, l.s);
        store8<BF16, INTER>(out, l.a, l.b, f);
      }
    }
  };
  if (h0 < n.heads) range(std::integral_constant<int, 0>{}, h0, min(h1, n.heads), w[0]);
  if (h1 > n.heads && h0 < n.heads + n.kv_heads)
    range(std::integral_constant<int, 1>{}, max(h0 - n.heads, 0), min(h1 - n.heads, n.kv_heads), w[1]);
  if constexpr (STORE) {
    const int v0 = n.heads + n.kv_heads;
    if (h1 > v0) range(std::integral_constant<int, 2>{}, max(h0 - v0, 0), h1 - v0, w[0]);
  }
}

// Backward: y holds the incoming gradients.  Each workgroup walks over token
// blocks at a fixed stride, and leaves its sums for the weights' gradients in
// ws[block][2][D].
template <int D, bool BF16, bool INTER>
__global__ void __launch_bounds__(256) fa_norm_bwd_kernel(const NormArgs n) {
  using L = Lane<D, BF16, INTER>;
  constexpr int LPR = L::LPR, TPW = 256 / LPR, R = 2;
  __shared__ float part[4][2][D];
  L l;
  l.place(n);
  float w[2][8], dw[2][8];
  l.weights(n, 0, w[0]);
  l.weights(n, 1, w[1]);
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[0][i] = dw[1][i] = 0.0f;

  const int heads = n.heads + n.kv_heads;
  const int chunks = (heads + n.head_chunk - 1) / n.head_chunk;
  const int blocks = (n.tokens + TPW - 1) / TPW * chunks;
  for (int blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int tb = blk / chunks, h0 = (blk - tb * chunks) * n.head_chunk, h1 = min(heads, h0 + n.head_chunk);
    const int token = tb * TPW + (int)threadIdx.x / LPR;
    if (token >= n.tokens) continue;
    const int b = fast_div(token, n.by_seq), t = token - b * n.seq_len;
    const int pos = n.positions == nullptr ? t : n.positions[b * n.pos_stride + t];
    l.angles(n, pos);
    auto range = [&](auto x_c, int lo, int hi) FA_INLINE {
      constexpr int X = decltype(x_c)::value;
      const char* xs = n.x[X] + b * n.x_sb[X] + t * n.x_st[X];
      const char* gs = n.y[X] + b * n.y_sb[X] + t * n.y_st[X];
      char* ds = n.dx[X] + b * n.dx_sb[X] + t * n.dx_st[X];
      for (int h = lo; h < hi; h += R) {
        Raw xr[R], gr[R];
#pragma unroll
        for (int r = 0; r < R; ++r)
          if (h + r < hi) {
            xr[r] = load_raw<INTER>(xs + (h + r) * n.x_sh[X], l.a, l.b);
            gr[r] = load_raw<INTER>(gs + (h + r) * n.y_sh[X], l.a, l.b);
          }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (h + r >= hi) break;
          float x[8], g[8];
          unpack4<BF16>(xr[r].a, x);
          unpack4<BF16>(xr[r].b, x + 4);
          unpack4<BF16>(gr[r].a, g);
          unpack4<BF16>(gr[r].b, g + 4);
          rotate<INTER, -1>(g, l.c, l.s);
          float ss = 0.0f, gx = 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            ss = fmaf(x[i], x[i], ss);
            gx = fmaf(g[i] * w[X][i], x[i], gx);
          }
          const float rstd = rsqrtf(row_sum<LPR>(ss) * (1.0f / D) + n.eps);
          const float mean = row_sum<LPR>(gx) * rstd * (1.0f / D);  // of g w xh
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float xh = x[i] * rstd;
            dw[X][i] = fmaf(g[i], xh, dw[X][i]);
            x[i] = rstd * (g[i] * w[X][i] - xh * mean);
          }
          store8<BF16, INTER>(ds + (h + r) * n.dx_sh[X], l.a, l.b, x);
        }
      }
    };
    if (h0 < n.heads) range(std::integral_constant<int, 0>{}, h0, min(h1, n.heads));
    if (h1 > n.heads) range(std::integral_constant<int, 1>{}, max(h0 - n.heads, 0), h1 - n.heads);
  }

  // The workgroup's sums: over a wave's lane groups, then over the waves.
  const int lane = threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = dw[x][i];
#pragma unroll
      for (int d = LPR; d < 64; d <<= 1) v += __shfl_xor(v, d);
      if (lane < LPR) part[wave][x][(i < 4 ? l.a / 2 + i : l.b / 2 + i - 4)] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += 256) {
    const int x = i / D, d = i % D;
    n.ws[(int64_t)blockIdx.x * 2 * D + i] = (part[0][x][d] + part[1][x][d]) + (part[2][x][d] + part[3][x][d]);
  }
}

// Sums the workgroups' parts in a fixed order: 8 columns of a workgroup, 32
// threads a column, eight loads of each in flight.
template <int D>
__global__ void __launch_bounds__(256) fa_norm_dw_kernel(const NormArgs n, int blocks) {
  constexpr int P = 32, BATCH = 8;
  __shared__ float part[P][9];
  const int c = threadIdx.x & 7, p = (int)threadIdx.x >> 3;
  const int col = blockIdx.x * 8 + c;
  float sum = 0.0f;
  for (int i = p; i < blocks; i += P * BATCH) {
    float x[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
      x[j] = i + j * P < blocks ? n.ws[(int64_t)(i + j * P) * 2 * D + col] : 0.0f;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) sum += x[j];
  }
  part[p][c] = sum;
  __syncthreads();
  if (p == 0) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) total += part[i][c];
    n.dw[col / D][col % D] = total;
  }
}

template <class F>
hipError_t launch(F* fn, int64_t grid, const NormArgs& args, hipStream_t stream) {
  if (grid > 0x7fffffff) return hipErrorInvalidValue;
  void* kargs[] = {const_cast<NormArgs*>(&args)};
  return hipLaunchKernel(reinterpret_cast<const void*>(fn), dim3((unsigned)grid), dim3(256), kargs, 0,
                         stream);
}

template <int D, bool BF16, bool INTER>
hipError_t launch_fwd_as(const NormArgs& n, bool store, int64_t grid, hipStream_t stream) {
  return store ? launch(&fa_norm_kernel<D, BF16, INTER, true>, grid, n, stream)
               : launch(&fa_norm_kernel<D, BF16, INTER, false>, grid, n, stream);
}

template <int D, bool BF16, bool INTER>
hipError_t launch_bwd_as(const NormArgs& n, int blocks, hipStream_t stream) {
  const hipError_t e = launch(&fa_norm_bwd_kernel<D, BF16, INTER>, blocks, n, stream);
  if (e != hipSuccess) return e;
  int count = blocks;
  void* kargs[] = {const_cast<NormArgs*>(&n), &count};
  return hipLaunchKernel(reinterpret_cast<const void*>(&fa_norm_dw_kernel<D>), dim3(2 * D / 8), dim3(256),
                         kargs, 0, stream);
}

// f<D, BF16, INTER>(...) for runtime values.
#define FA_NORM_PICK(F, ...)                                                               \
  (n.head_dim == 128                                                                       \
       ? (bf16 ? (n.interleaved ? F<128, true, true>(__VA_ARGS__) : F<128, true, false>(__VA_ARGS__))     \
               : (n.interleaved ? F<128, false, true>(__VA_ARGS__) : F<128, false, false>(__VA_ARGS__)))  \
       : (bf16 ? (n.interleaved ? F<64, true, true>(__VA_ARGS__) : F<64, true, false>(__VA_ARGS__))       \
               : (n.interleaved ? F<64, false, true>(__VA_ARGS__) : F<64, false, false>(__VA_ARGS__))))

}  // namespace

hipError_t launch_norm(const NormArgs& args, bool bf16, bool store, int compute_units,
                       hipStream_t stream) {
  NormArgs n = args;
  const int per = 256 / (n.head_dim / 8);  // tokens of a workgroup
  const int heads = n.heads + (store ? 2 : 1) * n.kv_heads;
  n.blocks_x = (int)(((int64_t)n.tokens + per - 1) / per);
  // Heads of a lane group: all of them where that leaves four workgroups per
  // CU, else fewer (their tokens' tables are read again, from L2).
  const int64_t want = 4 * (int64_t)compute_units;
  const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>((heads + kRows - 1) / kRows,
                                                                (want + n.blocks_x - 1) / n.blocks_x));
  n.head_chunk = (int)((heads + chunks - 1) / chunks);
  n.head_chunk = (n.head_chunk + kRows - 1) / kRows * kRows;
  const int64_t grid = (int64_t)n.blocks_x * ((heads + n.head_chunk - 1) / n.head_chunk);
  return FA_NORM_PICK(launch_fwd_as, n, store, grid, stream);
}

int norm_bwd_blocks(int64_t tokens, int heads, int head_dim, int compute_units) {
  const int per = 256 / (head_dim / 8);
  const int64_t blocks = (tokens + per - 1) / per * ((heads + kBwdHeads - 1) / kBwdHeads);
  return (int)std::max<int64_t>(1, std::min<int64_t>(blocks, 4 * (int64_t)compute_units));
}

hipError_t launch_norm_bwd(const NormArgs& args, bool bf16, int compute_units, hipStream_t stream) {
  NormArgs n = args;
  n.head_chunk = kBwdHeads;
  const int blocks = norm_bwd_blocks(n.tokens, n.heads + n.kv_heads, n.head_dim, compute_units);
  return FA_NORM_PICK(launch_bwd_as, n, blocks, stream);
}

}  // namespace fa
