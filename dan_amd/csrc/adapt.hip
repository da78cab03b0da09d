// Low-rank adapters of many requests beside a shared projection, and their gradients
// (include/dan_adapt.h), for gfx950.
//
//   h = x A_i^T             out = y + c_i h B_i^T                       i = index[n], c = scale
//   g = G B_i               dx = c_i g A_i
//   dA_i = c_i sum g^T x    dB_i = c_i sum G^T h        over the rows of adapter i
//
// Two kinds of product make all of it: `down` sums over the wide side (h, g: [N, rank]) and `up` over the
// rank (out, dx); the gradients of A and B sum over rows (`outer`). All are bound by memory: x, y and out
// pass once, ranks are small.
//
// The values between two products (h, g) stay fp32 in memory and enter the second product as the sum of two
// 16-bit numbers, v = hi + lo, side by side along the product's inner dimension: it costs matrix operations,
// of which there are plenty, and keeps 16 bits or more of v. fp16 numbers are first brought near 1 by a power
// of 2 (of a row, or of a tile of rows), so that no v leaves their range.
//
// Rows of different adapters may lie in any order. A tile of 16 rows multiplies all of them by each adapter
// that occurs in it and keeps the rows that are its own by selection, not by adding zeros, so that an
// adapter that holds infinities or NaN reaches no other request's rows.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "dan_adapt.h"
#include "dan_tree_attn.h"
#include "tiles.h"

namespace dan {
int fail(int status, const char *fmt, ...);  // tree_attn.hip: sets the thread's last-error message
extern thread_local char g_err[512];

namespace {

using namespace tiles;

constexpr int kThreads = 256;
constexpr int kChunk = 128;     // values of the wide side that a wave of `down` takes at a time
constexpr int kUpCols = 256;    // columns of a work group of `up`, 64 a wave
constexpr int kOuterCols = 128; // columns of a work group of `outer`
constexpr int kOuterRows = 32;  // rows of a step of `outer`

// c += A B of a 16x16x32 product. Lane l holds row l % 16 of A (column of B) at k = 8 (l / 16) + 0..7, and of c
// column l % 16, rows 4 (l / 16) + 0..3.
template <typename T>
__device__ inline f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The power of 2 (as its exponent) that brings m into [1, 2); 0 for zeros, infinities and NaN.
__device__ inline int exponent_of(float m) { return m > 0.f && m < INFINITY ? -max(ilogbf(m), -126) : 0; }

__device__ inline int adapter_of(const int32_t *index, int n) { return index ? index[n] : 0; }

// ---------------------------------------------------------------- down: part[s][n][j] = sum over k of x[n][k] w_i[j][k]
struct DownParams {
  const void *x, *w;  // w [adapters][rank][n]
  const int32_t *index;
  float *part;  // [splits][rows][rank16]
  int64_t x_stride;
  int32_t rows, n, rank, adapters, rank16, chunks;  // chunks of kChunk values a work group
};

// 16 F rows, a range of chunks split over the four waves. A lane loads 32 contiguous bytes of a row (128 a row
// and four lanes) for two steps of the product; the order of k within a chunk is the same for both operands.
template <typename T, int JB, int F>
__global__ __launch_bounds__(kThreads) void down_kernel(const DownParams p) {
  __shared__ f32x4 red[4][JB][F][64];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const int n0 = blockIdx.x * 16 * F, first = blockIdx.y * p.chunks * kChunk, last = min(first + p.chunks * kChunk, p.n);
  int idx[F];
  const T *xr[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int n = n0 + 16 * f + l16;
    idx[f] = n < p.rows ? adapter_of(p.index, n) : -1;
    if (idx[f] >= p.adapters) idx[f] = -1;  // (`up` makes the row NaN)
    xr[f] = static_cast<const T *>(p.x) + (int64_t)min(n, p.rows - 1) * p.x_stride + 16 * g4;
  }
  f32x4 acc[JB][F];
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int f = 0; f < F; ++f) acc[jb][f] = f32x4{};
  for (int k0 = first + wave * kChunk; k0 < last; k0 += 4 * kChunk) {
    u32x4 xf[F][4];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int k = 64 * (s >> 1) + 8 * (s & 1);
        xf[f][s] = k0 + k + 16 * g4 < last ? load16(xr[f] + k0 + k) : u32x4{};
      }
    uint64_t left[F];
#pragma unroll
    for (int f = 0; f < F; ++f) left[f] = __ballot(idx[f] >= 0);
    for (;;) {  // each adapter of the tile
      int i = -1;
#pragma unroll
      for (int f = 0; f < F; ++f)
        if (i < 0 && left[f]) i = __builtin_amdgcn_readlane(idx[f], __builtin_ctzll(left[f]));
      if (i < 0) break;
      const T *w = static_cast<const T *>(p.w) + (int64_t)i * p.rank * p.n + 16 * g4 + k0;
      f32x4 t[JB][F];
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) {
        u32x4 wf[4];
        const int j = 16 * jb + l16;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int k = 64 * (s >> 1) + 8 * (s & 1);
          wf[s] = j < p.rank && k0 + k + 16 * g4 < last ? load16(w + (int64_t)j * p.n + k) : u32x4{};
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
          t[jb][f] = f32x4{};
#pragma unroll
          for (int s = 0; s < 4; ++s) t[jb][f] = mfma16<T>(wf[s], xf[f][s], t[jb][f]);
        }
      }
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const bool mine = idx[f] == i;
        left[f] &= ~__ballot(mine);
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[jb][f][e] += mine ? t[jb][f][e] : 0.f;
      }
    }
  }
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int f = 0; f < F; ++f) red[wave][jb][f][lane] = acc[jb][f];
  __syncthreads();
  for (int x = wave; x < JB * F; x += 4) {
    const int jb = x / F, f = x % F, n = n0 + 16 * f + l16;
    const f32x4 sum = (red[0][jb][f][lane] + red[1][jb][f][lane]) + (red[2][jb][f][lane] + red[3][jb][f][lane]);
    if (n < p.rows) *(DAN_TILE_GLOBAL f32x4 *)(p.part + ((int64_t)blockIdx.y * p.rows + n) * p.rank16 + 16 * jb + 4 * g4) = sum;
  }
}

// ---------------------------------------------------------------- up: out[n][m] = y[n][m] + c_i sum over j of v[n][j] w_i[m][j]
struct UpParams {
  const float *part;  // [splits][rows][rank16]
  const void *w, *y;  // w [adapters][cols][rank]; y may be NULL (zeros)
  void *out;
  const int32_t *index;
  const float *scale;
  int64_t y_stride, o_stride;
  int32_t rows, cols, rank, adapters, rank16, splits;
  float scale_value;
};

// 16 F rows by 256 columns: a wave takes 64 columns, of which a lane owns 16 contiguous ones of its row (128 bytes a
// row and four lanes): the product's row r of block b is column 16 (r / 4) + 4 b + r % 4. The inner dimension holds
// v's hi parts, then its lo parts, in pieces of 8: ST steps of four pieces.
template <typename T, int ST, int F>
__global__ __launch_bounds__(kThreads) void up_kernel(const UpParams p) {
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const int n0 = blockIdx.y * 16 * F, m0 = blockIdx.x * kUpCols + wave * 64;
  if (m0 >= p.cols) return;
  const int r8 = p.rank / 8, m = m0 + 16 * g4;
  u32x4 yv[F][2];
  int idx[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int n = n0 + 16 * f + l16;
    idx[f] = n < p.rows ? adapter_of(p.index, n) : -1;
#pragma unroll
    for (int h = 0; h < 2; ++h)
      yv[f][h] = p.y && n < p.rows && m + 8 * h < p.cols ? load16(static_cast<const T *>(p.y) + n * p.y_stride + m + 8 * h) : u32x4{};
  }
  int have = -1;  // the adapter whose B the wave holds
  u32x4 wf[ST][4];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int n = n0 + 16 * f + l16;
    if (n0 + 16 * f >= p.rows) break;
    f32x4 acc[4];
    {
      const f32x8 a = unpack8<T>(yv[f][0]), b = unpack8<T>(yv[f][1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc[0][e] = a[e];
        acc[1][e] = a[4 + e];
        acc[2][e] = b[e];
        acc[3][e] = b[4 + e];
      }
    }
    uint64_t left = __ballot(idx[f] >= 0);
    if (left) {
      // v's pieces of this lane, as hi or lo parts
      f32x8 v[ST];
      float top = 0.f;
#pragma unroll
      for (int t = 0; t < ST; ++t) {
        const int u = 4 * t + g4, j = 8 * (u >= r8 ? u - r8 : u);
        v[t] = f32x8{};
        if (u < 2 * r8 && n < p.rows)
          for (int s = 0; s < p.splits; ++s) {
            const float *at = p.part + ((int64_t)s * p.rows + n) * p.rank16 + j;
            const f32x4 a = *(const DAN_TILE_GLOBAL f32x4 *)at, b = *(const DAN_TILE_GLOBAL f32x4 *)(at + 4);
            v[t] += __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
          }
        if (kHalf)
#pragma unroll
          for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[t][e]));
      }
      int e2 = 0;
      if (kHalf) {
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        e2 = exponent_of(top);
      }
      u32x4 vf[ST];
#pragma unroll
      for (int t = 0; t < ST; ++t) {
        f32x8 x = v[t];
        if (kHalf)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = ldexpf(x[e], e2);
        const u32x4 hi = pack8<T>(x);
        vf[t] = 4 * t + g4 >= r8 ? pack8<T>(x - unpack8<T>(hi)) : hi;
      }
      while (left) {
        const int i = __builtin_amdgcn_readlane(idx[f], __builtin_ctzll(left));
        const bool mine = idx[f] == i;
        left &= ~__ballot(mine);
        if (i >= p.adapters) {  // no such adapter
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[b][e] = mine ? NAN : acc[b][e];
          continue;
        }
        if (i != have) {
          have = i;
          const T *w = static_cast<const T *>(p.w) + (int64_t)i * p.cols * p.rank;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int col = m0 + 16 * (l16 >> 2) + 4 * b + (l16 & 3);
#pragma unroll
            for (int t = 0; t < ST; ++t) {
              const int u = 4 * t + g4, j = 8 * (u >= r8 ? u - r8 : u);
              wf[t][b] = u < 2 * r8 && col < p.cols ? load16(w + (int64_t)col * p.rank + j) : u32x4{};
            }
          }
        }
        const float ci = p.scale ? p.scale[i] : p.scale_value, c = kHalf ? ldexpf(ci, -e2) : ci;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          f32x4 t4 = {};
#pragma unroll
          for (int t = 0; t < ST; ++t) t4 = mfma16<T>(wf[t][b], vf[t], t4);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[b][e] = mine ? fmaf(c, t4[e], acc[b][e]) : acc[b][e];
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (n < p.rows && m + 8 * h < p.cols)
        store16(static_cast<T *>(p.out) + n * p.o_stride + m + 8 * h, pack8<T>(__builtin_shufflevector(acc[2 * h], acc[2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7)));
  }
}

// ---------------------------------------------------------------- outer: d_i[j][c] = c_i sum over the rows of i of v[n][j] z[n][c]
struct OuterSide {
  const float *part;  // v [splits][rows][rank16]
  const void *z;
  int64_t z_stride;
  float *sums;  // [parts][adapters][rank * cols]
  int32_t cols, splits, tiles;
};
struct OuterParams {
  OuterSide a, b;  // dA [rank][n_in] of (g, x); dB [n_out][rank] of (h, G)
  const int32_t *index;
  const float *scale;
  int32_t rows, rank, rank16, adapters, part_rows;  // rows of a part
  float scale_value;
};

// One adapter, one part of the rows, 128 columns. The rows of the part that are the adapter's are listed in order;
// the waves take 32 of them in turn, each through a tile of its own in LDS, from where the transposing reads make the
// operand whose inner dimension is the rows. v's operand is loaded in place (a lane's 8 rows).
template <typename T, int JB>
__global__ __launch_bounds__(kThreads) void outer_kernel(const OuterParams p) {
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  using Tl = Tile<kOuterCols>;
  constexpr int CB = kOuterCols / 16;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lds = (uint32_t)(uintptr_t)(DAN_TILE_LDS uint8_t *)smem;
  __shared__ int counts[4];
  int32_t *list = reinterpret_cast<int32_t *>(smem + 4 * Tl::bytes);
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const bool side_b = (int)blockIdx.x >= p.a.tiles;
  const OuterSide &q = side_b ? p.b : p.a;
  const int c0 = ((int)blockIdx.x - (side_b ? p.a.tiles : 0)) * kOuterCols, i = blockIdx.y, part = blockIdx.z;
  const int r0 = part * p.part_rows, r1 = min(r0 + p.part_rows, p.rows);

  int count = 0;
  for (int base = r0; base < r1; base += kThreads) {
    const int n = base + threadIdx.x;
    const bool mine = n < r1 && adapter_of(p.index, n) == i;
    const uint64_t votes = __ballot(mine);
    __syncthreads();
    if (lane == 0) counts[wave] = __popcll(votes);
    __syncthreads();
    int at = count;
    for (int w = 0; w < wave; ++w) at += counts[w];
    if (mine) list[at + __popcll(votes & ((1ull << lane) - 1))] = n;
    count += counts[0] + counts[1] + counts[2] + counts[3];
  }
  __syncthreads();
  count = uni(count);

  f32x4 acc[JB][CB];
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) acc[jb][cb] = f32x4{};
  const uint32_t tile = lds + (uint32_t)(wave * Tl::bytes);
  const T *z = static_cast<const T *>(q.z) + (int64_t)r0 * q.z_stride + c0;
  const int left = min(kOuterCols, q.cols - c0);  // columns of the tile (a multiple of 8)
  for (int s0 = wave * kOuterRows; s0 < count; s0 += 4 * kOuterRows) {
    barrier_wave_lds();  // (the last step's reads of the tile)
#pragma unroll
    for (int x = 0; x < Tl::blocks; ++x) {
      const int n = list[min(s0 + Tl::block_row(x, lane), count - 1)];
      dma16(z, (uint32_t)(n - r0) * (uint32_t)(2 * q.z_stride) + min(Tl::block_byte(x, lane), (uint32_t)(2 * left - 16)), tile + (uint32_t)(x * 1024));
    }
    float v[JB][8];
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = s0 + 8 * g4 + e;
      const int n = list[min(at, count - 1)];
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) {
        v[jb][e] = 0.f;
        if (at < count)
          for (int s = 0; s < q.splits; ++s) v[jb][e] += q.part[((int64_t)s * p.rows + n) * p.rank16 + 16 * jb + l16];
        if (kHalf) top = fmaxf(top, fabsf(v[jb][e]));
      }
    }
    int e2 = 0;
    if (kHalf) {
#pragma unroll
      for (int m = 32; m; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
      e2 = exponent_of(top);
    }
    u32x4 hi[JB], lo[JB];
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
      f32x8 x;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = kHalf ? ldexpf(v[jb][e], e2) : v[jb][e];
      hi[jb] = pack8<T>(x);
      lo[jb] = pack8<T>(x - unpack8<T>(hi[jb]));
    }
    const float back = kHalf ? ldexpf(1.f, -e2) : 1.f;
    wait_vmem<0>();
    // (rows past the list are copies of its last one, and v is 0 there: not so where that row holds infinities)
    const int rows = min(count - s0, kOuterRows);
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      u32x4 zf;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 8 * g4 + 4 * h + (l16 >> 2);
        const uint32_t at = tile + (uint32_t)(r * Tl::row + (((2 * cb + ((l16 >> 1) & 1)) ^ Tl::swizzle(r)) << 4) + 8 * (l16 & 1));
        const u32x2 t = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((DAN_TILE_LDS i16x4 *)(uintptr_t)at));
        zf[2 * h] = t[0];
        zf[2 * h + 1] = t[1];
      }
      if (rows < kOuterRows) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (8 * g4 + e >= rows) zf[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
      }
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) {
        f32x4 t = kHalf ? f32x4{} : acc[jb][cb];
        t = side_b ? mfma16<T>(hi[jb], zf, t) : mfma16<T>(zf, hi[jb], t);
        t = side_b ? mfma16<T>(lo[jb], zf, t) : mfma16<T>(zf, lo[jb], t);
        if (kHalf)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[jb][cb][e] = fmaf(back, t[e], acc[jb][cb][e]);
        else acc[jb][cb] = t;
      }
    }
  }
  // The waves' sums, added in order.
  f32x4 *red = reinterpret_cast<f32x4 *>(smem);
  const float c = p.scale ? p.scale[i] : p.scale_value;
  float *to = q.sums + ((int64_t)part * p.adapters + i) * p.rank * q.cols;
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int cb = 0; cb < CB / 2; ++cb) red[(wave * (CB / 2) + cb) * 64 + lane] = acc[jb][half * (CB / 2) + cb];
      __syncthreads();
      const f32x4 sum = (red[wave * 64 + lane] + red[(CB / 2 + wave) * 64 + lane]) + (red[(CB + wave) * 64 + lane] + red[(3 * CB / 2 + wave) * 64 + lane]);
      const int cb = half * (CB / 2) + wave, row = 4 * g4;
      if (side_b) {  // lane: column l16, ranks row..
        if (c0 + 16 * cb + l16 < q.cols && 16 * jb + row < p.rank)
          *(DAN_TILE_GLOBAL f32x4 *)(to + (int64_t)(c0 + 16 * cb + l16) * p.rank + 16 * jb + row) = sum * c;
      } else {  // lane: rank l16, columns row..
        if (c0 + 16 * cb + row < q.cols && 16 * jb + l16 < p.rank)
          *(DAN_TILE_GLOBAL f32x4 *)(to + (int64_t)(16 * jb + l16) * q.cols + c0 + 16 * cb + row) = sum * c;
      }
    }
}

// The parts of dA and dB added up in order, rounded once: 8 values a thread.
struct SumParams {
  const float *a, *b;
  void *da, *db;
  int64_t na, nb;  // values of dA, dB (multiples of 8)
  int32_t parts;
};
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_kernel(const SumParams p) {
  int64_t at = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  const bool b = at >= p.na;
  if (b) at -= p.na;
  const int64_t n = b ? p.nb : p.na;
  if (at >= n) return;
  const float *from = (b ? p.b : p.a) + at;
  f32x4 x = {}, y = {};
  for (int i = 0; i < p.parts; ++i, from += n) {
    x += *(const DAN_TILE_GLOBAL f32x4 *)from;
    y += *(const DAN_TILE_GLOBAL f32x4 *)(from + 4);
  }
  store16(static_cast<T *>(b ? p.db : p.da) + at, pack8<T>(__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)));
}

// ---------------------------------------------------------------- transposes of A [R][rank][n_in] and B [R][n_out][rank], 16-bit
struct TurnParams {
  const uint16_t *a, *b;
  uint16_t *at, *bt;  // [R][n_in][rank], [R][rank][n_out]
  int32_t rank, n_in, n_out, adapters, a_tiles, b_tiles;  // tiles of 64 columns an adapter
};
// 64 positions of the wide side and all ranks a work group.
__global__ __launch_bounds__(kThreads) void turn_kernel(const TurnParams p) {
  __shared__ uint16_t tile[DAN_ADAPT_MAX_RANK][64 + 2];
  int x = blockIdx.x;
  const bool b = x >= p.a_tiles * p.adapters;
  if (b) x -= p.a_tiles * p.adapters;
  const int tiles = b ? p.b_tiles : p.a_tiles, i = x / tiles, c0 = x % tiles * 64, wide = b ? p.n_out : p.n_in;
  const int64_t base = (int64_t)i * p.rank * wide;
  const int cols = min(64, wide - c0);
  for (int e = threadIdx.x; e < 64 * p.rank; e += kThreads) {  // A: columns contiguous; B: ranks
    const int j = b ? e % p.rank : e / 64, c = b ? e / p.rank : e % 64;
    if (c < cols) tile[j][c] = b ? p.b[base + (int64_t)(c0 + c) * p.rank + j] : p.a[base + (int64_t)j * wide + c0 + c];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 64 * p.rank; e += kThreads) {
    const int j = b ? e / 64 : e % p.rank, c = b ? e % 64 : e / p.rank;
    if (c >= cols) continue;
    if (b) p.bt[base + (int64_t)j * wide + c0 + c] = tile[j][c];
    else p.at[base + (int64_t)(c0 + c) * p.rank + j] = tile[j][c];
  }
}

// ---------------------------------------------------------------- host
// Ranks as the kernels are built for: 16, 32, 64 or 128.
int rank16(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }
int down_frags(int rows) { return rows > 512 ? 2 : 1; }

// Parts of `down`'s sum: as many work groups as fill the chip a few times over, at least one chunk a wave.
int splits_of(int rows, int n) {
  const int tiles = (rows + 16 * down_frags(rows) - 1) / (16 * down_frags(rows)), chunks = (n + kChunk - 1) / kChunk;
  return std::max(1, std::min({(1024 + tiles - 1) / tiles, (chunks + 3) / 4, 16}));
}
// Parts of `outer`'s rows.
int parts_of(int rows, int n_in, int n_out, int adapters) {
  const int64_t groups = (int64_t)((n_in + kOuterCols - 1) / kOuterCols + (n_out + kOuterCols - 1) / kOuterCols) * adapters;
  const int by_rows = (rows + 4 * kOuterRows - 1) / (4 * kOuterRows);
  return (int)std::max<int64_t>({1, std::min<int64_t>({(2048 + groups - 1) / groups, by_rows, 16}), (rows + 8191) / 8192});
}
int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

template <typename T, int JB>
hipError_t launch_down(const DownParams &p, int splits, hipStream_t s) {
  const int f = down_frags(p.rows);
  const dim3 grid((p.rows + 16 * f - 1) / (16 * f), splits);
  if (f == 2) hipLaunchKernelGGL((down_kernel<T, JB, 2>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((down_kernel<T, JB, 1>), grid, dim3(kThreads), 0, s, p);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_down(DownParams p, int splits, hipStream_t s) {
  const int chunks = (p.n + kChunk - 1) / kChunk;
  p.chunks = (chunks + splits - 1) / splits;
  const int jb = p.rank16 / 16;
  return jb <= 1 ? launch_down<T, 1>(p, splits, s) : jb <= 2 ? launch_down<T, 2>(p, splits, s) : jb <= 4 ? launch_down<T, 4>(p, splits, s) : launch_down<T, 8>(p, splits, s);
}

template <typename T, int ST>
hipError_t launch_up(const UpParams &p, hipStream_t s) {
  const int cols = (p.cols + kUpCols - 1) / kUpCols;
  if (p.rows > 512) hipLaunchKernelGGL((up_kernel<T, ST, 4>), dim3(cols, (p.rows + 63) / 64), dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((up_kernel<T, ST, 1>), dim3(cols, (p.rows + 15) / 16), dim3(kThreads), 0, s, p);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_up(const UpParams &p, hipStream_t s) {
  const int steps = (p.rank / 8 + 1) / 2;
  return steps <= 1 ? launch_up<T, 1>(p, s) : steps <= 2 ? launch_up<T, 2>(p, s) : steps <= 4 ? launch_up<T, 4>(p, s) : launch_up<T, 8>(p, s);
}

template <typename T, int JB>
hipError_t launch_outer(const OuterParams &p, int parts, hipStream_t s) {
  const int bytes = std::max(4 * Tile<kOuterCols>::bytes + p.part_rows * 4, 4 * (kOuterCols / 32) * 64 * 16);
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(outer_kernel<T, JB>), hipFuncAttributeMaxDynamicSharedMemorySize, 96 * 1024);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL((outer_kernel<T, JB>), dim3(p.a.tiles + p.b.tiles, p.adapters, parts), dim3(kThreads), bytes, s, p);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_outer(const OuterParams &p, int parts, hipStream_t s) {
  const int jb = p.rank16 / 16;
  return jb <= 1 ? launch_outer<T, 1>(p, parts, s) : jb <= 2 ? launch_outer<T, 2>(p, parts, s) : jb <= 4 ? launch_outer<T, 4>(p, parts, s) : launch_outer<T, 8>(p, parts, s);
}

template <typename T>
hipError_t forward(const DanAdaptArgs &a, hipStream_t s) {
  DownParams d;
  d.x = a.x; d.x_stride = a.x_stride; d.w = a.a; d.index = a.index; d.part = a.down;
  d.rows = a.rows; d.n = a.n_in; d.rank = a.rank; d.adapters = a.adapters; d.rank16 = rank16(a.rank);
  hipError_t err = launch_down<T>(d, a.splits, s);
  if (err != hipSuccess) return err;
  UpParams u;
  u.part = a.down; u.w = a.b; u.y = a.y; u.y_stride = a.y_stride; u.out = a.out; u.o_stride = a.out_stride; u.index = a.index; u.scale = a.scale;
  u.rows = a.rows; u.cols = a.n_out; u.rank = a.rank; u.adapters = a.adapters; u.rank16 = rank16(a.rank); u.splits = a.splits; u.scale_value = a.scale_value;
  return launch_up<T>(u, s);
}

// The workspace of the gradient: A^T, B^T, g's parts, and the parts of dA and dB.
struct GradSpace {
  int64_t at, bt, down, da, db, total;
  int splits, parts;
  GradSpace(int rows, int n_in, int n_out, int rank, int adapters) {
    splits = splits_of(rows, n_out);
    parts = parts_of(rows, n_in, n_out, adapters);
    at = 0;
    bt = align256(at + (int64_t)adapters * rank * n_in * 2);
    down = align256(bt + (int64_t)adapters * rank * n_out * 2);
    da = align256(down + (int64_t)splits * rows * rank16(rank) * 4);
    db = align256(da + (int64_t)parts * adapters * rank * n_in * 4);
    total = align256(db + (int64_t)parts * adapters * rank * n_out * 4);
  }
};

template <typename T>
hipError_t backward(const DanAdaptGradArgs &a, const GradSpace &w, hipStream_t s) {
  uint8_t *ws = static_cast<uint8_t *>(a.workspace);
  TurnParams t;
  t.a = static_cast<const uint16_t *>(a.a); t.b = static_cast<const uint16_t *>(a.b);
  t.at = reinterpret_cast<uint16_t *>(ws + w.at); t.bt = reinterpret_cast<uint16_t *>(ws + w.bt);
  t.rank = a.rank; t.n_in = a.n_in; t.n_out = a.n_out; t.adapters = a.adapters;
  t.a_tiles = a.dx ? (a.n_in + 63) / 64 : 0;
  t.b_tiles = (a.n_out + 63) / 64;
  hipLaunchKernelGGL(turn_kernel, dim3((t.a_tiles + t.b_tiles) * a.adapters), dim3(kThreads), 0, s, t);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  DownParams d;
  d.x = a.g; d.x_stride = a.g_stride; d.w = t.bt; d.index = a.index; d.part = reinterpret_cast<float *>(ws + w.down);
  d.rows = a.rows; d.n = a.n_out; d.rank = a.rank; d.adapters = a.adapters; d.rank16 = rank16(a.rank);
  if ((err = launch_down<T>(d, w.splits, s)) != hipSuccess) return err;
  if (a.dx) {
    UpParams u;
    u.part = d.part; u.w = t.at; u.y = nullptr; u.y_stride = 0; u.out = a.dx; u.o_stride = a.dx_stride; u.index = a.index; u.scale = a.scale;
    u.rows = a.rows; u.cols = a.n_in; u.rank = a.rank; u.adapters = a.adapters; u.rank16 = d.rank16; u.splits = w.splits; u.scale_value = a.scale_value;
    if ((err = launch_up<T>(u, s)) != hipSuccess) return err;
  }
  if (!a.da && !a.db) return hipSuccess;
  OuterParams o;
  o.a = {d.part, a.x, a.x_stride, reinterpret_cast<float *>(ws + w.da), a.n_in, w.splits, a.da ? (a.n_in + kOuterCols - 1) / kOuterCols : 0};
  o.b = {a.down, a.g, a.g_stride, reinterpret_cast<float *>(ws + w.db), a.n_out, a.splits, a.db ? (a.n_out + kOuterCols - 1) / kOuterCols : 0};
  o.index = a.index; o.scale = a.scale; o.rows = a.rows; o.rank = a.rank; o.rank16 = d.rank16; o.adapters = a.adapters;
  o.part_rows = (a.rows + w.parts - 1) / w.parts; o.scale_value = a.scale_value;
  if ((err = launch_outer<T>(o, w.parts, s)) != hipSuccess) return err;
  SumParams m;
  m.a = o.a.sums; m.b = o.b.sums; m.da = a.da; m.db = a.db; m.parts = w.parts;
  m.na = a.da ? (int64_t)a.adapters * a.rank * a.n_in : 0;
  m.nb = a.db ? (int64_t)a.adapters * a.rank * a.n_out : 0;
  hipLaunchKernelGGL(sum_kernel<T>, dim3((uint32_t)(((m.na + m.nb) / 8 + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, m);
  return hipGetLastError();
}

// A launch holds fewer than 2^32 threads.
bool too_many(int64_t groups) { return groups * kThreads >= int64_t(1) << 32; }
int64_t over(int64_t x, int64_t by) { return (x + by - 1) / by; }

int check_sizes(int dtype, int rows, int n_in, int n_out, int rank, int adapters, float scale_value) {
  if (dtype != DAN_DTYPE_BF16 && dtype != DAN_DTYPE_F16) return fail(DAN_ERR_UNSUPPORTED, "dtype %d: bf16 or fp16", dtype);
  if (rows < 0 || rows > 1 << 20) return fail(DAN_ERR_UNSUPPORTED, "rows %d: at most 2^20", rows);
  if (n_in <= 0 || n_out <= 0 || n_in % 8 || n_out % 8 || n_in > 1 << 20 || n_out > 1 << 20)
    return fail(DAN_ERR_UNSUPPORTED, "n_in %d and n_out %d: multiples of 8 up to 2^20", n_in, n_out);
  if (rank <= 0 || rank % 8 || rank > DAN_ADAPT_MAX_RANK) return fail(DAN_ERR_UNSUPPORTED, "rank %d: a multiple of 8 up to %d", rank, DAN_ADAPT_MAX_RANK);
  if (adapters <= 0 || adapters > 65535) return fail(DAN_ERR_UNSUPPORTED, "%d adapters: 1 to 65535", adapters);
  if (!(isfinite(scale_value))) return fail(DAN_ERR_INVALID_ARGUMENT, "scale_value must be finite");
  const int64_t wide = std::max(n_in, n_out), f = rows > 512 ? 64 : 16;
  if (too_many(over(wide, kUpCols) * over(rows, f)) || too_many(over(rows, 16) * splits_of(rows, (int)wide)) ||
      too_many((over(n_in, kOuterCols) + over(n_out, kOuterCols)) * adapters * std::max(2, parts_of(rows, n_in, n_out, adapters))) ||
      too_many(over((int64_t)adapters * rank * ((int64_t)n_in + n_out), 8 * kThreads)))
    return fail(DAN_ERR_UNSUPPORTED, "%d rows, %d to %d, %d adapters: more than one launch holds", rows, n_in, n_out, adapters);
  return DAN_OK;
}
bool bad_rows(const void *p, int64_t stride) { return ((uintptr_t)p & 15) || stride % 8 || stride < 0; }

}  // namespace
}  // namespace dan

extern "C" {

int dan_adapt_abi_version(void) { return DAN_ADAPT_ABI_VERSION; }

int32_t dan_adapt_splits(int32_t rows, int32_t n) { return rows <= 0 || n <= 0 ? 1 : dan::splits_of(rows, n); }

int64_t dan_adapt_grad_workspace_size(int32_t rows, int32_t n_in, int32_t n_out, int32_t rank, int32_t adapters) {
  using namespace dan;
  if (rows <= 0 || check_sizes(DAN_DTYPE_BF16, rows, n_in, n_out, rank, adapters, 0.f) != DAN_OK) return 0;
  return GradSpace(rows, n_in, n_out, rank, adapters).total;
}

int dan_adapt(const DanAdaptArgs *a, void *stream) {
  using namespace dan;
  g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->abi_version != DAN_ADAPT_ABI_VERSION)
    return fail(DAN_ERR_VERSION, "abi_version %d, library speaks %d", a->abi_version, DAN_ADAPT_ABI_VERSION);
  if (const int rc = check_sizes(a->dtype, a->rows, a->n_in, a->n_out, a->rank, a->adapters, a->scale_value)) return rc;
  if (a->splits != dan_adapt_splits(a->rows, a->n_in)) return fail(DAN_ERR_INVALID_ARGUMENT, "splits %d: dan_adapt_splits", a->splits);
  if (a->rows == 0) return DAN_OK;
  if (!a->x || !a->y || !a->a || !a->b || !a->out || !a->down) return fail(DAN_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (bad_rows(a->x, a->x_stride) || bad_rows(a->y, a->y_stride) || bad_rows(a->out, a->out_stride) || (a->rows > 1 && a->out_stride < a->n_out) ||
      (((uintptr_t)a->a | (uintptr_t)a->b | (uintptr_t)a->down) & 15))
    return fail(DAN_ERR_INVALID_ARGUMENT, "rows must start 16-byte aligned, and written ones must not overlap");
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = a->dtype == DAN_DTYPE_BF16 ? forward<__bf16>(*a, s) : forward<_Float16>(*a, s);
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "adapter launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

int dan_adapt_grad(const DanAdaptGradArgs *a, void *stream) {
  using namespace dan;
  g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->abi_version != DAN_ADAPT_ABI_VERSION)
    return fail(DAN_ERR_VERSION, "abi_version %d, library speaks %d", a->abi_version, DAN_ADAPT_ABI_VERSION);
  if (const int rc = check_sizes(a->dtype, a->rows, a->n_in, a->n_out, a->rank, a->adapters, a->scale_value)) return rc;
  if (a->splits != dan_adapt_splits(a->rows, a->n_in)) return fail(DAN_ERR_INVALID_ARGUMENT, "splits %d: dan_adapt_splits", a->splits);
  if (a->rows == 0) return DAN_OK;
  if (!a->x || !a->g || !a->a || !a->b || !a->down) return fail(DAN_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (bad_rows(a->x, a->x_stride) || bad_rows(a->g, a->g_stride) || bad_rows(a->dx, a->dx ? a->dx_stride : 0) ||
      (a->dx && a->rows > 1 && a->dx_stride < a->n_in) ||
      (((uintptr_t)a->a | (uintptr_t)a->b | (uintptr_t)a->da | (uintptr_t)a->db | (uintptr_t)a->down) & 15))
    return fail(DAN_ERR_INVALID_ARGUMENT, "rows must start 16-byte aligned, and written ones must not overlap");
  const GradSpace w(a->rows, a->n_in, a->n_out, a->rank, a->adapters);
  if (!a->workspace || a->workspace_bytes < w.total || ((uintptr_t)a->workspace & 255))
    return fail(DAN_ERR_INVALID_ARGUMENT, "workspace needs %lld bytes, 256-byte aligned", (long long)w.total);
  // `outer` keeps a row's offset from its part's first one in 32 bits.
  const int64_t part_rows = (a->rows + w.parts - 1) / w.parts;
  if (part_rows * a->x_stride * 2 >= int64_t(1) << 32 || part_rows * a->g_stride * 2 >= int64_t(1) << 32)
    return fail(DAN_ERR_UNSUPPORTED, "row strides %lld and %lld are too large", (long long)a->x_stride, (long long)a->g_stride);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = a->dtype == DAN_DTYPE_BF16 ? backward<__bf16>(*a, w, s) : backward<_Float16>(*a, w, s);
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "adapter gradient launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

}  // extern "C"
