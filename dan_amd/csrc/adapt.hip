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
// of which there are plenty, and keeps 16 bits or more of v; an infinite v is hi alone. fp16 numbers are first brought to the upper end
// of their range by a power of 2 (of a row, or of a tile of rows): no v leaves it there, and one that is 2^-22 of the largest still has
// its 16 bits.
//
// Measured, 8192 rows, one adapter of rank 16, 4096 -> 28672: down 21 us (67 MB), up 205 us (940 MB, 4.6 TB/s); gradients: g and dB in one
// pass 100 us (500 MB, 5 TB/s; in two, 130 + 83), g's parts 7, up 20, dA 19, the parts' sum 8. 64 rows of 24 adapters, 4096 -> 4096: 5 + 5 us, launches
// and chains of index, weights and sums; 1037 rows, 5 adapters of rank 64, 4096 -> 4096, fp16: down 14, up 10.5, outer 26 (the same
// chains: 1024 values instead of 4096 take down 13.4 us). Gradients of 2 rows of rank 4, 4096 -> 4096: six launches of 2.5 to 5 us each.
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
constexpr int kChunk = 128;      // values of the wide side that a wave of `down` takes at a time
constexpr int kUpCols = 64;      // columns of a wave of `up`
constexpr int kOuterCols = 128;  // columns of a work group of `outer`
constexpr int kOuterRows = 32;   // rows of a step of `outer`
// Bytes of G from which dB and g come from one pass. Backward passes of one adapter, 4096 wide, one pass / two, us: 8192 x 4096 (64 MB) 82 / 79,
// 2048 x 28672 (112 MB) 64 / 71, 8192 x 14336 (224 MB) 107 / 148, 8192 x 28672 (448 MB) 160 / 263: what the caches keep is cheap to read twice.
constexpr int64_t kBothBytes = 96 << 20;

// c += A B of a 16x16x32 product. Lane l holds row l % 16 of A (column of B) at k = 8 (l / 16) + 0..7, and of c
// column l % 16, rows 4 (l / 16) + 0..3.
template <typename T>
__device__ inline f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (std::is_same<T, __bf16>::value)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// What 8 values leave of themselves when they are rounded to `hi`; zeros where that is infinite, whose sum with them it stays.
template <typename T>
__device__ inline u32x4 low_part(f32x8 x, u32x4 hi) {
  x -= unpack8<T>(hi);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = fabsf(x[e]) < INFINITY ? x[e] : 0.f;
  return pack8<T>(x);
}
// |x|, or 0 for infinities and NaN: they have no part in a power of 2.
__device__ inline float finite_size(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }

// The power of 2 (as its exponent) that brings m into [2^14, 2^15), or as far as its inverse is a normal number; 0 for zeros.
__device__ inline int exponent_of(float m) { return m > 0.f ? min(14 - ilogbf(m), 126) : 0; }

__device__ inline int adapter_of(const int32_t *index, int n) { return index ? index[n] : 0; }

// The next adapter of a tile whose lanes' rows have the adapters `idx` and are not done yet (`left`), or -1.
__device__ inline int next_adapter(int idx, uint64_t left) { return left ? __builtin_amdgcn_readlane(idx, __builtin_ctzll(left)) : -1; }

// ---------------------------------------------------------------- down: part[s][n][j] = sum over k of x[n][k] w_i[j][k]
struct DownParams {
  const void *x, *w;  // w [adapters][rank][n]
  const int32_t *index;
  float *part;  // [splits][rows][ranks]
  int64_t x_stride;
  int32_t rows, n, rank, adapters, ranks, chunks;  // ranks: 16, 32, 64 or 128; chunks of kChunk values a work group
};

// Rows as operands: 16 F of them, four steps of 32 values from k0 on. A lane loads 16 bytes, four lanes 64 of a row.
// (Here and below every load is made, at a clamped place where there is none to make: a load under a condition of
// its own is a branch, and waits for the ones before it. Values past the row's end become zeros in x and in w: either's last ones
// may be infinite.)
template <typename T, int F>
__device__ inline void load_rows(const T *const (&row)[F], int k0, int last, int g4, u32x4 (&to)[F][4]) {
#pragma unroll
  for (int f = 0; f < F; ++f)
#pragma unroll
    for (int s = 0; s < 4; ++s) to[f][s] = load16(row[f] + min(k0 + 32 * s + 8 * g4, last - 8));
  if (k0 + kChunk > last)
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (k0 + 32 * s + 8 * g4 >= last) to[f][s] = u32x4{};
}
// One chunk of adapter i's w (ranks past the last one: copies of it, never used).
template <typename T, int JB>
__device__ inline void load_chunk(const DownParams &p, int i, int k0, int last, int l16, int g4, u32x4 (&wf)[JB][4]) {
  const T *w = static_cast<const T *>(p.w) + (int64_t)i * p.rank * p.n;
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int s = 0; s < 4; ++s) wf[jb][s] = load16(w + (int64_t)min(16 * jb + l16, p.rank - 1) * p.n + min(k0 + 32 * s + 8 * g4, last - 8));
  if (k0 + kChunk > last)
#pragma unroll
    for (int jb = 0; jb < JB; ++jb)
#pragma unroll
      for (int s = 0; s < 4; ++s)
        if (k0 + 32 * s + 8 * g4 >= last) wf[jb][s] = u32x4{};
}
// t += w x^T over it.
template <typename T, int JB, int F>
__device__ inline void chunk_product(const u32x4 (&wf)[JB][4], const u32x4 (&xf)[F][4], f32x4 (&t)[JB][F]) {
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int s = 0; s < 4; ++s) t[jb][f] = mfma16<T>(wf[jb][s], xf[f][s], t[jb][f]);
}

// Both, for ranks up to 128, whose w fills the registers: zeros past the row's end (as load_chunk makes them) a rank block at a time,
// in a chunk that has any. (Behind all of w's loads they would hold all of it at once: 4096 rows, 4096 -> 4096, rank 128, 61.3 us, and 57.4 so.)
template <typename T, int JB, int F>
__device__ inline void chunk_at_once(const DownParams &p, int i, int k0, int last, int l16, int g4, const u32x4 (&xf)[F][4], f32x4 (&t)[JB][F]) {
  const T *w = static_cast<const T *>(p.w) + (int64_t)i * p.rank * p.n;
  if (k0 + kChunk <= last) {
    u32x4 wf[JB][4];
#pragma unroll
    for (int jb = 0; jb < JB; ++jb)
#pragma unroll
      for (int s = 0; s < 4; ++s) wf[jb][s] = load16(w + (int64_t)min(16 * jb + l16, p.rank - 1) * p.n + k0 + 32 * s + 8 * g4);
    chunk_product<T, JB, F>(wf, xf, t);
    return;
  }
#pragma unroll
  for (int jb = 0; jb < JB; ++jb) {
    u32x4 wf[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) wf[s] = load16(w + (int64_t)min(16 * jb + l16, p.rank - 1) * p.n + min(k0 + 32 * s + 8 * g4, last - 8));
#pragma unroll
    for (int s = 0; s < 4; ++s)
      if (k0 + 32 * s + 8 * g4 >= last) wf[s] = u32x4{};
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int s = 0; s < 4; ++s) t[jb][f] = mfma16<T>(wf[s], xf[f][s], t[jb][f]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Many rows: 32 a work group, whose W waves split the chunks and add up over LDS. Work groups begin at different chunks:
// where a row's bytes are a multiple of a large power of 2, all of them at one place of their rows ask few channels of the memory.
// Neighbours in the grid are the splits of a tile of rows, so that a die reads few of w's columns.
template <int JB>
constexpr int kDownWaves = JB <= 2 ? 16 : 8;  // (1024 threads leave 128 registers each)
template <typename T, int JB>
__global__ __launch_bounds__(64 * kDownWaves<JB>) void down_kernel(const DownParams p) {
  constexpr int F = 2, W = kDownWaves<JB>;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  f32x4 *red = reinterpret_cast<f32x4 *>(smem);  // [W / 2][JB * F][64]
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const int n0 = blockIdx.y * 16 * F, first = blockIdx.x * p.chunks * kChunk, last = min(first + p.chunks * kChunk, p.n);
  int idx[F];
  const T *xr[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int n = n0 + 16 * f + l16;
    idx[f] = n < p.rows ? adapter_of(p.index, n) : -1;
    if (idx[f] >= p.adapters) idx[f] = -1;  // (`up` makes the row NaN)
    xr[f] = static_cast<const T *>(p.x) + (int64_t)min(n, p.rows - 1) * p.x_stride;
  }
  f32x4 acc[JB][F];
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int f = 0; f < F; ++f) acc[jb][f] = f32x4{};
  constexpr bool kAhead = JB < 8;  // the first adapter's w is loaded with the rows (at rank 128 the registers do not hold both)
  const uint64_t own[F] = {__ballot(idx[0] >= 0), __ballot(idx[1] >= 0)};
  const int i0 = own[0] ? next_adapter(idx[0], own[0]) : next_adapter(idx[1], own[1]);
  const int begin = first + wave * kChunk, turns = (last - begin + W * kChunk - 1) / (W * kChunk);  // (0 or fewer: no chunk)
  for (int turn = 0, at = turns > 0 ? blockIdx.y % turns : 0; turn < turns; ++turn, at = at + 1 < turns ? at + 1 : 0) {
    const int k0 = begin + at * W * kChunk;
    u32x4 xf[F][4];
    u32x4 wf[JB][4];
    load_rows<T, F>(xr, k0, last, g4, xf);
    if constexpr (kAhead) load_chunk<T, JB>(p, max(i0, 0), k0, last, l16, g4, wf);
    uint64_t left[F] = {own[0], own[1]};
    for (int i = i0; i >= 0;) {  // each adapter of the tile
      if (kAhead && i != i0) load_chunk<T, JB>(p, i, k0, last, l16, g4, wf);
      f32x4 t[JB][F];
#pragma unroll
      for (int jb = 0; jb < JB; ++jb)
#pragma unroll
        for (int f = 0; f < F; ++f) t[jb][f] = f32x4{};
      if constexpr (kAhead) chunk_product<T, JB, F>(wf, xf, t);
      else chunk_at_once<T, JB, F>(p, i, k0, last, l16, g4, xf, t);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const bool mine = idx[f] == i;
        left[f] &= ~__ballot(mine);
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[jb][f][e] += mine ? t[jb][f][e] : 0.f;
      }
      i = left[0] ? next_adapter(idx[0], left[0]) : next_adapter(idx[1], left[1]);
    }
  }
  for (int h = W / 2; h; h >>= 1) {  // pairs of waves, in a fixed order
    if (h < W / 2) __syncthreads();
    if (wave >= h && wave < 2 * h)
#pragma unroll
      for (int x = 0; x < JB * F; ++x) red[((wave - h) * JB * F + x) * 64 + lane] = acc[x / F][x % F];
    __syncthreads();
    if (wave < h)
#pragma unroll
      for (int x = 0; x < JB * F; ++x) acc[x / F][x % F] += red[(wave * JB * F + x) * 64 + lane];
  }
  if (wave == 0)
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int n = n0 + 16 * f + l16;
      if (n < p.rows)
#pragma unroll
        for (int jb = 0; jb < JB; ++jb)
          *(DAN_TILE_GLOBAL f32x4 *)(p.part + ((int64_t)blockIdx.x * p.rows + n) * p.ranks + 16 * jb + 4 * g4) = acc[jb][f];
    }
}

// Few rows: 16 a work group, whose eight waves split the tile's adapters (each row is one wave's), so that the
// adapters' loads do not wait for each other. The wide side is split over many work groups.
constexpr int kFewWaves = 8;
template <typename T, int JB>
__global__ __launch_bounds__(64 * kFewWaves) void down_few_kernel(const DownParams p) {
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const int n = blockIdx.x * 16 + l16, first = blockIdx.y * p.chunks * kChunk, last = min(first + p.chunks * kChunk, p.n);
  int idx = n < p.rows ? adapter_of(p.index, n) : -1;
  if (idx >= p.adapters) idx = -1;  // (`up` makes the row NaN)
  const T *xr[1] = {static_cast<const T *>(p.x) + (int64_t)min(n, p.rows - 1) * p.x_stride};
  float *to = p.part + ((int64_t)blockIdx.y * p.rows + n) * p.ranks + 4 * g4;
  u32x4 xf[1][4];
  load_rows<T, 1>(xr, first, last, g4, xf);
  if (wave == 0 && n < p.rows && idx < 0)
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) *(DAN_TILE_GLOBAL f32x4 *)(to + 16 * jb) = f32x4{};
  uint64_t left = __ballot(idx >= 0);
  for (int turn = 0; left; ++turn) {
    const int i = next_adapter(idx, left);
    const bool mine = idx == i;
    left &= ~__ballot(mine);
    if (turn % kFewWaves != wave) continue;
    f32x4 t[JB][1];
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) t[jb][0] = f32x4{};
    u32x4 wf[JB][4];
    load_chunk<T, JB>(p, i, first, last, l16, g4, wf);
    chunk_product<T, JB, 1>(wf, xf, t);
    for (int k0 = first + kChunk; k0 < last; k0 += kChunk) {
      u32x4 more[1][4];
      load_rows<T, 1>(xr, k0, last, g4, more);
      load_chunk<T, JB>(p, i, k0, last, l16, g4, wf);
      chunk_product<T, JB, 1>(wf, more, t);
    }
    if (mine)
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) *(DAN_TILE_GLOBAL f32x4 *)(to + 16 * jb) = t[jb][0];
  }
}

// ---------------------------------------------------------------- up: out[n][m] = y[n][m] + c_i sum over j of v[n][j] w_i[m][j]
struct UpParams {
  const float *part;  // [splits][rows][ranks]
  float *sum;         // [rows][ranks]: v, for the gradient, or NULL
  const void *w, *y;  // w [adapters][cols][w_rank]; y may be NULL (zeros)
  void *out;
  const int32_t *index;
  const float *scale;
  int64_t y_stride, o_stride;
  int32_t rows, cols, rank, w_rank, adapters, ranks, splits, steps;  // w_rank: rank, or with zeros a multiple of 8; steps of 256 columns a work group (many rows)
  float scale_value;
};

// v of 16 F rows as the second product's operand: the parts added up in order, then hi and lo numbers in pieces of 8,
// hi pieces first, at [f][step][lane] (16 bytes each). With fp16 a row is multiplied by 2^exponent_of(top) first.
template <typename T, int ST, int F, int TH>
struct Operand {
  f32x4 v[16 * F][4 * ST];
  u32x4 piece[F * ST * 64];
  uint32_t top[16 * F];  // fp16: the bits of a row's largest |v|
  __device__ void make(const UpParams &p, int n0) {
    constexpr bool kHalf = std::is_same<T, _Float16>::value;
    if (kHalf)
      for (int r = threadIdx.x; r < 16 * F; r += TH) top[r] = 0u;
    if (kHalf) __syncthreads();
    // Four parts of all of a thread's quarters of 16 bytes are loaded at a time. Where there are more threads than quarters,
    // P of a wave's lanes share one and add up every P-th part.
    constexpr int Q = 16 * F * 4 * ST, P = TH >= Q ? TH / Q : 1, L = 64 / P, NQ = Q * P / TH;
    static_assert(NQ * TH == Q * P, "every thread has as many");
    const int64_t plane = (int64_t)p.rows * p.ranks;
    const int s0 = (threadIdx.x & 63) / L;
    auto quad = [&](int x) { return (int)(threadIdx.x + x * TH) / 64 * L + (int)threadIdx.x % L; };
    const float *from[NQ];
    f32x4 sum[NQ];
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      from[x] = p.part + (int64_t)min(n0 + quad(x) / (4 * ST), p.rows - 1) * p.ranks + quad(x) % (4 * ST) * 4;
      sum[x] = f32x4{};
    }
    for (int s = s0; s < p.splits; s += 4 * P) {
      f32x4 part[NQ][4];
#pragma unroll
      for (int x = 0; x < NQ; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) part[x][y] = *(const DAN_TILE_GLOBAL f32x4 *)(from[x] + min(s + y * P, p.splits - 1) * plane);
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < NQ; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[x][e] += s + y * P < p.splits ? part[x][y][e] : 0.f;
    }
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
#pragma unroll
      for (int m = L; m < 64; m <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[x][e] += __shfl_xor(sum[x][e], m);
      if (s0) continue;
      const int r = quad(x) / (4 * ST), j4 = quad(x) % (4 * ST), n = n0 + r;
      if (p.sum && blockIdx.x == 0 && n < p.rows) *(DAN_TILE_GLOBAL f32x4 *)(p.sum + (int64_t)n * p.ranks + 4 * j4) = sum[x];
      v[r][j4] = sum[x];
      if (kHalf) {
        const float m = fmaxf(fmaxf(finite_size(sum[x][0]), finite_size(sum[x][1])), fmaxf(finite_size(sum[x][2]), finite_size(sum[x][3])));
        atomicMax(&top[r], __builtin_bit_cast(uint32_t, m));  // (of values that are not negative: in any order)
      }
    }
    __syncthreads();
    const int r8 = (p.rank + 7) / 8;
    for (int q = threadIdx.x; q < F * ST * 64; q += TH) {
      const int r = q / (64 * ST) * 16 + (q & 15), u = (q / 64) % ST * 4 + (q >> 4) % 4, j8 = u >= r8 ? u - r8 : u;
      u32x4 to = {};
      if (u < 2 * r8) {
        f32x8 x = __builtin_shufflevector(v[r][2 * j8], v[r][2 * j8 + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        if (p.rank % 8)
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = 8 * j8 + e < p.rank ? x[e] : 0.f;
        if (kHalf) {
          const int e2 = exponent_of(__builtin_bit_cast(float, top[r]));
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = ldexpf(x[e], e2);
        }
        to = pack8<T>(x);
        if (u >= r8) to = low_part<T>(x, to);
      }
      piece[q] = to;
    }
    __syncthreads();
  }
};

// The operand of 64 columns from m0 on. Lane (l16, g4) of the result owns 8 columns from m0 + 8 g4 on and 8 from m0 + 32 +
// 8 g4 on, so that four lanes store 64 bytes of a row: row r of block b is column 32 (b / 2) + 8 (r / 4) + 4 (b % 2) + r % 4.
// Ranks in memory: kAny, one number at a time; kPieces, a multiple of 8, whose pieces lie 16-byte aligned; kFull, 32, 64 or 128, where
// the second half of the steps (v's low parts) takes the first half's operands again. Each by kernels of its own: in one with the others
// they would take registers, and waves, from them (rank 64, fp16, 1037 rows of 4096 columns: 10.5 us in full, 14.3 in pieces).
enum Form { kAny, kPieces, kFull };
template <int ST, Form FORM>
constexpr int kColumnSteps = FORM == kFull ? ST / 2 : ST;
template <typename T, int ST, Form FORM>
__device__ inline void load_columns(const UpParams &p, int i, int m0, int l16, int g4, u32x4 (&wf)[kColumnSteps<ST, FORM>][4]) {
  const T *w = static_cast<const T *>(p.w) + (int64_t)i * p.cols * p.w_rank;
  const int r8 = (p.rank + 7) / 8;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const int col = min(m0 + 32 * (b >> 1) + 8 * (l16 >> 2) + 4 * (b & 1) + (l16 & 3), p.cols - 1);
#pragma unroll
    for (int t = 0; t < kColumnSteps<ST, FORM>; ++t) {
      const int u = 4 * t + g4, j = u >= 2 * r8 ? 0 : 8 * (u >= r8 ? u - r8 : u);  // (past the last piece v holds zeros)
      const T *at = w + (int64_t)col * p.w_rank;
      if constexpr (FORM != kAny) {
        wf[t][b] = load16(at + j);
      } else {
        typedef T t8 __attribute__((ext_vector_type(8)));
        t8 x;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = ((const DAN_TILE_GLOBAL T *)at)[min(j + e, p.rank - 1)];
        wf[t][b] = __builtin_bit_cast(u32x4, x);  // (past the last rank v holds zeros: times a finite copy of it)
      }
    }
  }
}

// The factor of a row's product with adapter i.
template <typename T>
__device__ inline float factor_of(const UpParams &p, int i, uint32_t top) {
  const float c = p.scale ? p.scale[i] : p.scale_value;
  return std::is_same<T, _Float16>::value ? ldexpf(c, -exponent_of(__builtin_bit_cast(float, top))) : c;
}

// Many rows: 32 by `steps` times 256 columns, 64 a wave. y of the next step is loaded before this one's. (64 rows halve the
// loads of w, but leave two waves a SIMD instead of four: 8192 rows of 6144 columns took 53.7 us, and take 46.6.)
constexpr int kUpFrags = 2;
template <typename T, int ST, Form FORM>
__global__ __launch_bounds__(kThreads) void up_kernel(const UpParams p) {
  constexpr int F = kUpFrags;
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  __shared__ Operand<T, ST, F, kThreads> op;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const int n0 = blockIdx.y * 16 * F, first = blockIdx.x * p.steps * 4 * kUpCols + wave * kUpCols;
  int idx[F];
  u32x4 yv[F][2];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    const int n = n0 + 16 * f + l16;
    idx[f] = n < p.rows ? adapter_of(p.index, n) : -1;
  }
  auto load_y = [&](int m0) __attribute__((always_inline)) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const T *row = static_cast<const T *>(p.y) + min(n0 + 16 * f + l16, p.rows - 1) * p.y_stride;
#pragma unroll
      for (int h = 0; h < 2; ++h) yv[f][h] = load16(row + min(m0 + 32 * h + 8 * g4, p.cols - 8));
    }
  };
#pragma unroll
  for (int f = 0; f < F; ++f) yv[f][0] = yv[f][1] = u32x4{};
  if (p.y) load_y(first);
  int loaded = -1;  // the adapter that wf holds this step's columns of
  u32x4 wf[kColumnSteps<ST, FORM>][4];
  auto load_w = [&](int i, int m0) __attribute__((always_inline)) {
    load_columns<T, ST, FORM>(p, i, m0, l16, g4, wf);
    loaded = i;
  };
  {
    const uint64_t some = __ballot(idx[0] >= 0 && idx[0] < p.adapters);
    if (some && first < p.cols) load_w(next_adapter(idx[0], some), first);
  }
  op.make(p, n0);
  for (int step = 0; step < p.steps; ++step) {
    const int m0 = first + step * 4 * kUpCols;
    if (m0 >= p.cols) break;  // (at once where there are no columns: v alone is wanted)
    f32x4 acc[F][4];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x8 y = unpack8<T>(yv[f][h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[f][2 * h][e] = y[e];
          acc[f][2 * h + 1][e] = y[4 + e];
        }
      }
    if (p.y && step + 1 < p.steps) load_y(m0 + 4 * kUpCols);
    if (step) loaded = -1;
    uint64_t left[F];
#pragma unroll
    for (int f = 0; f < F; ++f) left[f] = __ballot(idx[f] >= 0);
    for (;;) {
      int i = -1;
#pragma unroll
      for (int f = F - 1; f >= 0; --f)
        if (left[f]) i = next_adapter(idx[f], left[f]);
      if (i < 0) break;
      if (i < p.adapters && i != loaded) load_w(i, m0);
#pragma unroll
      for (int f = 0; f < F; ++f) {
        const bool mine = idx[f] == i;
        const uint64_t votes = __ballot(mine);
        if (!votes) continue;
        left[f] &= ~votes;
        if (i >= p.adapters) {  // no such adapter
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[f][b][e] = mine ? NAN : acc[f][b][e];
          continue;
        }
        const float c = factor_of<T>(p, i, kHalf ? op.top[16 * f + l16] : 0u);
        u32x4 vf[ST];
#pragma unroll
        for (int t = 0; t < ST; ++t) vf[t] = op.piece[(f * ST + t) * 64 + lane];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          f32x4 t4 = {};
#pragma unroll
          for (int t = 0; t < ST; ++t) t4 = mfma16<T>(wf[t % kColumnSteps<ST, FORM>][b], vf[t], t4);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[f][b][e] = mine ? fmaf(c, t4[e], acc[f][b][e]) : acc[f][b][e];
        }
      }
    }
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const int n = n0 + 16 * f + l16;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int m = m0 + 32 * h + 8 * g4;
        if (n < p.rows && m < p.cols)
          store16(static_cast<T *>(p.out) + n * p.o_stride + m, pack8<T>(__builtin_shufflevector(acc[f][2 * h], acc[f][2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7)));
      }
    }
  }
}

// Few rows: 16 by 64 columns; the waves split the tile's adapters, and the first two store. (Ranks from 65 on that are no multiple of 8 take
// 1.3 KB of scratch memory a lane for the numbers that they read one at a time: 100 rows of 4 adapters, 4096 -> 4096, rank 100 in 100 us, rank
// 104 in 14.)
template <typename T, int ST, Form FORM>
__global__ __launch_bounds__(64 * kFewWaves) void up_few_kernel(const UpParams p) {
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  __shared__ Operand<T, ST, 1, 64 * kFewWaves> op;
  __shared__ f32x4 sums[4][64];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const int n = blockIdx.y * 16 + l16, m0 = blockIdx.x * kUpCols, m = m0 + 32 * wave + 8 * g4;
  const int idx = n < p.rows ? adapter_of(p.index, n) : -1;
  const bool store = wave < 2 && n < p.rows && m < p.cols;
  u32x4 yv = {};
  if (store && p.y) yv = load16(static_cast<const T *>(p.y) + n * p.y_stride + m);
  op.make(p, blockIdx.y * 16);
  if (p.cols == 0) return;  // v alone is wanted
  u32x4 vf[ST];
#pragma unroll
  for (int t = 0; t < ST; ++t) vf[t] = op.piece[t * 64 + lane];
  uint64_t left = __ballot(idx >= 0);
  for (int turn = 0; left; ++turn) {
    const int i = next_adapter(idx, left);
    const bool mine = idx == i;
    left &= ~__ballot(mine);
    if (turn % kFewWaves != wave) continue;
    float c = NAN;  // no such adapter
    u32x4 wf[kColumnSteps<ST, FORM>][4];
    if (i < p.adapters) {
      load_columns<T, ST, FORM>(p, i, m0, l16, g4, wf);
      c = factor_of<T>(p, i, kHalf ? op.top[l16] : 0u);
    } else {
#pragma unroll
      for (int t = 0; t < kColumnSteps<ST, FORM>; ++t)
#pragma unroll
        for (int b = 0; b < 4; ++b) wf[t][b] = u32x4{};
    }
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      f32x4 t4 = {};
#pragma unroll
      for (int t = 0; t < ST; ++t) t4 = mfma16<T>(wf[t % kColumnSteps<ST, FORM>][b], vf[t], t4);
      if (mine) sums[b][lane] = t4 * c;
    }
  }
  __syncthreads();
  if (!store) return;
  f32x8 out = unpack8<T>(yv);
  if (idx >= 0) out += __builtin_shufflevector(sums[2 * wave][lane], sums[2 * wave + 1][lane], 0, 1, 2, 3, 4, 5, 6, 7);
  store16(static_cast<T *>(p.out) + n * p.o_stride + m, pack8<T>(out));
}

// ---------------------------------------------------------------- outer: d_i[j][c] = c_i sum over the rows of i of v[n][j] z[n][c]
struct OuterSide {
  const float *v;  // [rows][ranks]
  const void *z;
  int64_t z_stride;
  float *sums;  // [parts][adapters][rank * cols], or
  void *out;    // with one part, the result itself
  int32_t cols, tiles;
};
struct OuterParams {
  OuterSide a, b;  // dA [rank][n_in] of (g, x); dB [n_out][rank] of (h, G)
  const int32_t *list, *starts;  // the rows in the order of their adapters, and where each adapter's begin [adapters + 1]; or NULL (one adapter, all rows)
  const float *scale;
  int32_t rows, rank, ranks, adapters, parts;
  float scale_value;
};

// Up to 4 numbers of a column of dB whose ranks are no multiple of 4: rounded to `out`, or as sums.
template <typename T>
__device__ inline void store_ranks(T *out, float *sums, f32x4 x, int count) {
  const u32x2 r = pack4<T>(x);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < count) {
      if (out) ((DAN_TILE_GLOBAL uint16_t *)out)[e] = (uint16_t)(r[e >> 1] >> 16 * (e & 1));
      else ((DAN_TILE_GLOBAL float *)sums)[e] = x[e];
    }
}

// (fp16's sums of a tile beside those of all rows fill the registers of one wave a SIMD from rank 33 on, bf16's own from 65; fp16's from 65 on
// keep 97 of them in scratch memory: 1037 rows of 5 adapters, 4096 -> 4096, the whole gradient at rank 64 56 us, bf16 44, at 128 114 and 83.)
// One adapter, 128 columns, a part of the adapter's rows; the waves take 32 of them in turn,
// each through a tile of its own in LDS, from where the transposing reads make the operand whose inner dimension is
// the rows. v's operand is loaded in place (a lane's 8 rows).
template <typename T, int JB>
__global__ __launch_bounds__(kThreads) void outer_kernel(const OuterParams p) {
  constexpr bool kHalf = std::is_same<T, _Float16>::value;
  using Tl = Tile<kOuterCols>;
  constexpr int CB = kOuterCols / 16;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lds = (uint32_t)(uintptr_t)(DAN_TILE_LDS uint8_t *)smem;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const bool side_b = (int)blockIdx.x >= p.a.tiles;
  const OuterSide &q = side_b ? p.b : p.a;
  const int c0 = ((int)blockIdx.x - (side_b ? p.a.tiles : 0)) * kOuterCols, i = blockIdx.y, part = blockIdx.z;

  const int start = p.starts ? p.starts[i] : 0, total = p.starts ? p.starts[i + 1] - start : i == 0 ? p.rows : 0;
  const int from = start + (int)((int64_t)total * part / p.parts), count = start + (int)((int64_t)total * (part + 1) / p.parts) - from;
  auto row_of = [&](int k) { return p.list ? p.list[from + k] : from + k; };
  f32x4 acc[JB][CB];
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) acc[jb][cb] = f32x4{};
  const uint32_t tile = lds + (uint32_t)(wave * Tl::bytes);
  const T *z = static_cast<const T *>(q.z) + c0;
  const int left = min(kOuterCols, q.cols - c0);  // columns of the tile (a multiple of 8)
  int next = wave * kOuterRows < count ? row_of(min(wave * kOuterRows + (lane & 31), count - 1)) : 0;
  for (int s0 = wave * kOuterRows; s0 < count; s0 += 4 * kOuterRows) {
    const int mine = next;  // lane l: the step's row l % 32
    next = row_of(min(s0 + 4 * kOuterRows + (lane & 31), count - 1));
    barrier_wave_lds();  // (the last step's reads of the tile)
#pragma unroll
    for (int x = 0; x < Tl::blocks; ++x) {
      const int n = __shfl(mine, Tl::block_row(x, lane));
      dma16_at(z + (int64_t)n * q.z_stride + min(Tl::block_byte(x, lane) / 2, (uint32_t)(left - 8)), tile + (uint32_t)(x * 1024));
    }
    const int rows = min(count - s0, kOuterRows);
    float v[JB][8];
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = 8 * g4 + e < rows;
      const float *at = q.v + (int64_t)__shfl(mine, 8 * g4 + e) * p.ranks + l16;
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) v[jb][e] = at[16 * jb];
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) v[jb][e] = in ? v[jb][e] : 0.f;
    }
    int e2 = 0;
    if (kHalf) {
#pragma unroll
      for (int jb = 0; jb < JB; ++jb)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, finite_size(v[jb][e]));
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
      lo[jb] = low_part<T>(x, hi[jb]);
    }
    const float back = kHalf ? ldexpf(1.f, -e2) : 1.f;
    wait_vmem<0>();
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
      if (rows < kOuterRows) {  // rows past the list: zeros, whatever its last row (whose copies they are) holds
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
  T *out = static_cast<T *>(q.out) + (int64_t)i * p.rank * q.cols;
#pragma unroll
  for (int jb = 0; jb < JB; ++jb)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int cb = 0; cb < CB / 2; ++cb) red[(wave * (CB / 2) + cb) * 64 + lane] = acc[jb][half * (CB / 2) + cb];
      __syncthreads();
      const f32x4 sum = ((red[wave * 64 + lane] + red[(CB / 2 + wave) * 64 + lane]) + (red[(CB + wave) * 64 + lane] + red[(3 * CB / 2 + wave) * 64 + lane])) * c;
      const int cb = half * (CB / 2) + wave, row = 4 * g4;
      // Lane: side b: column l16, ranks row..; side a: rank l16, columns row..
      const int col = c0 + 16 * cb + (side_b ? l16 : row), j = 16 * jb + (side_b ? row : l16);
      const int64_t at = side_b ? (int64_t)col * p.rank + j : (int64_t)j * q.cols + col;
      if (col < q.cols && j < p.rank) {
        if (side_b && p.rank % 4) store_ranks<T>(p.parts == 1 ? out + at : nullptr, to + at, sum, p.rank - j);
        else if (p.parts == 1) *(DAN_TILE_GLOBAL u32x2 *)(out + at) = pack4<T>(sum);
        else *(DAN_TILE_GLOBAL f32x4 *)(to + at) = sum;
      }
    }
}

// dB and g = G B_i for ranks up to 16 in bf16, from one pass over G: one adapter, 512 columns in four tiles, a part of the adapter's rows.
// A wave takes 32 rows at a time, and of them a tile after the other, the next one on its way into its second buffer; from
// LDS the tile is read twice, as `outer`'s operand and as rows. g is summed over the work group's columns alone: parts, a
// sixteenth of G's bytes, for gather_kernel.
constexpr int kBothTiles = 4;
struct BothParams {
  OuterParams o;   // its side b
  const void *bt;  // B^T [adapters][rank][n_out]
  float *g;        // [column tiles][rows][16]
};
__global__ __launch_bounds__(kThreads, 2) void both_kernel(const BothParams p) {
  using T = __bf16;
  using Tl = Tile<kOuterCols>;
  constexpr int CB = kOuterCols / 16, CT = kBothTiles;
  static_assert(CT % 2 == 0, "the buffers' turn");
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lds = (uint32_t)(uintptr_t)(DAN_TILE_LDS uint8_t *)smem;
  const OuterSide &q = p.o.b;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), l16 = lane & 15, g4 = lane >> 4;
  const int c0 = blockIdx.x * CT * kOuterCols, i = blockIdx.y, part = blockIdx.z, last = q.cols - 8;
  const int start = p.o.starts ? p.o.starts[i] : 0, total = p.o.starts ? p.o.starts[i + 1] - start : i == 0 ? p.o.rows : 0;
  const int from = start + (int)((int64_t)total * part / p.o.parts), count = start + (int)((int64_t)total * (part + 1) / p.o.parts) - from;
  auto row_of = [&](int k) { return p.o.list ? p.o.list[from + k] : from + k; };
  // The columns' B^T as operands, behind the waves' buffers: [tile][step of 32 columns][lane].
  u32x4 *bf = reinterpret_cast<u32x4 *>(smem + 8 * Tl::bytes);
  {
    static_assert(CT == 4, "a tile a wave");
    const T *row = static_cast<const T *>(p.bt) + ((int64_t)i * p.o.rank + min(l16, p.o.rank - 1)) * q.cols;
    u32x4 b[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) b[s] = load16(row + min(c0 + wave * kOuterCols + 32 * s + 8 * g4, last));
#pragma unroll
    for (int s = 0; s < 4; ++s) bf[(4 * wave + s) * 64 + lane] = c0 + wave * kOuterCols + 32 * s + 8 * g4 > last ? u32x4{} : b[s];
    __syncthreads();
  }
  f32x4 acc[CT][CB];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) acc[ct][cb] = f32x4{};
  const uint32_t tile = lds + (uint32_t)(wave * 2 * Tl::bytes);
  auto issue = [&](int ct, int mine) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < Tl::blocks; ++x) {
      const int64_t n = __shfl(mine, Tl::block_row(x, lane));
      const int c = min(c0 + ct * kOuterCols + (int)(Tl::block_byte(x, lane) / 2), last);
      dma16_at(static_cast<const T *>(q.z) + n * q.z_stride + c, tile + (uint32_t)((ct & 1) * Tl::bytes + x * 1024));
    }
  };
  float vn[8];  // the next step's v
  auto load_v = [&](int mine) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) vn[e] = q.v[(int64_t)__shfl(mine, 8 * g4 + e) * p.o.ranks + l16];
  };
  int mine = 0, next = 0;  // lane l: the step's row l % 32, and the next step's
  auto rows_at = [&](int s0) { return row_of(min(s0 + (lane & 31), count - 1)); };
  if (wave * kOuterRows < count) {
    mine = rows_at(wave * kOuterRows);
    next = rows_at((wave + 4) * kOuterRows);
    issue(0, mine);
    load_v(mine);
  }
  for (int s0 = wave * kOuterRows; s0 < count; s0 += 4 * kOuterRows) {
    const int rows = min(count - s0, kOuterRows), after = next;
    f32x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 8 * g4 + e < rows ? vn[e] : 0.f;
    const u32x4 hi = pack8<T>(x), lo = low_part<T>(x, hi);
    f32x4 g[2] = {};
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      wait_vmem<0>();
      barrier_wave_lds();  // (the reads of the buffer that is filled next)
      // (places in memory and in LDS are worked out again for each tile: kept, they would not leave registers for the sums)
      int l = lane;
      asm volatile("" : "+v"(mine), "+v"(l));
      const int m16 = l & 15, h4 = l >> 4;
      if (ct + 1 < CT) {
        issue(ct + 1, mine);
      } else {
        issue(0, after);
        load_v(after);
        next = rows_at(s0 + 8 * kOuterRows);
      }
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t at_tile = tile + (uint32_t)((ct & 1) * Tl::bytes);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const u32x4 b = bf[(4 * ct + s) * 64 + lane];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const int r = 16 * f + m16;
          g[f] = mfma16<T>(b, lds_read16(at_tile + (uint32_t)(r * Tl::row + (((4 * s + h4) ^ Tl::swizzle(r)) << 4))), g[f]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        u32x4 zf;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 8 * h4 + 4 * h + (m16 >> 2);
          const uint32_t at = at_tile + (uint32_t)(r * Tl::row + (((2 * cb + ((m16 >> 1) & 1)) ^ Tl::swizzle(r)) << 4) + 8 * (m16 & 1));
          const u32x2 t = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((DAN_TILE_LDS i16x4 *)(uintptr_t)at));
          zf[2 * h] = t[0];
          zf[2 * h + 1] = t[1];
        }
        if (rows < kOuterRows) {  // rows past the list: zeros, whatever its last row (whose copies they are) holds
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (8 * g4 + e >= rows) zf[e >> 1] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
        }
        acc[ct][cb] = mfma16<T>(lo, zf, mfma16<T>(hi, zf, acc[ct][cb]));
        __builtin_amdgcn_sched_barrier(0);  // (reads of one block at a time: the registers hold no more)
      }
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int64_t n = __shfl(mine, 16 * f + l16);
      if (16 * f + l16 < rows) *(DAN_TILE_GLOBAL f32x4 *)(p.g + ((int64_t)blockIdx.x * p.o.rows + n) * 16 + 4 * g4) = g[f];
    }
    mine = after;
  }
  wait_vmem<0>();  // (the last step's loads of a next one)
  // The waves' sums, added in order.
  f32x4 *red = reinterpret_cast<f32x4 *>(smem);
  const float c = p.o.scale ? p.o.scale[i] : p.o.scale_value;
  float *to = q.sums + ((int64_t)part * p.o.adapters + i) * p.o.rank * q.cols;
  T *out = static_cast<T *>(q.out) + (int64_t)i * p.o.rank * q.cols;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    __syncthreads();
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) red[(wave * CB + cb) * 64 + lane] = acc[ct][cb];
    __syncthreads();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int cb = half * 4 + wave, col = c0 + ct * kOuterCols + 16 * cb + l16;
      const f32x4 sum = ((red[cb * 64 + lane] + red[(CB + cb) * 64 + lane]) + (red[(2 * CB + cb) * 64 + lane] + red[(3 * CB + cb) * 64 + lane])) * c;
      if (col < q.cols && 4 * g4 < p.o.rank) {
        const int64_t at = (int64_t)col * p.o.rank + 4 * g4;
        if (p.o.rank % 4) store_ranks<T>(p.o.parts == 1 ? out + at : nullptr, to + at, sum, p.o.rank - 4 * g4);
        else if (p.o.parts == 1) *(DAN_TILE_GLOBAL u32x2 *)(out + at) = pack4<T>(sum);
        else *(DAN_TILE_GLOBAL f32x4 *)(to + at) = sum;
      }
    }
  }
}

// g's parts added up in order: four lanes share 16 bytes of the result. (Rows of no adapter have no parts, and nothing reads
// what they get.)
__global__ __launch_bounds__(kThreads) void gather_kernel(const float *parts, float *g, int rows, int tiles) {
  const int lane = threadIdx.x & 63, share = lane >> 4;
  const int64_t quad = ((int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * 16 + (lane & 15), quads = 4 * (int64_t)rows;
  const float *from = parts + 4 * min(quad, quads - 1);
  f32x4 x = {};
#pragma unroll 8
  for (int t = share; t < tiles; t += 4) x += *(const DAN_TILE_GLOBAL f32x4 *)(from + t * 4 * quads);
#pragma unroll
  for (int m = 16; m < 64; m <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], m);
  if (share == 0 && quad < quads) *(DAN_TILE_GLOBAL f32x4 *)(g + 4 * quad) = x;
}

// The parts of dA and dB added up in order, rounded once: 8 values a thread.
struct SumParams {
  const float *a, *b;
  void *da, *db;
  int64_t na, nb;  // values of dA, dB (multiples of 8)
  int32_t parts_a, parts_b;
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
  for (int i = 0, parts = b ? p.parts_b : p.parts_a; i < parts; ++i, from += n) {
    x += *(const DAN_TILE_GLOBAL f32x4 *)from;
    y += *(const DAN_TILE_GLOBAL f32x4 *)(from + 4);
  }
  store16(static_cast<T *>(b ? p.db : p.da) + at, pack8<T>(__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7)));
}

// ---------------------------------------------------------------- transposes of A [R][rank][n_in] and B [R][n_out][rank], 16-bit
struct TurnParams {
  const uint16_t *a, *b;
  uint16_t *at, *bt;  // [R][n_in][rank, with zeros a multiple of 8], [R][rank][n_out]
  const int32_t *index;      // NULL: no list
  int32_t *list, *starts;    // [rows], [adapters + 1]
  int32_t rows, rank, n_in, n_out, adapters, a_tiles, b_tiles;  // tiles of 64 columns an adapter
};
// The rows of adapter i, in order, at their place among all adapters' (rows of no adapter, or of one past the last, are left
// out): each wave counts its share, then writes it.
__device__ inline void list_rows(const TurnParams &p, int i) {
  constexpr int W = kThreads / 64, U = 8;
  __shared__ int before[W], here[W];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), share = (p.rows + W * 64 - 1) / (W * 64) * 64;
  const int r0 = min(wave * share, p.rows), r1 = min(r0 + share, p.rows);
  auto each = [&](auto &&f) {
    for (int r = r0; r < r1; r += U * 64) {
      int x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = p.index[min(r + u * 64 + lane, p.rows - 1)];
#pragma unroll
      for (int u = 0; u < U; ++u) f(r + u * 64 + lane, r + u * 64 + lane < r1 ? x[u] : -1);
    }
  };
  int below = 0, mine = 0;
  each([&](int, int x) {
    below += __popcll(__ballot(x >= 0 && x < i));
    mine += __popcll(__ballot(x == i));
  });
  if (lane == 0) {
    before[wave] = below;
    here[wave] = mine;
  }
  __syncthreads();
  int start = 0, to = 0, total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    start += before[w];
    to += w < wave ? here[w] : 0;
    total += here[w];
  }
  to += start;
  if (threadIdx.x == 0) {
    p.starts[i] = start;
    if (i == p.adapters - 1) p.starts[i + 1] = start + total;
  }
  each([&](int n, int x) {
    const uint64_t votes = __ballot(x == i);
    if (x == i) p.list[to + __popcll(votes & ((uint64_t(1) << lane) - 1))] = n;
    to += __popcll(votes);
  });
}

// 64 positions of the wide side and all ranks a work group, 16 bytes a load and a store.
__global__ __launch_bounds__(kThreads) void turn_kernel(const TurnParams p) {
  __shared__ __attribute__((aligned(16))) uint16_t tile[DAN_ADAPT_MAX_RANK][64 + 8];
  int x = blockIdx.x;
  if (p.index) {  // (first: they take longest)
    if (x < p.adapters) return list_rows(p, x);
    x -= p.adapters;
  }
  const bool b = x >= p.a_tiles * p.adapters;
  if (b) x -= p.a_tiles * p.adapters;
  const int tiles = b ? p.b_tiles : p.a_tiles, i = x / tiles, c0 = x % tiles * 64, wide = b ? p.n_out : p.n_in, r8 = (p.rank + 7) / 8;
  const int64_t base = (int64_t)i * p.rank * wide;
  const uint16_t *from = (b ? p.b : p.a) + base;
  uint16_t *to = b ? p.bt + base : p.at + (int64_t)i * 8 * r8 * wide;
  const int c8 = min(64, wide - c0) / 8;  // pieces of 8 columns
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
  for (int e = threadIdx.x; e < (b && p.rank % 8 ? 64 * p.rank : b ? 64 * r8 : 8 * p.rank); e += kThreads) {
    if (b && p.rank % 8) {  // a column's ranks are contiguous, in pieces of no certain alignment
      const int c = e / p.rank, j = e % p.rank;
      tile[j][c] = from[(int64_t)(c0 + min(c, 8 * c8 - 1)) * p.rank + j];
    } else if (b) {  // a column's ranks are contiguous
      const int c = e / r8, j = 8 * (e % r8);
      const u16x8 v = __builtin_bit_cast(u16x8, load16(from + (int64_t)(c0 + min(c, 8 * c8 - 1)) * p.rank + j));
#pragma unroll
      for (int y = 0; y < 8; ++y) tile[j + y][c] = v[y];
    } else {  // a rank's columns are
      const int j = e / 8, c = 8 * (e % 8);
      *reinterpret_cast<u32x4 *>(&tile[j][c]) = load16(from + (int64_t)j * wide + c0 + min(c, 8 * c8 - 8));
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < (b ? 8 * p.rank : 64 * r8); e += kThreads) {
    if (b) {
      const int j = e / 8, c = e % 8;
      if (c < c8) store16(to + (int64_t)j * wide + c0 + 8 * c, *reinterpret_cast<const u32x4 *>(&tile[j][8 * c]));
    } else {
      const int c = e / r8, j = 8 * (e % r8);
      u16x8 v;
#pragma unroll
      for (int y = 0; y < 8; ++y) v[y] = j + y < p.rank ? tile[j + y][c] : (uint16_t)0;
      if (c < 8 * c8) store16(to + (int64_t)(c0 + c) * 8 * r8 + j, __builtin_bit_cast(u32x4, v));
    }
  }
}

// ---------------------------------------------------------------- host
// Ranks as the kernels are built for: 16, 32, 64 or 128.
int ranks_of(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// The kernels for few rows or those for many. The former take 5 us and more with every row and rank, the latter 13 us and 4 more with each
// adapter of a tile of 32 rows. 4096 -> 4096, us, few / many: one adapter of rank 16, 256 rows 9.6 / 12.7, 512 rows 15.4 / 13.0; of rank 128,
// 128 rows 19.8 / 22.6, 256 rows 34.6 / 23.1; 24 adapters of rank 16 in any order, 512 rows 24.9 / 53.9, 1024 rows 45.6 / 56.5; 8 of rank 64, 384 rows
// 47.6 / 53.2, 640 rows 83.4 / 66.5. (The order of the rows is on the device alone; 5 adapters of rank 64 one behind the other, 384 rows: 26.4 / 21.4.)
bool few(int rows, int rank, int adapters) { return rows <= (128 + 4096 / ranks_of(rank)) * (adapters > 4 ? 2 : 1); }

// Parts of `down`'s sum over n: as many work groups as fill the chip, of at least a chunk a wave (many rows) or two.
int splits_of(int rows, int n, int rank, int adapters) {
  const int chunks = (n + kChunk - 1) / kChunk;
  if (few(rows, rank, adapters)) return std::max(1, std::min({chunks, std::max(2, 1024 / ((rows + 15) / 16)), 32}));
  const int tiles = (rows + 31) / 32, waves = ranks_of(rank) <= 32 ? 16 : 8;
  return std::max(1, std::min((256 + tiles - 1) / tiles, chunks / waves));
}
// Parts of an adapter's rows in `outer`: enough work groups for the chip, but parts are written and read again in fp32.
int parts_of(int rows, int n_in, int n_out, int adapters) {
  const int64_t groups = (int64_t)((n_in + kOuterCols - 1) / kOuterCols + (n_out + kOuterCols - 1) / kOuterCols) * adapters;
  const int64_t by_rows = rows / (512 * (int64_t)adapters);
  return (int)std::max<int64_t>(1, std::min<int64_t>((1024 + groups - 1) / groups, by_rows));
}
// g and dB from one pass (both_kernel; fp16's powers of 2 of each step would leave it no registers): where G does not fit the caches from one pass to the next.
bool both(int rows, int n_out, int rank) { return ranks_of(rank) == 16 && (int64_t)rows * n_out * 2 >= kBothBytes; }
int both_tiles(int n_out) { return (n_out + kBothTiles * kOuterCols - 1) / (kBothTiles * kOuterCols); }
int both_parts(int rows, int n_out, int adapters) {  // (two work groups fit a compute unit)
  return (int)std::max<int64_t>(1, std::min<int64_t>(512 / ((int64_t)both_tiles(n_out) * adapters), rows / (512 * (int64_t)adapters)));
}
int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

template <typename T, int JB>
hipError_t launch_down(const DownParams &p, int splits, hipStream_t s) {
  if (few(p.rows, p.rank, p.adapters)) {
    hipLaunchKernelGGL((down_few_kernel<T, JB>), dim3((p.rows + 15) / 16, splits), dim3(64 * kFewWaves), 0, s, p);
    return hipGetLastError();
  }
  constexpr int W = kDownWaves<JB>, bytes = W / 2 * JB * 2 * 1024;
  const hipError_t err = allow_lds<&down_kernel<T, JB>>(bytes);
  if (err != hipSuccess) return err;
  hipLaunchKernelGGL((down_kernel<T, JB>), dim3(splits, (p.rows + 31) / 32), dim3(64 * W), bytes, s, p);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_down(DownParams p, int splits, hipStream_t s) {
  const int chunks = (p.n + kChunk - 1) / kChunk;
  p.chunks = (chunks + splits - 1) / splits;
  return p.ranks == 16 ? launch_down<T, 1>(p, splits, s) : p.ranks == 32 ? launch_down<T, 2>(p, splits, s)
       : p.ranks == 64 ? launch_down<T, 4>(p, splits, s) : launch_down<T, 8>(p, splits, s);
}

// The grid of `up`, and the steps of a work group (many rows).
struct UpGrid {
  int x, y, threads, steps;
  UpGrid(int rows, int cols, int rank, int adapters) : steps(1) {
    if (few(rows, rank, adapters)) {
      x = std::max(1, (cols + kUpCols - 1) / kUpCols);
      y = (rows + 15) / 16;
      threads = 64 * kFewWaves;
      return;
    }
    const int groups = std::max(1, (cols + 4 * kUpCols - 1) / (4 * kUpCols));
    y = (rows + 16 * kUpFrags - 1) / (16 * kUpFrags);
    steps = std::max(1, std::min(4, (int)((int64_t)y * groups / 768)));
    x = (groups + steps - 1) / steps;
    threads = kThreads;
  }
};
template <typename T, int ST, Form FORM>
hipError_t launch_up(UpParams p, hipStream_t s) {
  const UpGrid g(p.rows, p.cols, p.rank, p.adapters);
  p.steps = g.steps;
  if (few(p.rows, p.rank, p.adapters)) hipLaunchKernelGGL((up_few_kernel<T, ST, FORM>), dim3(g.x, g.y), dim3(g.threads), 0, s, p);
  else hipLaunchKernelGGL((up_kernel<T, ST, FORM>), dim3(g.x, g.y), dim3(g.threads), 0, s, p);
  return hipGetLastError();
}
template <typename T, int ST>
hipError_t launch_up(const UpParams &p, hipStream_t s) {
  if constexpr (ST > 1)
    if (p.w_rank == p.ranks) return launch_up<T, ST, kFull>(p, s);
  return p.w_rank % 8 == 0 ? launch_up<T, ST, kPieces>(p, s) : launch_up<T, ST, kAny>(p, s);
}
template <typename T>
hipError_t launch_up(const UpParams &p, hipStream_t s) {
  return p.ranks == 16 ? launch_up<T, 1>(p, s) : p.ranks == 32 ? launch_up<T, 2>(p, s) : p.ranks == 64 ? launch_up<T, 4>(p, s) : launch_up<T, 8>(p, s);
}

template <typename T, int JB>
hipError_t launch_outer(const OuterParams &p, hipStream_t s) {
  constexpr int bytes = 4 * Tile<kOuterCols>::bytes;
  hipLaunchKernelGGL((outer_kernel<T, JB>), dim3(p.a.tiles + p.b.tiles, p.adapters, p.parts), dim3(kThreads), bytes, s, p);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_outer(const OuterParams &p, hipStream_t s) {
  return p.ranks == 16 ? launch_outer<T, 1>(p, s) : p.ranks == 32 ? launch_outer<T, 2>(p, s) : p.ranks == 64 ? launch_outer<T, 4>(p, s) : launch_outer<T, 8>(p, s);
}

template <typename T>
hipError_t forward(const DanAdaptArgs &a, hipStream_t s) {
  DownParams d;
  d.x = a.x; d.x_stride = a.x_stride; d.w = a.a; d.index = a.index; d.part = static_cast<float *>(a.workspace);
  d.rows = a.rows; d.n = a.n_in; d.rank = a.rank; d.adapters = a.adapters; d.ranks = ranks_of(a.rank);
  const int splits = splits_of(a.rows, a.n_in, a.rank, a.adapters);
  hipError_t err = launch_down<T>(d, splits, s);
  if (err != hipSuccess) return err;
  UpParams u;
  u.part = d.part; u.sum = a.down; u.w = a.b; u.y = a.y; u.y_stride = a.y_stride; u.out = a.out; u.o_stride = a.out_stride;
  u.index = a.index; u.scale = a.scale; u.scale_value = a.scale_value;
  u.rows = a.rows; u.cols = a.n_out; u.rank = u.w_rank = a.rank; u.adapters = a.adapters; u.ranks = d.ranks; u.splits = splits; u.steps = 1;
  return launch_up<T>(u, s);
}

// The workspace of the gradient: A^T, B^T, the list of rows, g in parts and added up, and the parts of dA and dB.
struct GradSpace {
  int64_t at, bt, list, starts, part, g, da, db, total;
  int splits, parts, parts_a, parts_b;  // (parts_a, parts_b: where g and dB come from one pass, which fp16's size holds, too: it is asked for without a type)
  GradSpace(int rows, int n_in, int n_out, int rank, int adapters) {
    splits = splits_of(rows, n_out, rank, adapters);
    parts = parts_of(rows, n_in, n_out, adapters);
    const bool one = both(rows, n_out, rank);
    parts_a = one ? parts_of(rows, n_in, 0, adapters) : parts;
    parts_b = one ? both_parts(rows, n_out, adapters) : parts;
    at = 0;
    bt = align256(at + (int64_t)adapters * ((rank + 7) / 8 * 8) * n_in * 2);
    list = align256(bt + (int64_t)adapters * rank * n_out * 2);
    starts = list + (int64_t)rows * 4;
    part = align256(starts + ((int64_t)adapters + 1) * 4);
    g = align256(part + (int64_t)std::max(splits, one ? both_tiles(n_out) : 0) * rows * ranks_of(rank) * 4);
    da = align256(g + (int64_t)rows * ranks_of(rank) * 4);
    auto kept = [&](int other) { return (int64_t)std::max({parts > 1 ? parts : 0, other > 1 ? other : 0}); };
    db = align256(da + kept(parts_a) * adapters * rank * n_in * 4);
    total = align256(db + kept(parts_b) * adapters * rank * n_out * 4);
  }
};

template <typename T>
hipError_t backward(const DanAdaptGradArgs &a, const GradSpace &w, hipStream_t s) {
  uint8_t *ws = static_cast<uint8_t *>(a.workspace);
  OuterParams o;
  o.a = {reinterpret_cast<float *>(ws + w.g), a.x, a.x_stride, reinterpret_cast<float *>(ws + w.da), a.da, a.n_in, a.da ? (a.n_in + kOuterCols - 1) / kOuterCols : 0};
  o.b = {a.down, a.g, a.g_stride, reinterpret_cast<float *>(ws + w.db), a.db, a.n_out, a.db ? (a.n_out + kOuterCols - 1) / kOuterCols : 0};
  o.list = a.index ? reinterpret_cast<int32_t *>(ws + w.list) : nullptr; o.starts = a.index ? reinterpret_cast<int32_t *>(ws + w.starts) : nullptr;
  o.scale = a.scale; o.scale_value = a.scale_value; o.rows = a.rows; o.rank = a.rank; o.ranks = ranks_of(a.rank);
  o.adapters = a.adapters; o.parts = w.parts;
  hipError_t err;
  {
    TurnParams t;
    t.a = static_cast<const uint16_t *>(a.a); t.b = static_cast<const uint16_t *>(a.b);
    t.at = reinterpret_cast<uint16_t *>(ws + w.at); t.bt = reinterpret_cast<uint16_t *>(ws + w.bt);
    t.rank = a.rank; t.n_in = a.n_in; t.n_out = a.n_out; t.adapters = a.adapters;
    t.rows = a.rows; t.list = reinterpret_cast<int32_t *>(ws + w.list); t.starts = reinterpret_cast<int32_t *>(ws + w.starts);
    t.index = a.da || a.db ? a.index : nullptr;
    t.a_tiles = a.dx ? (a.n_in + 63) / 64 : 0;
    t.b_tiles = a.dx || a.da ? (a.n_out + 63) / 64 : 0;
    if (const int groups = (t.a_tiles + t.b_tiles + (t.index ? 1 : 0)) * a.adapters)
      hipLaunchKernelGGL(turn_kernel, dim3(groups), dim3(kThreads), 0, s, t);
    if ((err = hipGetLastError()) != hipSuccess) return err;
  }
  const bool one = a.db && (a.dx || a.da) && std::is_same<T, __bf16>::value && both(a.rows, a.n_out, a.rank);
  float *g = reinterpret_cast<float *>(ws + w.g);
  if (one) {
    BothParams b;
    b.o = o; b.o.parts = w.parts_b; b.bt = ws + w.bt; b.g = reinterpret_cast<float *>(ws + w.part);
    const int tiles = both_tiles(a.n_out);
    constexpr int bytes = 8 * Tile<kOuterCols>::bytes + kBothTiles * 4096;
    if ((err = allow_lds<&both_kernel>(bytes)) != hipSuccess) return err;
    hipLaunchKernelGGL(both_kernel, dim3(tiles, a.adapters, w.parts_b), dim3(kThreads), bytes, s, b);
    if ((err = hipGetLastError()) != hipSuccess) return err;
    hipLaunchKernelGGL(gather_kernel, dim3((a.rows + 15) / 16), dim3(kThreads), 0, s, b.g, g, a.rows, tiles);
    if ((err = hipGetLastError()) != hipSuccess) return err;
  } else if (a.dx || a.da) {
    DownParams d;
    d.x = a.g; d.x_stride = a.g_stride; d.w = ws + w.bt; d.index = a.index; d.part = reinterpret_cast<float *>(ws + w.part);
    d.rows = a.rows; d.n = a.n_out; d.rank = a.rank; d.adapters = a.adapters; d.ranks = o.ranks;
    if ((err = launch_down<T>(d, w.splits, s)) != hipSuccess) return err;
  }
  if (a.dx || (a.da && !one)) {
    UpParams u;  // (without dx: no columns, the sum of the parts alone)
    u.part = one ? g : reinterpret_cast<float *>(ws + w.part); u.sum = one ? nullptr : g; u.w = ws + w.at; u.y = nullptr; u.y_stride = 0; u.out = a.dx; u.o_stride = a.dx_stride;
    u.index = a.index; u.scale = a.scale; u.scale_value = a.scale_value;
    u.rows = a.rows; u.cols = a.dx ? a.n_in : 0; u.rank = a.rank; u.w_rank = (a.rank + 7) / 8 * 8; u.adapters = a.adapters; u.ranks = o.ranks; u.splits = one ? 1 : w.splits; u.steps = 1;
    if ((err = launch_up<T>(u, s)) != hipSuccess) return err;
  }
  if (!a.da && !a.db) return hipSuccess;
  if (one) {
    o.b.tiles = 0;
    o.parts = w.parts_a;
  }
  if (o.a.tiles + o.b.tiles && (err = launch_outer<T>(o, s)) != hipSuccess) return err;
  SumParams m;
  m.a = o.a.sums; m.b = o.b.sums; m.da = a.da; m.db = a.db;
  m.parts_a = one ? w.parts_a : w.parts;
  m.parts_b = one ? w.parts_b : w.parts;
  m.na = a.da && m.parts_a > 1 ? (int64_t)a.adapters * a.rank * a.n_in : 0;
  m.nb = a.db && m.parts_b > 1 ? (int64_t)a.adapters * a.rank * a.n_out : 0;
  if (!m.na && !m.nb) return hipSuccess;
  hipLaunchKernelGGL(sum_kernel<T>, dim3((uint32_t)(((m.na + m.nb) / 8 + kThreads - 1) / kThreads)), dim3(kThreads), 0, s, m);
  return hipGetLastError();
}

// A launch holds fewer than 2^32 threads.
bool too_many(int64_t groups, int threads = kThreads) { return groups * threads >= int64_t(1) << 32; }
int64_t over(int64_t x, int64_t by) { return (x + by - 1) / by; }

int check_sizes(int dtype, int rows, int n_in, int n_out, int rank, int adapters, float scale_value) {
  if (dtype != DAN_DTYPE_BF16 && dtype != DAN_DTYPE_F16) return fail(DAN_ERR_UNSUPPORTED, "dtype %d: bf16 or fp16", dtype);
  if (rows < 0 || rows > 1 << 20) return fail(DAN_ERR_UNSUPPORTED, "rows %d: at most 2^20", rows);
  if (n_in <= 0 || n_out <= 0 || n_in % 8 || n_out % 8 || n_in > 1 << 20 || n_out > 1 << 20)
    return fail(DAN_ERR_UNSUPPORTED, "n_in %d and n_out %d: multiples of 8 up to 2^20", n_in, n_out);
  if (rank <= 0 || rank > DAN_ADAPT_MAX_RANK) return fail(DAN_ERR_UNSUPPORTED, "rank %d: 1 to %d", rank, DAN_ADAPT_MAX_RANK);
  if (adapters <= 0 || adapters > 65535) return fail(DAN_ERR_UNSUPPORTED, "%d adapters: 1 to 65535", adapters);
  if (!(isfinite(scale_value))) return fail(DAN_ERR_INVALID_ARGUMENT, "scale_value must be finite");
  // (`up` has the most threads by far: one for 2 values, or with many rows for 32 to 128. `down` has 2^26 at most.)
  const UpGrid up(rows, std::max(n_in, n_out), rank, adapters);
  if (too_many((int64_t)up.x * up.y, up.threads))
    return fail(DAN_ERR_UNSUPPORTED, "%d rows of %d columns: more than one launch holds (2^39 values)", rows, std::max(n_in, n_out));
  return DAN_OK;
}
// And of the gradient, whose other launches grow with the adapters.
int check_grad_sizes(int rows, int n_in, int n_out, int rank, int adapters) {
  const int64_t groups = (over(n_in, kOuterCols) + over(n_out, kOuterCols)) * adapters;
  if (too_many(groups * std::max(parts_of(rows, n_in, n_out, adapters), parts_of(rows, n_in, 0, adapters))) ||
      too_many((over(n_in, 64) + over(n_out, 64) + 1) * adapters) || too_many(over((int64_t)adapters * rank * ((int64_t)n_in + n_out), 8 * kThreads)))
    return fail(DAN_ERR_UNSUPPORTED, "%d adapters of rank %d, %d to %d: more than one launch holds (columns 2^30, numbers 2^35)", adapters, rank, n_in, n_out);
  return DAN_OK;
}
bool bad_rows(const void *p, int64_t stride) { return ((uintptr_t)p & 15) || stride % 8 || stride < 0; }

}  // namespace
}  // namespace dan

extern "C" {

int dan_adapt_abi_version(void) { return DAN_ADAPT_ABI_VERSION; }

int64_t dan_adapt_workspace_size(int32_t rows, int32_t n_in, int32_t rank, int32_t adapters) {
  if (rows <= 0 || n_in <= 0 || rank <= 0 || rank > DAN_ADAPT_MAX_RANK || adapters <= 0) return 0;
  return (int64_t)dan::splits_of(rows, n_in, rank, adapters) * rows * dan::ranks_of(rank) * 4;
}

int64_t dan_adapt_grad_workspace_size(int32_t rows, int32_t n_in, int32_t n_out, int32_t rank, int32_t adapters) {
  using namespace dan;
  if (rows <= 0 || check_sizes(DAN_DTYPE_BF16, rows, n_in, n_out, rank, adapters, 0.f) != DAN_OK ||
      check_grad_sizes(rows, n_in, n_out, rank, adapters) != DAN_OK)
    return 0;
  return GradSpace(rows, n_in, n_out, rank, adapters).total;
}

int dan_adapt(const DanAdaptArgs *a, void *stream) {
  using namespace dan;
  g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->abi_version != DAN_ADAPT_ABI_VERSION)
    return fail(DAN_ERR_VERSION, "abi_version %d, library speaks %d", a->abi_version, DAN_ADAPT_ABI_VERSION);
  if (const int rc = check_sizes(a->dtype, a->rows, a->n_in, a->n_out, a->rank, a->adapters, a->scale_value)) return rc;
  if (a->rows == 0) return DAN_OK;
  if (!a->x || !a->y || !a->a || !a->b || !a->out) return fail(DAN_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (bad_rows(a->x, a->x_stride) || bad_rows(a->y, a->y_stride) || bad_rows(a->out, a->out_stride) || (a->rows > 1 && a->out_stride < a->n_out) ||
      (((uintptr_t)a->a | (uintptr_t)a->b | (uintptr_t)a->down) & 15))
    return fail(DAN_ERR_INVALID_ARGUMENT, "rows must start 16-byte aligned, and written ones must not overlap");
  const int64_t need = dan_adapt_workspace_size(a->rows, a->n_in, a->rank, a->adapters);
  if (!a->workspace || a->workspace_bytes < need || ((uintptr_t)a->workspace & 15))
    return fail(DAN_ERR_INVALID_ARGUMENT, "workspace needs %lld bytes, 16-byte aligned", (long long)need);
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
  if (const int rc = check_grad_sizes(a->rows, a->n_in, a->n_out, a->rank, a->adapters)) return rc;
  if (a->rows == 0) return DAN_OK;
  if (!a->x || !a->g || !a->a || !a->b || !a->down) return fail(DAN_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (bad_rows(a->x, a->x_stride) || bad_rows(a->g, a->g_stride) || bad_rows(a->dx, a->dx ? a->dx_stride : 0) ||
      (a->dx && a->rows > 1 && a->dx_stride < a->n_in) ||
      (((uintptr_t)a->a | (uintptr_t)a->b | (uintptr_t)a->da | (uintptr_t)a->db | (uintptr_t)a->down) & 15))
    return fail(DAN_ERR_INVALID_ARGUMENT, "rows must start 16-byte aligned, and written ones must not overlap");
  const GradSpace w(a->rows, a->n_in, a->n_out, a->rank, a->adapters);
  if (!a->workspace || a->workspace_bytes < w.total || ((uintptr_t)a->workspace & 255))
    return fail(DAN_ERR_INVALID_ARGUMENT, "workspace needs %lld bytes, 256-byte aligned", (long long)w.total);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = a->dtype == DAN_DTYPE_BF16 ? backward<__bf16>(*a, w, s) : backward<_Float16>(*a, w, s);
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "adapter gradient launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

}  // extern "C"
