// The residual's addition and root-mean-square norm in front of a projection, and their gradient
// (include/dan_norm.h), for gfx950.
//
//   s = x + r       rs = 1 / sqrt(mean(s^2) + eps)       y = s rs w'      (w' = weight or 1 + weight)
//   c = max(max |y|, 1e-12) / 448, codes e4m3(y / c)
// and with G and Gs the gradients of y and s:
//   dx = dr = rs (w' G - s rs mean(w' G s rs)) + Gs       dw = sum over rows of G s rs
//
// All of it is bound by memory: every tensor passes once. A row stays in registers as fp32 between its sum of
// squares, its largest value and its stores; y is rounded once, from fp32, also where it becomes codes. The
// gradient reads s as it was stored (rounded to 16 bits): the two addends would be one tensor more to read,
// and what the rounding moves is of the size of the result's own.
//
// Measured, warm: 8192 x 4096 in bf16 to stream and codes 38 us (235 MB, 6.1 TB/s), to tiled codes 43, 7 x 4096 3.9 us (a launch, its
// loads, two reductions; tiled 4.0); 4096 x 14336 to stream and out 149 us (470 MB, 3.2 TB/s: above 8192 columns a row's values fill the
// registers of one wave a SIMD, as they do in the gradient); 4099 x 2048 in fp16 to stream and out 13.0 us (67 MB, 5.2 TB/s), its gradient 14.8 (67 MB, 4.5) and dw's sum 6.8.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "dan_fp8.h"
#include "dan_norm.h"
#include "dan_tree_attn.h"
#include "fp8_layout.h"
#include "tiles.h"

namespace dan {
int fail(int status, const char *fmt, ...);  // tree_attn.hip: sets the thread's last-error message
extern thread_local char g_err[512];

namespace {

using namespace tiles;

constexpr int kThreads = 256;

struct NormParams {
  const void *x, *r, *w;
  void *stream, *out;
  uint8_t *codes;
  float *scale, *rstd;
  int64_t x_stride, r_stride, s_stride, o_stride;
  int32_t rows, cols, kt, tiled;
  float eps, shift;  // shift: 1 for zero-centered weights
};

struct GradParams {
  const void *s, *w, *g, *gs;
  const float *rstd;
  void *ds;
  float *partial;  // [groups][cols] of dw, or NULL
  int64_t s_stride, g_stride, gs_stride, d_stride;
  int32_t rows, cols;
  float shift;
};

// Sum, or maximum of bits, over the L threads of a row.
template <int L>
__device__ inline float row_sum(float v, float *red) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}
template <int L>
__device__ inline uint32_t row_max(uint32_t v, uint32_t *red) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
  if constexpr (L > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = max(max(red[0], red[1]), max(red[2], red[3]));
  }
  return v;
}

__device__ inline u32x2 codes8(f32x8 y, float scale) {
  u32x2 q;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h] / scale, y[4 * h + 1] / scale, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * h + 2] / scale, y[4 * h + 3] / scale, w, true);
    q[h] = (uint32_t)w;
  }
  return q;
}

// A row is L threads of NC pieces of 8 values. With codes in the tiled layout the padding rows of the last panel,
// and each row's last k-step, are zeros.
template <typename T, int L, int NC>
__global__ __launch_bounds__(kThreads) void add_norm_kernel(const NormParams p) {
  __shared__ float sums[4];
  __shared__ uint32_t maxs[4];
  const int t = threadIdx.x % L, row = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  if (row >= p.rows) {  // (a whole wave, or work group)
    if (p.codes && p.tiled && row < (p.rows + 255) / 256 * 256)
      for (int c = 8 * t; c < 64 * p.kt; c += 8 * L) *(DAN_TILE_GLOBAL u32x2 *)(p.codes + dan_fp8::tiled_offset(row, c, p.kt)) = u32x2{0u, 0u};
    return;
  }
  const T *x = static_cast<const T *>(p.x) + row * p.x_stride, *r = static_cast<const T *>(p.r) + row * p.r_stride;
  f32x8 s[NC];
  u32x4 w[NC];
  {
    u32x4 a[NC], b[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {  // (past the row: its last piece, not used)
      const int c = min(8 * t + 8 * L * j, p.cols - 8);
      a[j] = load16(x + c);
      if (p.r) b[j] = load16(r + c);
      w[j] = load16(static_cast<const T *>(p.w) + c);
    }
#pragma unroll
    for (int j = 0; j < NC; ++j) s[j] = p.r ? unpack8<T>(a[j]) + unpack8<T>(b[j]) : unpack8<T>(a[j]);
  }
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = 8 * t + 8 * L * j;
    if (c >= p.cols) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) sq = fmaf(s[j][i], s[j][i], sq);
    if (p.stream) store16(static_cast<T *>(p.stream) + row * p.s_stride + c, pack8<T>(s[j]));
  }
  const float rs = 1.f / sqrtf(row_sum<L>(sq, sums) / (float)p.cols + p.eps);
  if (p.rstd && t == 0) p.rstd[row] = rs;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = 8 * t + 8 * L * j;
    const f32x8 wj = unpack8<T>(w[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) s[j][i] = s[j][i] * rs * (wj[i] + p.shift);
    if (c >= p.cols) continue;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, dan_fp8::abs_bits(s[j][i]));
    if (p.out) store16(static_cast<T *>(p.out) + row * p.o_stride + c, pack8<T>(s[j]));
  }
  if (!p.codes) return;
  const float scale = dan_fp8::scale_of(row_max<L>(top, maxs));
  if (t == 0) p.scale[row] = scale;
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    const int c = 8 * t + 8 * L * j;
    if (c < p.cols) *(DAN_TILE_GLOBAL u32x2 *)(p.codes + (p.tiled ? dan_fp8::tiled_offset(row, c, p.kt) : (int64_t)row * p.cols + c)) = codes8(s[j], scale);
  }
  if (p.tiled)
    for (int c = p.cols + 8 * t; c < 64 * p.kt; c += 8 * L) *(DAN_TILE_GLOBAL u32x2 *)(p.codes + dan_fp8::tiled_offset(row, c, p.kt)) = u32x2{0u, 0u};
}

// Rows blockIdx.x, + gridDim.x, ...: each group keeps its rows' sum of dw in registers, so that dw takes one pass over s and
// G with ds, in an order that the number of rows alone fixes.
template <typename T, int NC>
__global__ __launch_bounds__(kThreads) void norm_grad_kernel(const GradParams p) {
  __shared__ float sums[2][4];
  const int t = threadIdx.x;
  f32x8 w[NC], dw[NC];
#pragma unroll
  for (int j = 0; j < NC; ++j) {
    w[j] = unpack8<T>(load16(static_cast<const T *>(p.w) + min(8 * t + 8 * kThreads * j, p.cols - 8))) + p.shift;
    dw[j] = f32x8{};
  }
  int turn = 0;
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const T *s = static_cast<const T *>(p.s) + row * p.s_stride, *g = static_cast<const T *>(p.g) + row * p.g_stride;
    const T *gs = static_cast<const T *>(p.gs) + row * p.gs_stride;
    u32x4 sv[NC], gv[NC], av[NC];
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = min(8 * t + 8 * kThreads * j, p.cols - 8);
      sv[j] = load16(s + c);
      gv[j] = load16(g + c);
      if (p.gs) av[j] = load16(gs + c);
    }
    const float rs = p.rstd[row];
    f32x8 hat[NC], wg[NC];
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      hat[j] = unpack8<T>(sv[j]) * rs;
      wg[j] = unpack8<T>(gv[j]);
      const bool in = 8 * t + 8 * kThreads * j < p.cols;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[j][i] = fmaf(wg[j][i], hat[j][i], dw[j][i]);
        wg[j][i] *= w[j][i];
        dot = fmaf(in ? wg[j][i] : 0.f, hat[j][i], dot);
      }
    }
    // (two buffers by turns: a row's sums are read before the next row's barrier)
    const float mean = row_sum<kThreads>(dot, sums[turn]) / (float)p.cols;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = 8 * t + 8 * kThreads * j;
      f32x8 d = (wg[j] - hat[j] * mean) * rs;
      if (p.gs) d += unpack8<T>(av[j]);
      if (c < p.cols) store16(static_cast<T *>(p.ds) + row * p.d_stride + c, pack8<T>(d));
    }
  }
  if (p.partial) {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = 8 * t + 8 * kThreads * j;
      if (c >= p.cols) continue;
      float *to = p.partial + (int64_t)blockIdx.x * p.cols + c;
      *(DAN_TILE_GLOBAL f32x4 *)to = f32x4{dw[j][0], dw[j][1], dw[j][2], dw[j][3]};
      *(DAN_TILE_GLOBAL f32x4 *)(to + 4) = f32x4{dw[j][4], dw[j][5], dw[j][6], dw[j][7]};
    }
  }
}

// dw: 32 columns a work group, 8 threads of 4 columns by 32 shares of the groups' sums.
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_weight_kernel(const float *partial, T *dw, int groups, int cols) {
  __shared__ f32x4 red[kThreads];
  const int c = blockIdx.x * 32 + 4 * (threadIdx.x & 7), share = threadIdx.x >> 3;
  f32x4 sum = {};
  if (c < cols)
    for (int i = share; i < groups; i += 32) sum += *(const DAN_TILE_GLOBAL f32x4 *)(partial + (int64_t)i * cols + c);
  red[threadIdx.x] = sum;
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    __syncthreads();
    if (share < m) red[threadIdx.x] += red[threadIdx.x + 8 * m];
  }
  if (share == 0 && c < cols) *(DAN_TILE_GLOBAL u32x2 *)(dw + c) = pack4<T>(red[threadIdx.x]);
}

int grad_groups(int rows) { return std::min(rows, 512); }

template <typename T, int L, int NC>
hipError_t launch_norm(const NormParams &p, hipStream_t s) {
  const int64_t rows = p.codes && p.tiled ? ((int64_t)p.rows + 255) / 256 * 256 : p.rows;
  hipLaunchKernelGGL((add_norm_kernel<T, L, NC>), dim3((uint32_t)((rows + kThreads / L - 1) / (kThreads / L))), dim3(kThreads), 0, s, p);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_norm(const NormParams &p, hipStream_t s) {
  const int pieces = (p.cols + 8 * kThreads - 1) / (8 * kThreads);
  // (a wave a row needs no barrier: 8192 rows with codes, 512 columns 7.6 us against a work group's 14.1, 1024 columns 11.8 against 17.3;
  // 7 rows of 1024 columns 3.4 against 3.3)
  if (p.cols <= 512) return launch_norm<T, 64, 1>(p, s);
  if (p.cols <= 1024) return launch_norm<T, 64, 2>(p, s);
  if (pieces <= 1) return launch_norm<T, kThreads, 1>(p, s);
  if (pieces <= 2) return launch_norm<T, kThreads, 2>(p, s);
  if (pieces <= 4) return launch_norm<T, kThreads, 4>(p, s);
  return launch_norm<T, kThreads, 8>(p, s);
}

template <typename T>
hipError_t launch_grad(const GradParams &p, void *dw, hipStream_t s) {
  const int pieces = (p.cols + 8 * kThreads - 1) / (8 * kThreads), groups = p.partial ? grad_groups(p.rows) : p.rows;
  const dim3 grid(groups), block(kThreads);
  if (pieces <= 1) hipLaunchKernelGGL((norm_grad_kernel<T, 1>), grid, block, 0, s, p);
  else if (pieces <= 2) hipLaunchKernelGGL((norm_grad_kernel<T, 2>), grid, block, 0, s, p);
  else if (pieces <= 4) hipLaunchKernelGGL((norm_grad_kernel<T, 4>), grid, block, 0, s, p);
  else hipLaunchKernelGGL((norm_grad_kernel<T, 8>), grid, block, 0, s, p);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || !p.partial) return err;
  hipLaunchKernelGGL(norm_weight_kernel<T>, dim3((p.cols + 31) / 32), block, 0, s, p.partial, static_cast<T *>(dw), groups, p.cols);
  return hipGetLastError();
}

// What the two calls' shapes have to be.
int check_shape(int dtype, int rows, int cols, int norm) {
  if (dtype != DAN_DTYPE_BF16 && dtype != DAN_DTYPE_F16) return fail(DAN_ERR_UNSUPPORTED, "dtype %d: bf16 or fp16", dtype);
  if (rows < 0 || rows >= 1 << 24) return fail(DAN_ERR_INVALID_ARGUMENT, "rows %d: fewer than 2^24", rows);
  if (cols <= 0 || cols % 8 || cols > DAN_NORM_MAX_COLS) return fail(DAN_ERR_UNSUPPORTED, "cols %d: a multiple of 8 up to %d", cols, DAN_NORM_MAX_COLS);
  if (norm != DAN_NORM_RMS && norm != DAN_NORM_ZERO_CENTERED) return fail(DAN_ERR_INVALID_ARGUMENT, "norm %d: 0 (rms) or 1 (zero-centered)", norm);
  return DAN_OK;
}
// A row operand: aligned, and for writing rows of its own.
bool bad_rows(const void *p, int64_t stride, int rows, int cols, bool write) {
  return ((uintptr_t)p & 15) || stride % 8 || stride < 0 || (write && rows > 1 && stride < cols);
}

}  // namespace
}  // namespace dan

extern "C" {

int dan_norm_abi_version(void) { return DAN_NORM_ABI_VERSION; }

int64_t dan_norm_grad_workspace_size(int32_t rows, int32_t cols) {
  if (rows <= 0 || cols <= 0 || cols % 8 || cols > DAN_NORM_MAX_COLS) return 0;
  return (int64_t)dan::grad_groups(rows) * cols * 4;
}

int dan_add_norm(const DanNormArgs *a, void *stream) {
  using namespace dan;
  g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->abi_version != DAN_NORM_ABI_VERSION)
    return fail(DAN_ERR_VERSION, "abi_version %d, library speaks %d", a->abi_version, DAN_NORM_ABI_VERSION);
  if (const int rc = check_shape(a->dtype, a->rows, a->cols, a->norm)) return rc;
  if (!(a->eps >= 0.f && isfinite(a->eps))) return fail(DAN_ERR_INVALID_ARGUMENT, "eps must be finite and >= 0");
  if (a->layout != DAN_FP8_LAYOUT_ROWS && a->layout != DAN_FP8_LAYOUT_TILED)
    return fail(DAN_ERR_INVALID_ARGUMENT, "layout %d: 0 (rows) or 1 (tiled)", a->layout);
  if (a->rows == 0) return DAN_OK;
  if (!a->x || !a->weight || (!a->out && !a->codes) || (a->codes && !a->scale)) return fail(DAN_ERR_INVALID_ARGUMENT, "NULL pointer");
  // (a work group each row, also those of the last panel; up to 1024 columns four rows share one)
  if (a->codes && a->layout == DAN_FP8_LAYOUT_TILED && a->cols > 1024 && a->rows > (1 << 24) - 256)
    return fail(DAN_ERR_INVALID_ARGUMENT, "rows %d: at most 2^24 - 256 with %d columns in the tiled layout", a->rows, a->cols);
  if (a->codes && a->cols % 16) return fail(DAN_ERR_UNSUPPORTED, "cols %d: a multiple of 16 for codes", a->cols);
  if (bad_rows(a->x, a->x_stride, a->rows, a->cols, false) || (a->residual && bad_rows(a->residual, a->residual_stride, a->rows, a->cols, false)) ||
      (a->stream && bad_rows(a->stream, a->stream_stride, a->rows, a->cols, true)) ||
      (a->out && bad_rows(a->out, a->out_stride, a->rows, a->cols, true)) || ((uintptr_t)a->weight & 15) || ((uintptr_t)a->codes & 15) ||
      ((uintptr_t)a->scale & 3) || ((uintptr_t)a->rstd & 3))
    return fail(DAN_ERR_INVALID_ARGUMENT, "rows must start 16-byte aligned, and written ones must not overlap");
  NormParams p;
  p.x = a->x; p.x_stride = a->x_stride;
  p.r = a->residual; p.r_stride = a->residual_stride;
  p.w = a->weight;
  p.stream = a->stream; p.s_stride = a->stream_stride;
  p.out = a->out; p.o_stride = a->out_stride;
  p.codes = static_cast<uint8_t *>(a->codes); p.scale = a->scale; p.rstd = a->rstd;
  p.rows = a->rows; p.cols = a->cols;
  p.kt = (a->cols + 63) / 64; p.tiled = a->layout == DAN_FP8_LAYOUT_TILED;
  p.eps = a->eps; p.shift = a->norm == DAN_NORM_ZERO_CENTERED ? 1.f : 0.f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = a->dtype == DAN_DTYPE_BF16 ? launch_norm<__bf16>(p, s) : launch_norm<_Float16>(p, s);
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "norm launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

int dan_add_norm_grad(const DanNormGradArgs *a, void *stream) {
  using namespace dan;
  g_err[0] = 0;
  if (!a) return fail(DAN_ERR_INVALID_ARGUMENT, "args is NULL");
  if (a->abi_version != DAN_NORM_ABI_VERSION)
    return fail(DAN_ERR_VERSION, "abi_version %d, library speaks %d", a->abi_version, DAN_NORM_ABI_VERSION);
  if (const int rc = check_shape(a->dtype, a->rows, a->cols, a->norm)) return rc;
  if (a->rows == 0) return DAN_OK;
  if (!a->s || !a->weight || !a->rstd || !a->g || !a->ds) return fail(DAN_ERR_INVALID_ARGUMENT, "NULL pointer");
  if (bad_rows(a->s, a->s_stride, a->rows, a->cols, false) || bad_rows(a->g, a->g_stride, a->rows, a->cols, false) ||
      (a->g_stream && bad_rows(a->g_stream, a->g_stream_stride, a->rows, a->cols, false)) ||
      bad_rows(a->ds, a->ds_stride, a->rows, a->cols, true) || ((uintptr_t)a->weight & 15) || ((uintptr_t)a->dw & 15))
    return fail(DAN_ERR_INVALID_ARGUMENT, "rows must start 16-byte aligned, and written ones must not overlap");
  const int64_t need = a->dw ? dan_norm_grad_workspace_size(a->rows, a->cols) : 0;
  if (a->dw && (!a->workspace || a->workspace_bytes < need || ((uintptr_t)a->workspace & 15)))
    return fail(DAN_ERR_INVALID_ARGUMENT, "workspace needs %lld bytes, 16-byte aligned", (long long)need);
  GradParams p;
  p.s = a->s; p.s_stride = a->s_stride;
  p.w = a->weight; p.rstd = a->rstd;
  p.g = a->g; p.g_stride = a->g_stride;
  p.gs = a->g_stream; p.gs_stride = a->g_stream_stride;
  p.ds = a->ds; p.d_stride = a->ds_stride;
  p.partial = a->dw ? static_cast<float *>(a->workspace) : nullptr;
  p.rows = a->rows; p.cols = a->cols;
  p.shift = a->norm == DAN_NORM_ZERO_CENTERED ? 1.f : 0.f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t err = a->dtype == DAN_DTYPE_BF16 ? launch_grad<__bf16>(p, a->dw, s) : launch_grad<_Float16>(p, a->dw, s);
  if (err != hipSuccess) return fail(DAN_ERR_LAUNCH, "norm gradient launch failed: %s", hipGetErrorString(err));
  return DAN_OK;
}

}  // extern "C"
