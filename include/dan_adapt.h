/* dan_adapt: low-rank adapters of many requests beside a shared projection,
 * and their gradients (C ABI).
 *
 * dan trains one adapter and merges it into the weights (dan/lora.py,
 * dan/tuning.py:82-133). Here the projection stays shared and every row of the
 * batch adds its own adapter's product:
 *
 *   out[n] = y[n] + scale_i (x[n] A_i^T) B_i^T,      i = index[n]
 *
 * x [N, n_in] is the projection's input, y [N, n_out] its output, A_i [rank,
 * n_in], B_i [n_out, rank]. A negative index: no adapter (out = y). An index
 * past the last adapter gives NaN. An infinite x A^T (or G B) gives the formula's
 * infinities; an infinity that is itself a factor of it (in B, and for the gradients
 * in A, x or G) gives an infinity or NaN.
 *
 * Conventions as in dan_tree_attn.h: device memory of the caller, rows of unit
 * stride that start 16 bytes aligned, 0 on success, dan_tree_attn_last_error().
 */
#ifndef DAN_ADAPT_H
#define DAN_ADAPT_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DAN_ADAPT_ABI_VERSION 1
#define DAN_ADAPT_MAX_RANK 128

/* Sizes: rows to 2^20, n_in and n_out multiples of 8 to 2^20, ranks to 128, 65535 adapters; together, as far as one launch
 * goes: rows * max(n_in, n_out) below 2^39, and for the gradient adapters * (n_in + n_out) below 2^30 and that times rank
 * below 2^35. */

typedef struct {
  int32_t abi_version; /* DAN_ADAPT_ABI_VERSION */
  int32_t dtype;       /* DAN_DTYPE_BF16 or DAN_DTYPE_F16: x, y, a, b, out */
  int32_t rows, n_in, n_out, rank, adapters;
  int32_t reserved;
  const void *x; int64_t x_stride;
  const void *y; int64_t y_stride;
  const void *a;          /* [adapters][rank][n_in] */
  const void *b;          /* [adapters][n_out][rank] */
  const int32_t *index;   /* [rows]; NULL: adapter 0 for every row */
  const float *scale;     /* [adapters]; NULL: scale_value for every adapter */
  float scale_value;
  void *out; int64_t out_stride; /* may be y itself */
  float *down; /* [rows][rank rounded up to 16, 32, 64 or 128]: x A^T, for the gradient; NULL: not wanted */
  void *workspace; int64_t workspace_bytes; /* dan_adapt_workspace_size() bytes, 16-byte aligned */
} DanAdaptArgs;

typedef struct {
  int32_t abi_version;
  int32_t dtype;
  int32_t rows, n_in, n_out, rank, adapters;
  int32_t reserved;
  const void *x; int64_t x_stride;
  const void *g; int64_t g_stride; /* the gradient of out (which is that of y, too) */
  const void *a, *b;
  const int32_t *index;
  const float *scale;
  float scale_value;
  const float *down;   /* what the forward call wrote */
  void *dx; int64_t dx_stride; /* the adapters' part of the gradient of x; NULL: not wanted */
  void *da, *db;       /* as a and b; NULL: not wanted */
  void *workspace; int64_t workspace_bytes; /* dan_adapt_grad_workspace_size() bytes, 256-byte aligned */
} DanAdaptGradArgs;

int dan_adapt_abi_version(void);
/* 0: invalid arguments. */
int64_t dan_adapt_workspace_size(int32_t rows, int32_t n_in, int32_t rank, int32_t adapters);
int64_t dan_adapt_grad_workspace_size(int32_t rows, int32_t n_in, int32_t n_out, int32_t rank, int32_t adapters);
int dan_adapt(const DanAdaptArgs *args, void *stream);
int dan_adapt_grad(const DanAdaptGradArgs *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif
