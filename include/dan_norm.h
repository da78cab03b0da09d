/* dan_norm: the residual's addition and the root-mean-square norm in front of
 * a projection, and its gradient (C ABI).
 *
 * dan's decoder layers add and normalise in eager steps (dan/fused.py:35-48
 * behind a torch addition) and quantise what comes out in another
 * (dan/fused.py:85-91). Here one launch reads both addends once:
 *
 *   s = x + residual                 (fp32; stored rounded, as `stream`)
 *   y = s / sqrt(mean(s^2) + eps) * weight          (DAN_NORM_RMS)
 *                              or * (1 + weight)    (DAN_NORM_ZERO_CENTERED)
 *   stored rounded to the inputs' type (`out`), and / or as e4m3 codes with a
 *   scale for each row as dan_fp8_quantize makes them (`codes`, `scale`).
 *
 * Conventions as in dan_tree_attn.h: device memory of the caller, rows of unit
 * stride that start 16 bytes aligned, 0 on success, dan_tree_attn_last_error().
 */
#ifndef DAN_NORM_H
#define DAN_NORM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define DAN_NORM_ABI_VERSION 1
#define DAN_NORM_MAX_COLS 16384

enum { DAN_NORM_RMS = 0, DAN_NORM_ZERO_CENTERED = 1 };

typedef struct {
  int32_t abi_version; /* DAN_NORM_ABI_VERSION */
  int32_t dtype;       /* DAN_DTYPE_BF16 or DAN_DTYPE_F16: x, residual, weight, stream, out */
  int32_t rows, cols;  /* rows: below 2^24 (at most 2^24 - 256 with tiled codes of more than 1024 columns); cols: a multiple of 8 (16 with codes), at most DAN_NORM_MAX_COLS */
  int32_t norm;        /* DAN_NORM_* */
  int32_t layout;      /* of codes: DAN_FP8_LAYOUT_ROWS or DAN_FP8_LAYOUT_TILED (dan_fp8.h) */
  float eps;           /* finite, >= 0 */
  int32_t reserved;
  const void *x;        int64_t x_stride;
  const void *residual; int64_t residual_stride; /* NULL: none */
  const void *weight;                            /* [cols] */
  void *stream;         int64_t stream_stride;   /* NULL: not wanted; may be x or residual itself */
  void *out;            int64_t out_stride;      /* NULL: not wanted */
  void *codes;                                   /* NULL: not wanted; rows * cols bytes, or dan_fp8_tiled_bytes() */
  float *scale;                                  /* [rows], with codes */
  float *rstd;                                   /* [rows]: 1 / sqrt(mean + eps), for the gradient; NULL: not wanted */
} DanNormArgs;

typedef struct {
  int32_t abi_version;
  int32_t dtype;
  int32_t rows, cols;
  int32_t norm;
  int32_t reserved;
  const void *s;        int64_t s_stride;        /* stream (x itself without a residual) */
  const void *weight;
  const float *rstd;
  const void *g;        int64_t g_stride;        /* the gradient of out */
  const void *g_stream; int64_t g_stream_stride; /* the gradient of stream; NULL: none */
  void *ds;             int64_t ds_stride;       /* the gradient of x and of residual */
  void *dw;                                      /* [cols], the gradient of weight; NULL: not wanted */
  void *workspace; int64_t workspace_bytes;      /* with dw: dan_norm_grad_workspace_size() bytes, 16-byte aligned */
} DanNormGradArgs;

int dan_norm_abi_version(void);
int dan_add_norm(const DanNormArgs *args, void *stream);
int dan_add_norm_grad(const DanNormGradArgs *args, void *stream);
/* 0: invalid arguments. */
int64_t dan_norm_grad_workspace_size(int32_t rows, int32_t cols);

#ifdef __cplusplus
}
#endif

#endif
