/* dan_tree_grad: the gradient of tree attention (C ABI).
 *
 * dan trains through its reads (dan/tuning.py:82-133 calls attend with grad
 * enabled); dan_tree_attn_fwd (dan_tree_attn.h) has no gradient. Two entry
 * points add it:
 *
 *   dan_tree_attn_fwd_lse   dan_tree_attn_fwd that also writes each row's
 *                           logarithm of the sum of exponentials;
 *   dan_tree_attn_bwd       from it, q, k, v, the output and the output's
 *                           gradient: the gradients of q, k and v. The
 *                           probabilities are computed again, tile by tile.
 *
 * The conventions are dan_tree_attn.h's: device memory of the caller, strides
 * in elements, unit-stride head_dim, rows 16 bytes aligned, 0 on success and
 * dan_tree_attn_last_error() otherwise.
 */
#ifndef DAN_TREE_GRAD_H
#define DAN_TREE_GRAD_H

#include <stdint.h>

#include "dan_tree_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DAN_TREE_GRAD_ABI_VERSION 1

/* Keys [key0, key0 + keys) of one segment (rows are segment-local: row r is
 * packed row start + r). Rows [key0, q_end) are the ones that see any of them. */
typedef struct {
  int32_t start, n, trunk;
  int32_t key0, keys;
  int32_t q_end;
  int32_t reserved[2];
} DanGradKeyUnit;

/* Query rows [t0, t0 + tq) of one segment. They see the past_len keys of prefix
 * entry past_idx (-1: none), the trunk up to themselves and, if t0 + tq > trunk,
 * the branch rows from `branch0` (the first row of the branch that holds row
 * max(t0, trunk)). */
typedef struct {
  int32_t start, n, trunk;
  int32_t t0, tq;
  int32_t past_len, past_idx;
  int32_t branch0;
} DanGradQueryUnit;

typedef struct {
  int32_t abi_version; /* DAN_TREE_GRAD_ABI_VERSION */
  int32_t dtype;       /* DAN_DTYPE_BF16 or DAN_DTYPE_F16: q, k, v, out, their gradients and the prefix entries */
  int32_t num_heads, num_kv_heads, head_dim, num_tokens;
  float scale;         /* the softmax scale of the forward call */
  int32_t key_rows;    /* keys of a whole key unit: dan_tree_grad_key_rows(head_dim, 0 or 1) */
  const void *q;    int64_t q_stride_tok, q_stride_head;
  const void *k;    int64_t k_stride_tok, k_stride_head;
  const void *v;    int64_t v_stride_tok, v_stride_head;
  const void *out;  int64_t o_stride_tok, o_stride_head;
  const void *grad; int64_t g_stride_tok, g_stride_head; /* the gradient of out */
  const float *lse; /* [num_heads][num_tokens], from dan_tree_attn_fwd_lse */
  void *dq;         int64_t dq_stride_tok, dq_stride_head;
  void *dk;         int64_t dk_stride_tok, dk_stride_head;
  void *dv;         int64_t dv_stride_tok, dv_stride_head;
  /* Longest first: work groups start in this order. Rows outside every unit are left as they are. */
  const DanGradKeyUnit *key_units;     int32_t num_key_units;
  const DanGradQueryUnit *query_units; int32_t num_query_units;
  /* [num_tokens] each, segment-local: a row's first key of its own branch (0 for
   * a trunk row), and one past the last row that sees it as a key. */
  const int32_t *row_lo, *row_end;
  const DanPastDesc *pasts; int32_t num_pasts;
  void *workspace; int64_t workspace_bytes; /* dan_tree_grad_workspace_size() bytes, 256-byte aligned */
  /* Parts of the heads of a kv head that work groups of their own take for dK and dV, added up afterwards: 1 to num_heads / num_kv_heads. */
  int32_t key_splits, reserved;
} DanTreeGradArgs;

int dan_tree_grad_abi_version(void);
/* Keys of a key unit (`small` 0: the larger tile, 1: the smaller one, for batches of few units); 0: unsupported head_dim. */
int32_t dan_tree_grad_key_rows(int32_t head_dim, int32_t small);
/* Query rows of a query unit; 0: unsupported head layout. */
int32_t dan_tree_grad_query_rows(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim);
/* Bytes of workspace (0: invalid arguments). */
int64_t dan_tree_grad_workspace_size(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t num_tokens, int32_t key_splits);
/* dan_tree_attn_fwd of bf16 or fp16 inputs, and lse [num_heads][num_tokens]
 * (fp32): log2 of the sum over a row's visible keys of 2^(score * scale * log2 e). */
int dan_tree_attn_fwd_lse(const DanTreeAttnArgs *args, float *lse, void *stream);
int dan_tree_attn_bwd(const DanTreeGradArgs *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif
