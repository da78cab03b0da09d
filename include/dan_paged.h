/*
 * dan_paged.h -- C ABI of the gfx950 paged key-value cache: appending the
 * keys and values of new tokens, and attention of one new token per sequence.
 *
 * A cache is two tensors of pages, k and v, each [pages, Hkv, page_size, D]
 * (any page, head and token strides). A sequence's key at place t lies in page
 * table[seq][t / page_size], row t % page_size. dan reads prompts without
 * generating (dan/runner.py:66-82) and keeps whole prefixes
 * (dan/cache.py:11-39); this cache grows token by token instead, for
 * sequences that go on behind a read.
 *
 * Conventions: as dan_tree_attn.h (device pointers owned by the caller,
 * strides in elements, unit-stride head_dim, rows 16-byte aligned, status
 * codes with a thread-local message from dan_tree_attn_last_error(),
 * asynchronous on `stream`, nothing allocated or kept). What lies on the
 * device only (lengths, places, page numbers) is checked by the kernels: no
 * value of it makes them read or write outside the tensors described here.
 */
#ifndef DAN_PAGED_H
#define DAN_PAGED_H

#include <stdint.h>

#include "dan_qkv_front.h"
#include "dan_tree_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DAN_PAGED_ABI_VERSION 1

/* page_size is a multiple of this many keys. */
#define DAN_PAGED_KEY_BLOCK 16

typedef struct {
  int32_t abi_version;  /* DAN_PAGED_ABI_VERSION */
  int32_t dtype;        /* DanDtype of q, k, v, the norm weights and q_out: bf16 or f16 */
  int32_t cache_dtype;  /* the same, or e4m3 */
  int32_t table_dtype;  /* DanDtype of cos and sin: `dtype`, or f32 */
  int32_t num_tokens;   /* N */
  int32_t num_heads;    /* H; 0: no q (q and q_out are not read) */
  int32_t num_kv_heads; /* Hkv */
  int32_t head_dim;     /* D: 64, 128 or 256 */
  int32_t rotary_dim;   /* R: 0 or a multiple of 16 <= D */
  int32_t norm;         /* DanFrontNorm, the same for q and k */
  int32_t page_size, num_pages;
  int32_t table_width, num_seqs; /* table [num_seqs, table_width] */
  int32_t num_rope_rows;         /* rows of cos and sin */
  float eps;

  const void *q; int64_t q_stride_tok, q_stride_head; /* [N, H, D] */
  const void *k; int64_t k_stride_tok, k_stride_head; /* [N, Hkv, D] */
  const void *v; int64_t v_stride_tok, v_stride_head; /* [N, Hkv, D] */
  const void *cos; const void *sin; int64_t cs_stride_tok;
  const void *q_norm_weight, *k_norm_weight; /* [D], NULL when norm is NONE */
  void *q_out; int64_t qo_stride_tok, qo_stride_head; /* [N, H, D] */

  void *k_cache; int64_t kc_stride_page, kc_stride_head, kc_stride_tok;
  void *v_cache; int64_t vc_stride_page, vc_stride_head, vc_stride_tok;
  const float *k_scale, *v_scale; /* e4m3: one fp32 each on the device, x ~ xq * scale; else NULL */
  const int32_t *table; int64_t table_stride;
  const int32_t *places;    /* [N]: the token's place in its sequence; a negative one is not stored */
  const int32_t *seqs;      /* [N]: its row of the table; NULL: token n belongs to sequence n */
  const int32_t *rope_rows; /* [N]: its row of cos and sin; NULL: row n */
} DanPagedAppendArgs;

/* Normalizes and rotates q and k, writes q to q_out and k and v to the cache,
 * in fp32 with one rounding at each store (an e4m3 cache: x / scale, clamped to
 * +-448). A token without a place (negative, past its sequence's table, of a
 * sequence or in a page that does not exist) is not stored; a rotary row that
 * does not exist makes the rotated values NaN. Two tokens of one place leave
 * either one's row, or pieces of both. Stands beside dan_qkv_front
 * (dan/models/llama.py:78-86, dan/models/qwen3_5.py:318-326). */
int dan_paged_append(const DanPagedAppendArgs *args, void *stream);

typedef struct {
  int32_t abi_version;  /* DAN_PAGED_ABI_VERSION */
  int32_t dtype;        /* DanDtype of q and out: bf16 or f16 */
  int32_t cache_dtype;  /* the same, or e4m3 */
  int32_t num_seqs;     /* B */
  int32_t num_heads, num_kv_heads, head_dim;
  int32_t page_size, num_pages, table_width;
  int32_t max_len;      /* the longest sequence that the launch covers, <= table_width * page_size */
  float scale;          /* of the scores, > 0 and at most 2^127 */

  const void *q; int64_t q_stride_seq, q_stride_head; /* [B, H, D] */
  void *out; int64_t o_stride_seq, o_stride_head;     /* [B, H, D] */
  float *lse;           /* [B, H]: log of the sum of e^score, or NULL */
  const void *k_cache; int64_t kc_stride_page, kc_stride_head, kc_stride_tok;
  const void *v_cache; int64_t vc_stride_page, vc_stride_head, vc_stride_tok;
  const float *k_scale, *v_scale;
  const int32_t *table; int64_t table_stride;
  const int32_t *lens;  /* [B]: keys of each sequence */
  void *workspace; int64_t workspace_bytes; /* dan_paged_attn_workspace_size bytes, 16-byte aligned */
} DanPagedAttnArgs;

/* out[b, h] = softmax(scale q[b, h] . k) v over the sequence's first lens[b]
 * keys; zeros (lse -inf) where lens[b] is 0; NaN where lens[b] lies outside
 * [0, max_len] or one of its pages outside the cache. The whole table
 * [B, table_width], rows behind a sequence's end in its last page, and page 0
 * may be loaded; no result depends on what they hold. */
int dan_paged_attn(const DanPagedAttnArgs *args, void *stream);

/* Bytes of workspace of such a call on the current device (0: none is
 * needed; -1: invalid arguments). */
int64_t dan_paged_attn_workspace_size(int32_t cache_dtype, int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                      int32_t max_len);

/* DAN_PAGED_ABI_VERSION of the loaded library. */
int dan_paged_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* DAN_PAGED_H */
