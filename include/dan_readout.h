/*
 * dan_readout.h -- C ABI of the gfx950 readout: log probabilities of given
 * tokens, their distribution's logsumexp and entropy, and its top tokens,
 * with the gradient of the logits.
 *
 * dan answers with the softmax over the label tokens' logits of a read row
 * (dan/models/llama.py:163-165, dan/readout.py:13-17). These entry points
 * take whole rows of logits: the same labels against the whole vocabulary.
 *
 * Conventions: as dan_tree_attn.h. Rows of logits need no alignment beyond
 * their type's.
 */
#ifndef DAN_READOUT_H
#define DAN_READOUT_H

#include <stdint.h>

#include "dan_tree_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 2. The calls take version 1 as well: the structures without their last field, logsumexp_rest. */
#define DAN_READOUT_ABI_VERSION 2

/* At most so many top tokens, and so many values in a row whose top tokens are asked for. */
#define DAN_READOUT_MAX_TOP 32
#define DAN_READOUT_MAX_TOP_VOCAB 524288

typedef struct {
  int32_t abi_version; /* DAN_READOUT_ABI_VERSION, or 1 */
  int32_t dtype;       /* DanDtype of the logits (and of their gradient): bf16, f16 or f32 */
  int32_t rows;        /* N */
  int32_t vocab;       /* V >= 1 */
  int32_t labels;      /* L: given tokens of each row */
  int32_t top;         /* K: 0 .. DAN_READOUT_MAX_TOP, at most V */
  const void *logits; int64_t logits_stride;   /* [N, V] */
  const int64_t *tokens; int64_t tokens_stride; /* [N, L], unit stride along a row */
  float *logprobs;     /* [N, L] contiguous */
  float *logsumexp;    /* [N] */
  float *entropy;      /* [N] or NULL: not computed */
  float *top_logprobs; /* [N, K] */
  int64_t *top_ids;    /* [N, K] */
  void *workspace; int64_t workspace_bytes; /* dan_logprobs_workspace_size bytes, 16-byte aligned */
  float *logsumexp_rest; /* [N] or NULL: what rounding to fp32 took from logsumexp (0 where that is not finite) */
} DanLogprobsArgs;

/* logprobs[n, l] = x[n, tokens[n, l]] - logsumexp[n]; a negative token is
 * padding and gives 0, one >= V gives NaN. entropy in nats. The top tokens by
 * falling logit, equal ones by rising index. A row whose every logit is -inf
 * has logsumexp and log probabilities -inf and entropy 0; one that holds a NaN
 * or +inf has NaN throughout (its top_ids are some tokens of the row). */
int dan_logprobs_fwd(const DanLogprobsArgs *args, void *stream);

/* Bytes of workspace of such a call (0: invalid arguments). */
int64_t dan_logprobs_workspace_size(int32_t dtype, int32_t rows, int32_t vocab, int32_t top);

typedef struct {
  int32_t abi_version; /* DAN_READOUT_ABI_VERSION, or 1 */
  int32_t dtype, rows, vocab, labels, top;
  const void *logits; int64_t logits_stride;
  const int64_t *tokens; int64_t tokens_stride;
  const float *logsumexp;     /* [N], of the forward call */
  const float *entropy;       /* [N], of the forward call; NULL where g_entropy is */
  const int64_t *top_ids;     /* [N, K], of the forward call; NULL where g_top is */
  const float *g_logprobs;    /* [N, L] contiguous, or NULL */
  const float *g_logsumexp;   /* [N] or NULL */
  const float *g_entropy;     /* [N] or NULL */
  const float *g_top;         /* [N, K] contiguous, or NULL */
  void *grad; int64_t grad_stride; /* [N, V] of dtype */
  const float *logsumexp_rest; /* [N], of the forward call; NULL: zeros, which leaves each p off by half a unit of logsumexp
                                  (2^-24 |logsumexp| of p: all of it where that is 2^24 and more) */
} DanLogprobsGradArgs;

/* grad[n, j] = sum_l g_l [tokens_l = j] + sum_k h_k [top_k = j]
 *            + p_j (g_logsumexp - sum g - sum h - g_entropy (log p_j + entropy))
 * in fp32, rounded once; equal tokens add up; padding has no gradient. */
int dan_logprobs_bwd(const DanLogprobsGradArgs *args, void *stream);

/* DAN_READOUT_ABI_VERSION of the loaded library. */
int dan_readout_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* DAN_READOUT_H */
