/*
 * quantpack_ops.h - operators of libquantpack_hip.so around the quantised cache that quantpack.h serves: attention over a
 * prompt's own keys and values, the weight that cached keys receive, and the eviction of the others.
 *
 * None of them replaces an interface of vllm-quantpack. Conventions (pointers, strides, status codes, no allocation, no
 * waiting for the device) are those of quantpack.h.
 */
#ifndef QUANTPACK_OPS_H
#define QUANTPACK_OPS_H

#include "quantpack.h"

#ifdef __cplusplus
extern "C" {
#endif

#define QP_DTYPE_F16 2 /* beside QP_DTYPE_BF16 and QP_DTYPE_F32 */

/*
 * Attention of packed sequences over keys and values that are not quantised (a prompt's own, before they are stored):
 * row (t, h) of sequence i attends the keys j <= t + keys_i - tokens_i of its sequence (all of them when causal is 0)
 * of KV head h / (num_q_heads / num_kv_heads); out = sum_j p_j v_j with p the softmax of softmax_scale q.k, the two
 * products in the tensors' type with fp32 sums. A row that sees no key gives zeros and an lse of -inf; rows of q past
 * cu_seqlens_q[num_seqs] are left as they are. Keys and values that no row sees may hold anything, NaN included.
 * When the rows alone cannot fill the GPU the keys are split over workgroups (num_splits, 0 = automatic) whose fp32
 * partials go to the workspace; an automatic choice without enough workspace falls back to one split.
 */
typedef struct qp_prompt_args {
  const void *query;           /* [num_tokens, num_q_heads, head_size], channels contiguous, rows 16-byte aligned */
  int64_t query_stride[2];     /* elements: token, head (all strides) */
  const void *key;             /* [num_keys, num_kv_heads, head_size] */
  int64_t key_stride[2];
  const void *value;
  int64_t value_stride[2];
  const int32_t *cu_seqlens_q; /* [num_seqs + 1] */
  const int32_t *cu_seqlens_k; /* [num_seqs + 1]; the same as cu_seqlens_q for prompts with nothing before them */
  int32_t num_seqs;
  int32_t num_tokens;
  int32_t num_keys;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_size;           /* 64, 128, 256 or 512 */
  int32_t dtype;               /* QP_DTYPE_BF16 or QP_DTYPE_F16: query, key, value and out */
  int32_t max_seqlen_k;        /* longest sequence's keys: bounds the automatic split count */
  int32_t num_splits;          /* key splits per row block, at most 128; 0 = automatic */
  int32_t causal;
  float softmax_scale;         /* positive */
  void *out;                   /* [num_tokens, num_q_heads, head_size] */
  int64_t out_stride[2];
  float *lse;                  /* optional: fp32 [num_tokens, num_q_heads], natural log of the row's sum of exponentials */
  int64_t lse_stride[2];
  void *workspace;             /* >= qp_prompt_workspace_size bytes, 16-byte aligned; may be NULL */
  int64_t workspace_bytes;
} qp_prompt_args;

int qp_prompt(const qp_prompt_args *args, qp_stream_t stream);

/* Workspace bytes qp_prompt uses for these arguments on the current device (0 when it does not split). */
int64_t qp_prompt_workspace_size(const qp_prompt_args *args);

#ifdef __cplusplus
}
#endif

#endif /* QUANTPACK_OPS_H */
