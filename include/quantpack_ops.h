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
 * out may be query itself (the same address and strides); otherwise it shares no memory with query, key and value.
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
  int32_t max_seqlen_k;        /* longest sequence's keys: what the work is laid out by, with any value correct */
  int32_t num_splits;          /* key splits per row block, at most 128; 1 = one walk over the keys; 0 = automatic */
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

/*
 * The attention weight that each cached key receives from the query rows of its sequence, per KV head:
 *   out[i, g, j] = decay previous[i, g, j] + sum over tokens t and query heads h of KV head g of p(t, h, j),  j < seqused_k[i]
 * with p the softmax of softmax_scale q.k over the dequantised keys (of the int4 or int8 key half) at positions up to the
 * token's own; the tokens of sequence i are its last cu_seqlens_q[i + 1] - cu_seqlens_q[i] positions. Entries from
 * seqused_k[i] on are left as they are. A token that sees no key adds nothing; a sequence without tokens keeps its
 * decayed weights. A key on a page outside 0 .. num_blocks - 1 is not seen and gets no weight.
 * A query of NaN gives NaN to the keys that it sees, and nothing to the others.
 * previous may be out itself (the same address and strides); otherwise the two share no memory. With previous NULL, or
 * decay 0, earlier weights are not read.
 */
typedef struct qp_key_weights_args {
  qp_cache_half key;
  int32_t num_blocks;
  int32_t block_size;
  int32_t num_kv_heads;
  int32_t head_size;           /* 64, 128, 256 or 512 */
  const void *query;           /* bf16 [num_tokens, num_q_heads, head_size], in the cache's (rotated) domain */
  int64_t query_stride[2];     /* elements: token, head; rows 16-byte aligned */
  const int32_t *cu_seqlens_q; /* [num_seqs + 1] */
  const int32_t *seqused_k;    /* [num_seqs]: context length including the query tokens */
  const int32_t *block_table;  /* [num_seqs, block_table_stride], max_blocks entries of a row used */
  int64_t block_table_stride;
  int32_t max_blocks;
  int32_t num_seqs;
  int32_t num_tokens;
  int32_t num_q_heads;
  int32_t max_query_len;       /* longest sequence's query tokens; tokens beyond it are not counted */
  int32_t max_seqlen_k;        /* longest context (at most the last dimension of out); keys beyond it are not seen */
  float softmax_scale;         /* positive; multiplies q.k in the cache's domain */
  float decay;
  const float *query_signs;    /* optional: q is unrotated and rotated on load, as in qp_decode_args */
  const float *previous;       /* optional fp32 [num_seqs, num_kv_heads, >= max_seqlen_k], positions contiguous */
  int64_t previous_stride[2];  /* elements: sequence, head */
  float *out;                  /* fp32 [num_seqs, num_kv_heads, >= max_seqlen_k], positions contiguous */
  int64_t out_stride[2];
  void *workspace;             /* >= qp_key_weights_workspace_size bytes, 16-byte aligned */
  int64_t workspace_bytes;
} qp_key_weights_args;

int qp_key_weights(const qp_key_weights_args *args, qp_stream_t stream);

/* Workspace bytes qp_key_weights uses for these arguments on the current device. */
int64_t qp_key_weights_workspace_size(const qp_key_weights_args *args);

/*
 * Eviction from a paged cache: per sequence i and KV head g, of the n = seqused_k[i] keys the first `sinks` and last
 * `recent` stay, and of the others those of largest weight (NaN counts as the smallest, of equal weights the lower
 * position stays), min(n, budget) in all. Their positions go to kept[i, g, :] in ascending order, their weights to
 * new_weights[i, g, :], and their cells (key and value codes and words) to slots 0, 1, .. of new_block_table[i]; the
 * sequence's new length to new_seqused_k[i]. Heads choose for themselves, so a slot holds different positions in
 * different heads: keys carry their position with them (rotary embeddings are applied before the store).
 * The new blocks must not be blocks that the call still reads, of any sequence. Slots past the kept cells are left as they
 * are, as are entries of kept and new_weights past the count. A cell whose old or new page is outside 0 .. num_blocks - 1
 * is not moved.
 */
typedef struct qp_evict_args {
  const float *weights;           /* fp32 [num_seqs, num_kv_heads, >= max_seqlen_k], positions contiguous */
  int64_t weights_stride[2];      /* elements: sequence, head */
  const int32_t *seqused_k;       /* [num_seqs] */
  const int32_t *block_table;     /* [num_seqs, block_table_stride], max_blocks entries of a row used */
  int64_t block_table_stride;
  const int32_t *new_block_table; /* [num_seqs, new_block_table_stride], new_max_blocks entries of a row used */
  int64_t new_block_table_stride;
  int32_t max_blocks;
  int32_t new_max_blocks;         /* with room for min(max_seqlen_k, budget) positions */
  int32_t num_seqs;
  int32_t max_seqlen_k;           /* longest context; positions beyond it do not exist for the call */
  int32_t budget;                 /* at least sinks + recent, and 1 */
  int32_t sinks;
  int32_t recent;
  int32_t *kept;                  /* int32 [num_seqs, num_kv_heads, >= budget], contiguous in the last dimension;
                                     kept and new_weights share no memory with weights */
  int64_t kept_stride[2];
  float *new_weights;             /* fp32 [num_seqs, num_kv_heads, >= budget]; not the memory of weights */
  int64_t new_weights_stride[2];
  int32_t *new_seqused_k;         /* [num_seqs]; not the memory of seqused_k */
  void *workspace;                /* >= qp_evict_workspace_size bytes, 8-byte aligned */
  int64_t workspace_bytes;
} qp_evict_args;

int qp_evict(const qp_paged_cache *cache, const qp_evict_args *args, qp_stream_t stream);

/* Workspace bytes qp_evict uses for these arguments. */
int64_t qp_evict_workspace_size(const qp_paged_cache *cache, const qp_evict_args *args);

#ifdef __cplusplus
}
#endif

#endif /* QUANTPACK_OPS_H */
