/*
 * fcv_lm.h -- C ABI of the speech language model's operators in libfcvdit.so: a decoder layer's
 * products, rotation, cache append and attention.  Norms of whole rows and a gate's product with its
 * branch are not among them.  The reference leaves that
 * model to a separate engine process (faster_cosyvoice/llm/engine.py:94-141), so nothing here
 * mirrors one of its interfaces.
 *
 *   fcv_lm_linear            y = act(x W^T + bias) + residual
 *   fcv_lm_qk_norm_rope      norms of queries and keys per head, the position rotation and the
 *                            cache append, in one pass over a packed QKV projection
 *   fcv_lm_prefix_attention  attention of a batch whose sequences share one prompt (a voice's
 *                            reference) in front of caches of their own
 *
 * Conventions are those of fcv_dit.h: device pointers, FCV_OK or an error code (message in
 * fcv_last_error()), no allocation.  The calls are stateless and asynchronous on `stream`, which
 * belongs to the current device; they may be captured into a hipGraph, and calls on different
 * streams need different workspaces.  fp16 and bf16 tensors, sums and softmax statistics in fp32.
 * Strides are in elements, and the innermost dimension is contiguous; what is said of strides is not
 * asked of a dimension of one entry.  Results do not depend on earlier calls or on timing (but for two
 * tokens that name one cache row); they may differ in the last bits between batch sizes, because the
 * order of a sum follows the sizes.
 */
#ifndef FCV_LM_H
#define FCV_LM_H

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "fcv_dit.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define FCV_LM_F16 0
#define FCV_LM_BF16 1
#define FCV_LM_F32 2 /* bias, residual, norm weights and the linear layer's output only */

/* activations: max(z, 0); z sigmoid(z); z Phi(z) (erf); its tanh form */
#define FCV_LM_ACT_NONE 0
#define FCV_LM_ACT_RELU 1
#define FCV_LM_ACT_SILU 2
#define FCV_LM_ACT_GELU 3
#define FCV_LM_ACT_GELU_TANH 4

/* y[i][j] = act(sum_k x[i][k] w[j][k] + bias[j]) + residual[i][j], rounded once; m and n
 * up to 2^22, their product up to 2^34, k up to 2^28.  Rows may start on any
 * element's boundary; where all rows of x and w start on 16-byte ones and k is a multiple of 8, many
 * rows go faster.  y may be the residual itself (same type and stride); it
 * overlaps nothing else. */
typedef struct FcvLmLinear {
  const void* x;        /* [m][k], row stride ldx */
  const void* w;        /* [n][k], row stride ldw */
  const void* bias;     /* [n] or NULL */
  const void* residual; /* [m][n], row stride ldr, or NULL */
  void* y;              /* [m][n], row stride ldy */
  int64_t ldx;
  int64_t ldw;
  int64_t ldr;
  int64_t ldy;
  int32_t m;
  int32_t n;
  int32_t k;
  int32_t dtype;          /* of x and w: FCV_LM_F16 or FCV_LM_BF16 */
  int32_t bias_dtype;     /* dtype or FCV_LM_F32 */
  int32_t residual_dtype; /* dtype or FCV_LM_F32 */
  int32_t y_dtype;        /* dtype or FCV_LM_F32 */
  int32_t activation;
} FcvLmLinear;

/* Workspace of one call: 0 where none is needed (NULL is then fine), else 256-byte aligned. */
size_t fcv_lm_linear_workspace_bytes(const FcvLmLinear* args);
int fcv_lm_linear(const FcvLmLinear* args, void* workspace, size_t workspace_bytes,
                  hipStream_t stream);
/* Which kernel a call takes and into how many ranges it cuts k, for logs and tests.  form: 0 any
 * alignment, 1 up to 16 rows, else tiles of 2 64 x 64, 3 64 x 128, 4 128 x 128, 5 128 x 256, 6 192 x 256,
 * 7 256 x 256, 8 128 x 128 in launches of few. */
int fcv_lm_linear_plan(const FcvLmLinear* args, int32_t* form, int32_t* ranges);

/* Token t's row of qkv holds n_heads query heads, n_kv_heads key heads and n_kv_heads value heads
 * of head_dim (64 or 128) elements.  Every query and key head x becomes
 *   x / sqrt(mean(x^2) + eps) * weight      (unchanged where the weights are NULL),
 * then its first rope_dim elements are rotated by the angles of row positions[t] of the tables:
 * pairs (i, i + rope_dim / 2), or (2 i, 2 i + 1) where interleaved is set.  Both steps run in fp32
 * and round once.  Queries go to q_out; keys and values (as they are) go to row cache_rows[t] of
 * the caches, session cache_rows[t] / capacity, key cache_rows[t] % capacity.  A token whose
 * cache row is negative or past the caches writes no key and no value (a padded batch).  Of tokens
 * that name the same cache row any one's values may remain, elementwise.  A position outside the
 * tables reads their first or last row.  rope_dim is a multiple of 16 from 16 to head_dim; all
 * strides are multiples of 8 and all tensors start on 16-byte boundaries.  q_out may be the queries' own
 * columns of qkv (same start and row stride); it and the caches overlap nothing else. */
typedef struct FcvLmQkNormRope {
  const void* qkv;           /* [tokens][(n_heads + 2 n_kv_heads) head_dim], row stride qkv_row */
  const int32_t* positions;  /* [tokens] */
  const int32_t* cache_rows; /* [tokens] */
  const float* rope_cos;     /* [max_pos][rope_dim / 2] */
  const float* rope_sin;
  const void* q_weight;      /* [head_dim], or both NULL */
  const void* k_weight;
  void* q_out;               /* [tokens][n_heads][head_dim], row stride q_row */
  void* k_cache;             /* [sessions][capacity][n_kv_heads][head_dim] by its strides */
  void* v_cache;
  int64_t qkv_row;
  int64_t q_row;
  int64_t k_session;
  int64_t k_row;
  int64_t k_head;
  int64_t v_session;
  int64_t v_row;
  int64_t v_head;
  int32_t tokens;
  int32_t n_heads;
  int32_t n_kv_heads;
  int32_t head_dim;
  int32_t rope_dim;
  int32_t max_pos;
  int32_t sessions;
  int32_t capacity;
  int32_t dtype;
  int32_t weight_dtype;      /* dtype or FCV_LM_F32 */
  int32_t interleaved;
  float eps;
} FcvLmQkNormRope;

int fcv_lm_qk_norm_rope(const FcvLmQkNormRope* args, hipStream_t stream);

/* Rows cu_q[b] .. cu_q[b + 1] - 1 of q (cu_q[0] = 0, non-decreasing) are the last queries of sequence b,
 * n of them: query i sees
 * every key of the prefix (prefix_len of them, may be 0) and the keys of row slots[b] of the caches
 * up to its own, 0 .. lengths[b] - n + i (the new tokens' keys are in the cache already).  With
 * s = scale q.k over the visible keys
 *   out = sum exp(s) v / sum exp(s),   lse = log sum exp(s).
 * A query that sees no key gives out = 0 and lse = -inf; keys and values that a query does not see
 * do not touch its result, whatever they hold.  Of the values that it sees an infinity is what it
 * gets, however small the weight, and NaN for NaN or both infinities.  Query head h reads key head
 * h / (n_heads / n_kv_heads).  Rows of q past cu_q[batch] are not read, and their rows of out and lse stay as they
 * were.  cu_q NULL: tokens / batch rows for every sequence; slots NULL: sequence b has session b.
 * lengths are clipped to [0, capacity], and a slot outside [0, sessions) has no keys.
 * max_q and max_length bound the new tokens and the keys of a sequence: they shape the launch, and
 * a batch that passes them is computed all the same, more slowly.
 * prefix_len and capacity are at most 2^29, tokens * n_heads is below 2^26; head_dim is 64 or 128;
 * strides are multiples of 8 and tensors start on 16-byte boundaries; a key's or value's row stride is
 * below 2^24.  out may be q itself (same strides); it overlaps nothing else. */
typedef struct FcvLmAttention {
  const void* q;          /* [tokens][n_heads][head_dim], strides q_row, q_head */
  const void* prefix_k;   /* [prefix_len][n_kv_heads][head_dim] */
  const void* prefix_v;
  const void* k_cache;    /* [sessions][capacity][n_kv_heads][head_dim] */
  const void* v_cache;
  const int32_t* cu_q;    /* [batch + 1] or NULL */
  const int32_t* lengths; /* [batch] */
  const int32_t* slots;   /* [batch] or NULL */
  void* out;              /* [tokens][n_heads][head_dim], strides out_row, out_head */
  float* lse;             /* [tokens][n_heads] or NULL */
  int64_t q_row;
  int64_t q_head;
  int64_t out_row;
  int64_t out_head;
  int64_t pk_row;
  int64_t pk_head;
  int64_t pv_row;
  int64_t pv_head;
  int64_t k_session;
  int64_t k_row;
  int64_t k_head;
  int64_t v_session;
  int64_t v_row;
  int64_t v_head;
  int32_t tokens;
  int32_t batch;
  int32_t n_heads;
  int32_t n_kv_heads;
  int32_t head_dim;
  int32_t prefix_len;
  int32_t sessions;
  int32_t capacity;
  int32_t max_q;
  int32_t max_length;
  int32_t dtype;
  float scale;            /* > 0 */
} FcvLmAttention;

/* Workspace of one call (partial sums of the split key ranges): 256-byte aligned. */
size_t fcv_lm_prefix_attention_workspace_bytes(const FcvLmAttention* args);
int fcv_lm_prefix_attention(const FcvLmAttention* args, void* workspace, size_t workspace_bytes,
                            hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FCV_LM_H */
