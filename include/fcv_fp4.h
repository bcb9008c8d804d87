/*
 * fcv_fp4.h -- C ABI of the speech language model's operators in 4 bits, in libfcvdit.so: a linear
 * layer over 4-bit weights, and a key/value cache of 4-bit pages with its append, its attention and
 * copies of its pages.  Beside those of fcv_lm.h, whose conventions hold: device pointers unless a
 * name ends in _host, FCV_OK or an error code (message in fcv_last_error()), no allocation, stateless
 * and asynchronous on `stream` of the current device, fit for capture into a hipGraph.
 *
 *   fcv_fp4_quantize    rows of weights -> 4-bit numbers and scales
 *   fcv_fp4_linear      y = act(x W^T + bias) + residual over such weights
 *   fcv_fp4_append      norms of queries and keys per head, the rotation, and the append of keys and
 *                       values to the pages in 4 bits, in one pass over a packed QKV projection
 *   fcv_fp4_attention   causal attention of a batch over its pages
 *   fcv_fp4_read        keys and values of tokens in the pages, as 16-bit numbers
 *   fcv_copy_pages      pages copied to others, in all layers
 *
 * The 4-bit format is the microscaling one (OCP MXFP4) that the MI355X converts in hardware.  A code of
 * four bits is a sign, two exponent bits and one mantissa bit: the numbers 0, 1/2, 1, 3/2, 2, 3, 4, 6 and
 * their negatives.  Codes lie in pairs in a byte, the first in the low half.  A group of codes has a
 * scale byte b, 2^(b - 127); 255 is NaN and makes the whole group NaN.
 *
 * A group is quantized with the smallest exponent e for which every magnitude is below 7 2^e (so that
 * clipping to 6 2^e is off by half a step at most), kept within [-125, 125] for bf16 and fp32 and
 * [-23, 13] for fp16, where each number times 2^e is one of the type's; past these limits values clip to
 * 6 2^e, or go to 0.  Values go to the nearest number, ties to the even code.  A group that holds an
 * infinity or NaN gets the scale 255.
 */
#ifndef FCV_FP4_H
#define FCV_FP4_H

#include "fcv_lm.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FCV_FP4_GROUP 32 /* elements of a weight row or a key that share a scale */
#define FCV_FP4_PAGE 64  /* tokens of a page */

/* Rows [n][k] of weights to codes [n][16 ceil(k / 32)] bytes and scales [n][ceil(k / 32)] bytes; what
 * lies past k in a row's last group are zeros.  Strides: ldw in elements, the others in bytes. */
typedef struct FcvFp4Quantize {
  const void* w;
  uint8_t* codes;
  uint8_t* scales;
  int64_t ldw;
  int64_t ld_codes;  /* a multiple of 16, codes on a 16-byte boundary */
  int64_t ld_scales;
  int32_t n;
  int32_t k;
  int32_t dtype;     /* FCV_LM_F16, FCV_LM_BF16 or FCV_LM_F32 */
} FcvFp4Quantize;

int fcv_fp4_quantize(const FcvFp4Quantize* args, hipStream_t stream);

/* y[i][j] = act(sum_k x[i][k] w[j][k] + bias[j]) + residual[i][j] as fcv_lm_linear computes it, where
 * w[j][k] is code k of row j times the scale of its group of 32, rounded to x's type (exact within the
 * limits above).  Codes past k are not looked at.  m and n up to 2^22, their product up to 2^34, k up
 * to 2^21, ld_codes and ld_scales below 2^24. */
typedef struct FcvFp4Linear {
  const void* x;         /* [m][k], row stride ldx */
  const uint8_t* codes;  /* [n][16 ceil(k / 32)], row stride ld_codes */
  const uint8_t* scales; /* [n][ceil(k / 32)], row stride ld_scales */
  const void* bias;      /* [n] or NULL */
  const void* residual;  /* [m][n], row stride ldr, or NULL */
  void* y;               /* [m][n], row stride ldy */
  int64_t ldx;
  int64_t ld_codes;      /* bytes, a multiple of 16; codes on a 16-byte boundary */
  int64_t ld_scales;     /* bytes */
  int64_t ldr;
  int64_t ldy;
  int32_t m;
  int32_t n;
  int32_t k;
  int32_t dtype;          /* of x: FCV_LM_F16 or FCV_LM_BF16 */
  int32_t bias_dtype;     /* dtype or FCV_LM_F32 */
  int32_t residual_dtype; /* dtype or FCV_LM_F32 */
  int32_t y_dtype;        /* dtype or FCV_LM_F32 */
  int32_t activation;
} FcvFp4Linear;

/* Workspace of one call: 0 where none is needed (NULL is then fine), else 256-byte aligned. */
size_t fcv_fp4_linear_workspace_bytes(const FcvFp4Linear* args);
int fcv_fp4_linear(const FcvFp4Linear* args, void* workspace, size_t workspace_bytes,
                   hipStream_t stream);
/* Which kernel a call takes and into how many ranges it cuts k, for logs and tests.  form: 0 up to 32 rows,
 * else tiles of 1 64 x 64, 2 64 x 128, 3 128 x 128, 4 128 x 256, 5 192 x 256, 6 256 x 256. */
int fcv_fp4_linear_plan(const FcvFp4Linear* args, int32_t* form, int32_t* ranges);

/* Pages: a pool [pages][n_kv_heads][page bytes], strides page_stride and head_stride in bytes,
 * multiples of 16 and on 16-byte boundaries.  A page holds 64 tokens; per head, with D = head_dim,
 *   keys    [64][D / 2]    byte j of a token has elements 2 j and 2 j + 1
 *   values  [D / 2][64]    byte j of a token has elements 2 j and 2 j + 1
 *   scales of the keys    [64][D / 32]
 *   scales of the values  [64], one for a token's D elements
 * one behind the other: fcv_fp4_page_bytes(D) = 64 (D + D / 32 + 1) bytes; 0 for another D. */
size_t fcv_fp4_page_bytes(int32_t head_dim);

/* fcv_lm_qk_norm_rope over pages: token t's key and value go to place cache_rows[t] % 64 of page
 * cache_rows[t] / 64, in 4 bits; a negative row or one past the pool goes nowhere.  A key's norm and
 * rotation are computed in 64 bits, so that its codes are those of the formula.  q_out may be the queries' own
 * columns of qkv (same start and row stride); it and the pages overlap nothing else. */
typedef struct FcvFp4Append {
  const void* qkv;           /* [tokens][(n_heads + 2 n_kv_heads) head_dim], row stride qkv_row */
  const int32_t* positions;  /* [tokens] */
  const int32_t* cache_rows; /* [tokens] */
  const float* rope_cos;     /* [max_pos][rope_dim / 2] */
  const float* rope_sin;
  const void* q_weight;      /* [head_dim], or both NULL */
  const void* k_weight;
  void* q_out;               /* [tokens][n_heads][head_dim], row stride q_row */
  uint8_t* pages;
  int64_t qkv_row;
  int64_t q_row;
  int64_t page_stride;
  int64_t head_stride;
  int32_t tokens;
  int32_t n_heads;
  int32_t n_kv_heads;
  int32_t head_dim;
  int32_t rope_dim;
  int32_t max_pos;
  int32_t n_pages;
  int32_t dtype;
  int32_t weight_dtype;      /* dtype or FCV_LM_F32 */
  int32_t interleaved;
  float eps;
} FcvFp4Append;

int fcv_fp4_append(const FcvFp4Append* args, hipStream_t stream);

/* Token t's key and value heads, from place rows[t] of the pages: k and v [tokens][n_kv_heads][head_dim]
 * at row strides k_row and v_row, rounded to dtype.  A row outside the pool gives zeros. */
typedef struct FcvFp4Read {
  const uint8_t* pages;
  const int32_t* rows; /* [tokens] */
  void* k;
  void* v;
  int64_t page_stride;
  int64_t head_stride;
  int64_t k_row;
  int64_t v_row;
  int32_t tokens;
  int32_t n_kv_heads;
  int32_t head_dim;
  int32_t n_pages;
  int32_t dtype;
} FcvFp4Read;

int fcv_fp4_read(const FcvFp4Read* args, hipStream_t stream);

/* Rows cu_q[b] .. cu_q[b + 1] - 1 of q (cu_q[0] = 0, non-decreasing) are the last queries of sequence b,
 * n of them: query i sees keys 0 .. lengths[b] - n + i of the sequence, whose key j is place j % 64 of
 * page table[b][j / 64] (the new tokens' keys are there already).  With s = scale q.k over the visible
 * keys
 *   out = sum exp(s) v / sum exp(s),   lse = log sum exp(s).
 * A query that sees no key gives out = 0 and lse = -inf.  A page that is negative or past the pool
 * has no keys, lengths are clipped to [0, 64 max_pages], and what lies behind a sequence's last key does
 * not touch its result.  Query head h reads key head h / (n_heads / n_kv_heads).  Rows of q past
 * cu_q[batch] are not read, and their rows of out and lse stay as they were.  cu_q NULL: tokens / batch
 * rows for every sequence.  max_q and max_length bound the new tokens and the keys of a sequence: they
 * shape the launch, and a batch that passes them is computed all the same, more slowly.  Pages may be
 * shared between sequences.  tokens * n_heads is below 2^24, n_pages at most 2^24.  Numbers of the
 * pages are rounded to q's type (exact within the limits above for pages written in that type); results
 * below 2^-64 lose bits, because sums of bf16's largest values have to fit fp32. */
typedef struct FcvFp4Attention {
  const void* q;          /* [tokens][n_heads][head_dim], strides q_row, q_head */
  const uint8_t* pages;
  const int32_t* table;   /* [batch][max_pages], row stride table_row */
  const int32_t* lengths; /* [batch] */
  const int32_t* cu_q;    /* [batch + 1] or NULL */
  void* out;              /* [tokens][n_heads][head_dim], strides out_row, out_head; may be q itself */
  float* lse;             /* [tokens][n_heads] or NULL */
  int64_t q_row;
  int64_t q_head;
  int64_t out_row;
  int64_t out_head;
  int64_t page_stride;
  int64_t head_stride;
  int64_t table_row;
  int32_t tokens;
  int32_t batch;
  int32_t n_heads;
  int32_t n_kv_heads;
  int32_t head_dim;
  int32_t n_pages;
  int32_t max_pages;
  int32_t max_q;
  int32_t max_length;
  int32_t dtype;
  float scale;            /* > 0 */
} FcvFp4Attention;

/* Workspace of one call (partial sums of the split key ranges): 256-byte aligned. */
size_t fcv_fp4_attention_workspace_bytes(const FcvFp4Attention* args);
int fcv_fp4_attention(const FcvFp4Attention* args, void* workspace, size_t workspace_bytes,
                      hipStream_t stream);
/* How a call is launched, for logs and tests: tiles of 8, 16 or 128 rows (a row is a query's head), how many of
 * them a sequence's key head has (a batch that passes max_q gives each several in turn), into how many ranges its
 * pages are cut, and whether the longest sequences are taken first (1) or each in its place (0). */
int fcv_fp4_attention_plan(const FcvFp4Attention* args, int32_t* rows, int32_t* tiles, int32_t* ranges,
                           int32_t* ordered);

/* Page src_host[i] of every layer is copied to page dst_host[i], for i < count: a fork (one source, many
 * destinations) or a compaction.  No page is a destination twice, or both a source and a destination.
 * Any pool of `layers` layers of `n_pages` pages of page_bytes contiguous bytes; the host arrays are read
 * before the call returns. */
int fcv_copy_pages(void* pages, int32_t layers, int64_t layer_stride, int32_t n_pages,
                   int64_t page_stride, int64_t page_bytes, const int32_t* src_host,
                   const int32_t* dst_host, int32_t count, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* FCV_FP4_H */
