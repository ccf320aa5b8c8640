/*
 * C ABI of the operators around dense latent attention: rotary positions, the append of rotated rows to a
 * paged cache, attention over that cache in absorbed form, and attention of prompts in expanded form.
 *
 * A call is described by a struct (host memory, read before the function returns). All pointers in it are
 * device pointers valid on the current device. Strides are in elements. Functions only enqueue work on `stream`
 * (a cudaStream_t) and never synchronise; 0 is success, -1 a call outside of what is stated here (nothing is
 * enqueued), anything else the CUDA error code of the failed enqueue.
 *
 * Ragged batches: request b owns tokens cu_seqlens_q[b] .. cu_seqlens_q[b + 1] - 1. Entries are taken to lie
 * between 0 and the number of tokens, non-decreasing (others are clamped to that range); tokens in front of the first
 * and behind the last request are not read, and their outputs stay as they are.
 *
 * `status`: SPARSE_MLA_STATUS_WORDS int32 words (sparse_mla.h), set to the first report if word 0 is zero:
 * SPARSE_MLA_STATUS_BAD_PAGE, token, position for a block-table entry outside of the cache (or a position behind the table),
 * whose rows are not written or not seen; SPARSE_MLA_STATUS_WAIT_EXPIRED where an on-chip wait gave up.
 */
#ifndef ASCENDFLOW_B200_LATENT_H_
#define ASCENDFLOW_B200_LATENT_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LATENT_F16 0
#define LATENT_BF16 1
#define LATENT_F32 2 /* rotary only */

#define LATENT_VALUES 512 /* value features of a latent row: its first ones */
#define LATENT_NOPE 128   /* expanded form: features per head of keys and of values */
#define LATENT_ROPE 64    /* expanded form: the shared rope key's features */
#define LATENT_MOST_PAIRS 128

/* out[t, h] = x[t, h] with its last 2 `pairs` features turned by positions[t] * inv_freq[i] radians and
 * multiplied by `amplitude` (finite in FP32). layout 0: pair i is features (2 i, 2 i + 1) of the turned part; 1: (i, i + pairs).
 * inverse: turned back. The features in front are copied, unless out is x. x and out are the same memory with the same
 * strides, or disjoint. Base addresses and strides are multiples of 16 bytes, `features` a multiple of 8 up to 65536,
 * `heads` up to 65536, `pairs` a multiple of 8 up to LATENT_MOST_PAIRS. positions: int32, or int64 with `positions64`; any value. */
typedef struct {
  int32_t type, layout, inverse, positions64;
  const void* x;
  void* out;
  const void* positions;  /* [T] */
  const double* inv_freq; /* [pairs] */
  int64_t x_token, x_head, out_token, out_head; /* strides */
  int64_t tokens, heads, features, pairs;
  double amplitude;
} latent_rotary_call;
int launch_latent_rotary(void* stream, const latent_rotary_call* call);

/* Row j of the n of request b goes to logical position p = seqused_kv[b] - n + j of the paged cache (seqused_kv counts
 * the new rows): `latent`, then `rope` turned by p * inv_freq[i] as above. width = latent's features (a
 * multiple of 8) + 2 pairs. latent_token is a multiple of 8, addresses of latent and cache of 16 bytes. */
typedef struct {
  int32_t type, layout;
  const void* latent; /* [T, width - 2 pairs] */
  const void* rope;   /* [T, 2 pairs] */
  void* cache;        /* [blocks, page_rows, 1, width] */
  const int32_t *block_table, *cu_seqlens_q, *seqused_kv; /* [B, pages], [B + 1], [B] */
  const double* inv_freq;
  int32_t* status;
  int64_t latent_token, rope_token; /* strides */
  int64_t batches, tokens, pages, blocks, page_rows, width, pairs;
  double amplitude;
} latent_append_call;
int launch_latent_append(void* stream, const latent_append_call* call);

/* Causal attention of every request's tokens over its cached rows, keys and values in one: key k of token j of n is
 * seen if k < seqused_kv[b] - n + j + 1; scores scale (1e-30 to 1e30) * q . row over all `width` (512 or 576) features, values are the
 * row's first 512. sinks (or NULL): a logit per head in the denominator. lse (or NULL): the natural
 * logarithm of the denominator. A token that sees no key gets zeros. page_rows: a multiple of 64.
 * Rows behind a request's length are never multiplied; rows within it have to be finite. Addresses of q, cache and out are
 * multiples of 16 bytes. */
typedef struct {
  int32_t type, reserved;
  const void* q;     /* [T, heads, width] */
  const void* cache; /* [blocks, page_rows, 1, width] */
  const int32_t *block_table, *cu_seqlens_q, *seqused_kv;
  const float* sinks; /* [heads] */
  void* out;          /* [T, heads, 512] */
  float* lse;         /* [T, heads] */
  void* workspace;
  int32_t* status;
  int64_t batches, tokens, heads, width, pages, blocks, page_rows;
  double scale;
} latent_attention_call;
/* Bytes of `workspace` (32-byte aligned) on the current device; its contents matter to nobody between calls, but calls that may run at the same time need one each. */
int workspace_size_latent_attention(uint64_t* bytes);
int launch_latent_attention(void* stream, const latent_attention_call* call);

/* ---- rows held in 8 bits ------------------------------------------------------------------------------------------------
 *
 * A cache of e4m3 numbers [blocks, page_rows, 1, width] with a scale for every `block_rows` rows of a page, [blocks, page_rows / block_rows]: a byte e stands for
 * 2^(e - 127), 255 for NaN (the e8m0 format). block_rows: a power of two up to 64. A held value is its number times its row's scale. */

/* The append of rotated rows: as launch_latent_append, with page_rows a multiple of 64, `width` one of 16 and `cache` of 8 bits. What is held is worked out in FP32 and
 * rounded once: numbers to the nearest e4m3 number after the division by the scale. A block's scale is the least power of two s with |v| <= 448 s for
 * all its new rows v, and, unless the first of these begins the block, not below the scale that the block has: where that grows, the numbers of the rows in front of the
 * new ones are divided by the growth and rounded to nearest. From half rows, values beyond 61440 (the greatest whose number times its scale half holds) are taken
 * as that. A row that is not finite makes its block's scale NaN, also for the rows in front of it. What a row has done to its block's scale and to the numbers in front of it stays when
 * the row is given up (a shorter length in the next call), until a new row begins the block. Values below 2^-126 count as zero. */
typedef struct {
  latent_append_call append; /* cache: e4m3 */
  uint8_t* scales;
  int64_t block_rows;
} latent_append8_call;
int launch_latent_append8(void* stream, const latent_append8_call* call);

/* Attention as launch_latent_attention over such a cache; its workspace is as large as that one's. Held values are taken as they are (in the type of q, which holds them exactly
 * where they are finite and normal numbers there; for half: scales up to 2^22). In calls that are large if requests are as long as the table, bfloat16 queries are split into
 * two numbers of 8 bits, which leaves out what is below 2^-21.8 of a row's greatest (of 2^-118 where that is less), and scores of rows whose scale is less than 2^-62 of another's of
 * their 64 rows may count as zero: results have other bits than under a narrower table. NaN among the numbers of rows that are seen is not looked for. Scales that are NaN make what
 * sees their rows NaN, and leave alone what does not. */
typedef struct {
  latent_attention_call attention; /* cache: e4m3 */
  const uint8_t* scales;
  int64_t block_rows;
} latent_attention8_call;
int launch_latent_attention8(void* stream, const latent_attention8_call* call);

/* Attention in expanded form: keys are [k | k_rope], 128 features per head and 64 shared by all heads; values 128
 * per head. Request b owns keys cu_seqlens_k[b] .. ; causal: token j of n sees the first K - n + j + 1 of its K keys,
 * otherwise all. A request's values have to be finite (those of keys that a token does not see are multiplied by zero);
 * others are never multiplied. scale: as above. Strides are multiples of 8, addresses of q, k, v, k_rope and out of 16 bytes. */
typedef struct {
  int32_t type, causal;
  const void *q, *k, *v, *k_rope; /* [T, heads, 192], [S, heads, 128], [S, heads, 128], [S, 64] */
  const int32_t *cu_seqlens_q, *cu_seqlens_k;
  void* out;  /* [T, heads, 128], contiguous */
  float* lse; /* [T, heads] or NULL */
  void* workspace;
  int32_t* status;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, rope_token; /* strides */
  int64_t batches, tokens, keys, heads;
  double scale;
} latent_prefill_call;
/* Bytes of `workspace` (32-byte aligned; none: NULL will do) for a call of these batches, tokens, keys and heads on the current device; as above. */
int workspace_size_latent_prefill(uint64_t* bytes, const latent_prefill_call* call);
int launch_latent_prefill(void* stream, const latent_prefill_call* call);

#ifdef __cplusplus
}
#endif
#endif /* ASCENDFLOW_B200_LATENT_H_ */
