/*
 * C ABI of latent attention in libl20_paged_decode_hip.so: attention whose keys and values come from
 * one latent vector a token, shared by all heads, with a rotary key part beside it.  Three operators:
 *
 *   l20_pd_latent_rope_and_cache  the cache producer: norm of the latent, RoPE of the key and query
 *                                 parts, and the write of the rows into a paged cache
 *   l20_pd_paged_latent           decode and verification steps over that cache (absorbed form)
 *   l20_pd_latent_prompt          causal attention of prompts over expanded keys and values
 *
 * Plain pointers, sizes and strides (in elements; the last dimension is contiguous everywhere); a HIP
 * stream is passed as `void *`.  Return codes, dtype codes and l20_pd_last_error() are those of
 * l20_paged_decode.h.  The reference has no latent attention: these have no counterpart there.
 */
#ifndef L20_LATENT_ATTENTION_H_
#define L20_LATENT_ATTENTION_H_

#include <stdint.h>

#include "l20_paged_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The cache producer over num_tokens new tokens.
 *
 *   query          [num_tokens, num_heads, 64] dtype: the rotary part of the query heads (NULL: skipped)
 *   query_out      same shape: where the rotated parts go (may be `query` itself)
 *   latent         [num_tokens, rank] dtype; latent_out: same shape, the normalised latent (may be
 *                  `latent` itself)
 *   key            [num_tokens, 64] dtype; key_out: same shape, the rotated key part (may be `key`)
 *   positions      [num_tokens] int64
 *   cos_sin_cache  [max_position, 64] cs_dtype: 32 cosines, then 32 sines
 *   norm_weight    [rank] dtype, or NULL: the latent is stored as it is
 *   slot_mapping   [num_tokens] int64: page slot / page_size, row slot % page_size; < 0, or beyond the
 *                  cache: the token is not stored (its outputs are written all the same).  The slots of a
 *                  call differ: one that is named twice holds pieces of both rows
 *   cache          [num_pages, page_size, rank + 64] cache_dtype (e4m3fn, or the model dtype)
 *
 *   latent_out = latent * rsqrt(mean(latent^2) + eps) * weight          (fp32, rounded once to dtype)
 *   part_out   = x cos + (x_pair sin) sign                              (fp32, rounded once to dtype),
 *                pairs (d, d + 32) with is_neox, (2 i, 2 i + 1) without
 *   cache row  = [latent_out | key_out], in an fp8 cache RNE_e4m3fn(clamp(. / cache_scale, +-448)),
 *                NaN for NaN
 *
 * An output that is not its input (address and strides) must share no bytes with the inputs: the call refuses it.
 */
typedef struct l20_pd_latent_write_args {
  const void *query;
  int64_t q_stride_token, q_stride_head;
  void *query_out;
  int64_t qo_stride_token, qo_stride_head;
  int32_t num_heads;
  const void *latent;
  int64_t l_stride_token;
  void *latent_out;
  int64_t lo_stride_token;
  const void *key;
  int64_t k_stride_token;
  void *key_out;
  int64_t ko_stride_token;
  int32_t dtype; /* L20_PD_BF16 or L20_PD_FP16 */

  const int64_t *positions;
  const void *cos_sin_cache;
  int64_t cs_stride_position;
  int64_t max_position; /* rows of cos_sin_cache: positions outside [0, max_position) are clamped to it */
  int32_t cs_dtype; /* L20_PD_BF16, L20_PD_FP16 or L20_PD_FP32 */
  int32_t is_neox;
  const void *norm_weight;
  float norm_eps;

  const int64_t *slot_mapping;
  void *cache;
  int64_t c_stride_page, c_stride_token;
  int64_t num_pages;
  int32_t page_size;
  int32_t cache_dtype; /* enum l20_pd_kv_dtype */
  float cache_scale;

  int32_t num_tokens, rank, rope_dim;
} l20_pd_latent_write_args;

int32_t l20_pd_latent_write_check(const l20_pd_latent_write_args *args);
int32_t l20_pd_latent_rope_and_cache(const l20_pd_latent_write_args *args, void *stream);

/*
 * One decode (q_len = 1) or verification step over a paged latent cache.
 *
 *   query        [batch*q_len, num_heads, rank + 64] dtype: the absorbed query and its rotated part
 *   cache        [num_pages, page_size, rank + 64] (e4m3fn codes, read as code * cache_scale, or dtype);
 *                page_size a multiple of 16 through 4096, tokens of a page contiguous above 16
 *                (stride_page = page_size * stride_token)
 *   block_table  [batch, table_pages] int32; seq_lens [batch] int32, the q_len new tokens included
 *   output       [batch*q_len, num_heads, rank] dtype; lse [batch*q_len, num_heads] fp32 natural log or NULL.  An
 *                output that shares bytes with the query is refused by the call (interleaved views do not)
 *
 * Row b*q_len+i sees tokens 0 .. seq_lens[b]-q_len+i:
 *   s_t = softmax_scale q . row_t,  out = sum_t softmax(s)_t row_t[0 .. rank)
 * A row that sees nothing gives zeros and an LSE of -inf.  Tokens beyond the table's width, or on a
 * page outside [0, num_pages), or beyond max_seq_len, are masked for every row.  A value that is not finite
 * reaches only the rows that see its token.
 *
 * The work (tiles of tokens of all sequences) is split evenly over the CUs; what a workgroup has of a
 * sequence that others share goes to `workspace` (l20_pd_paged_latent_workspace bytes, 16-byte aligned)
 * and a second kernel joins the parts.  The workspace's contents before and after do not matter; calls
 * that may overlap each need their own.  max_seq_len sizes the grid and the workspace.
 */
typedef struct l20_pd_latent_args {
  const void *query;
  int64_t q_stride_row, q_stride_head;
  int32_t dtype;
  const void *cache;
  int64_t c_stride_page, c_stride_token;
  int64_t num_pages;
  int32_t page_size;
  int32_t cache_dtype;
  float cache_scale;
  const int32_t *block_table;
  int64_t bt_stride_row;
  int32_t table_pages;
  const int32_t *seq_lens;
  void *output;
  int64_t o_stride_row, o_stride_head;
  float *lse;
  int64_t lse_stride_row, lse_stride_head;
  void *workspace;
  int64_t workspace_bytes;
  float softmax_scale;
  int32_t batch, q_len, num_heads, rank, rope_dim, max_seq_len;
} l20_pd_latent_args;

int32_t l20_pd_paged_latent_check(const l20_pd_latent_args *args);
/* Workspace bytes on a device of cu_count compute units (0: the current device's), enough for every call of up
 * to `batch` sequences and up to `max_seq_len` with this q_len, num_heads, rank and cache_dtype; reads only
 * those.  0 where none of them needs a workspace. */
int64_t l20_pd_paged_latent_workspace(const l20_pd_latent_args *args, int32_t cu_count);
int32_t l20_pd_paged_latent(const l20_pd_latent_args *args, void *stream);

/*
 * Attention of packed prompts over expanded keys and values (128 dims a head, 64 shared rotary dims).
 *
 *   query      [total_q, num_heads, 192] dtype; output [total_q, num_heads, 128] dtype; an output that
 *              shares bytes with the query, the keys or the values is refused by the call
 *   key, value [total_k, num_heads, 128] dtype; key_rope [total_k, 64] dtype, shared by the heads
 *   cu_q, cu_k [batch + 1] int32: sequence b has query rows cu_q[b] .. cu_q[b+1] and keys
 *              cu_k[b] .. cu_k[b+1]; offsets are clamped to the tensors
 *   lse        [total_q, num_heads] fp32 natural log, or NULL
 *
 * s_ij = softmax_scale (q_i[0..128) . key_j + q_i[128..192) . key_rope_j); with causal != 0 query i of
 * n sees keys j <= i + (keys - n).  A row that sees nothing gives zeros and an LSE of -inf.  Query rows
 * outside cu_q's ranges, or beyond max_q_len of their sequence, keep what they held.
 *
 * Calls of few (row block, head) units and many keys split the keys over the CUs as l20_pd_paged_latent
 * does, with `workspace` (l20_pd_latent_prompt_workspace bytes, 16-byte aligned, one for each of the calls
 * that may overlap); with workspace = NULL they do not.
 */
typedef struct l20_pd_latent_prompt_args {
  const void *query;
  int64_t q_stride_token, q_stride_head;
  const void *key;
  int64_t k_stride_token, k_stride_head;
  const void *key_rope;
  int64_t kr_stride_token;
  const void *value;
  int64_t v_stride_token, v_stride_head;
  int32_t dtype;
  const int32_t *cu_q, *cu_k;
  void *output;
  int64_t o_stride_token, o_stride_head;
  float *lse;
  int64_t lse_stride_token, lse_stride_head;
  float softmax_scale;
  int32_t causal;
  int64_t total_q, total_k;
  int32_t batch, num_heads, max_q_len, head_dim, rope_dim, value_dim;
  void *workspace;
  int64_t workspace_bytes;
} l20_pd_latent_prompt_args;

int32_t l20_pd_latent_prompt_check(const l20_pd_latent_prompt_args *args);
/* Workspace bytes of a call on a device of cu_count compute units (0: the current device's); reads only
 * total_q, total_k, batch, num_heads and max_q_len.  0 where the keys are not split. */
int64_t l20_pd_latent_prompt_workspace(const l20_pd_latent_prompt_args *args, int32_t cu_count);
int32_t l20_pd_latent_prompt(const l20_pd_latent_prompt_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* L20_LATENT_ATTENTION_H_ */
