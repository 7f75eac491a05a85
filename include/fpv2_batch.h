/*
 * fpv2_batch.h — operators of serving a batch after the FPV2 prefill, exported
 * by libfpv2_hip.so: attention of sequences that share a prompt, a cache of
 * 8-bit codes with its writer, its reader and its attention, and the log
 * probabilities of tokens.
 *
 * The reference ends where one prompt is prefilled (fpv2/generate.py:97-130).
 *
 * Conventions as in fpv2_decode.h.
 */
#ifndef FPV2_BATCH_H_
#define FPV2_BATCH_H_

#include <stdint.h>

#include "fpv2_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of one new token per sequence over a shared prefix and its own keys. */
typedef struct fpv2_shared_prefix_params {
  fpv2_decode_params own;      /* the sequences' own keys; no window, no sinks   */
  int64_t prefix_pages;        /* pages of prefix_k / prefix_v                   */
  int64_t prefix_page_size;
  int64_t prefix_table_width;  /* pages of the prefix                            */
  int64_t prefix_length;       /* where `prefix_length` is NULL                  */
  int64_t pk_page_stride, pk_head_stride, pk_row_stride;
  int64_t pv_page_stride, pv_head_stride, pv_row_stride;
} fpv2_shared_prefix_params;

/*
 * out[b][h] = sum_t softmax_t(scale q[b][h].k_t) v_t over the keys t of the prefix,
 * which all sequences see, and of sequence b's own cache.  Token t of the prefix is row
 * t % prefix_page_size of page prefix_table[t / prefix_page_size] (int32; without
 * prefix_table of page 0); a sequence's own tokens as in fpv2_decode_attention.
 * Page ids and lengths are clipped as there; a sequence with no keys at all gives
 * zeros.  Weights are rounded to the inputs' type for their product with v, their sum is
 * not (f16: weights down to 2^-19 of the greatest of their 32 keys to 11 bits, smaller ones
 * to 2^-30 of it).  At most 2^24 - 1 query heads of the batch.  The prefix's
 * strides are multiples of 8 and its pointers 16-byte aligned; its pages may be of
 * the sequences' own pool.  workspace: fpv2_shared_prefix_attention_workspace_bytes
 * bytes, 16-byte aligned, not kept between calls; calls that share one on
 * different streams race.  Deterministic.
 */
int64_t fpv2_shared_prefix_attention_workspace_bytes(const fpv2_shared_prefix_params* params);
int fpv2_shared_prefix_attention(const void* q, const void* prefix_k, const void* prefix_v,
                                 const int32_t* prefix_table, const int32_t* prefix_length,
                                 const void* k_pages, const void* v_pages,
                                 const int32_t* page_table, const int32_t* lengths, void* out,
                                 int dtype, const fpv2_shared_prefix_params* params,
                                 void* workspace, int64_t workspace_bytes, void* stream);

/* A cache of 8-bit codes in pages: k_codes / v_codes [pages][kv_heads][page_size][head_dim]
 * int8 and one float32 scale for each row of a head [pages][kv_heads][page_size]. */
typedef struct fpv2_code_pages {
  int64_t kv_heads;
  int64_t head_dim;       /* 64, 96, 128 or 256                               */
  int64_t pages, page_size;
  int64_t k_page_stride, k_head_stride, k_row_stride;     /* codes, in bytes  */
  int64_t v_page_stride, v_head_stride, v_row_stride;
  int64_t ks_page_stride, ks_head_stride, ks_row_stride;  /* scales, elements */
  int64_t vs_page_stride, vs_head_stride, vs_row_stride;
} fpv2_code_pages;

/* Writing tokens into a cache of codes. */
typedef struct fpv2_quantize_params {
  fpv2_code_pages cache;
  int64_t tokens;
  int64_t slot_bytes;     /* 4 or 8: type of slots[t]; 0: first_slot + t      */
  int64_t first_slot;
  int64_t k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride;
} fpv2_quantize_params;

/*
 * A token's key (value) of a KV head, x[0 .. head_dim), becomes with a = max |x|
 *   codes[j] = 127 x[j] / a, rounded to the nearest whole number, of two the even one
 *   scale = a / 127 in float32
 * (all zeros for a = 0; codes 0 and scale NaN where x holds an infinity or NaN), in row
 * slots[t] % page_size of page slots[t] / page_size.  A token whose slot lies outside
 * the pages is padding and not written.  Slots must be distinct.  bf16 or f16; k and v
 * with strides that are multiples of 8 and 16-byte aligned, the codes' strides multiples of
 * 16 and their pointers 16-byte aligned.
 */
int fpv2_quantize_to_pages(const void* k, const void* v, const void* slots, void* k_codes,
                           float* k_scales, void* v_codes, float* v_scales, int dtype,
                           const fpv2_quantize_params* params, void* stream);

/* Reading a cache of codes back. */
typedef struct fpv2_dequantize_params {
  fpv2_code_pages cache;
  int64_t batch;
  int64_t table_width, table_stride;
  int64_t length;         /* every sequence's length where `lengths` is NULL  */
  int64_t tokens;         /* rows of a sequence's result                      */
  int64_t zero_rest;      /* 1: rows behind a length are zeros; 0: not written */
  int64_t k_batch_stride, k_head_stride, k_row_stride;  /* results            */
  int64_t v_batch_stride, v_head_stride, v_row_stride;
} fpv2_dequantize_params;

/*
 * k_out[b][h][t][j] = codes[j] scale of token t of sequence b, t < min(length, tokens),
 * rounded once to bf16 or f16; likewise v_out.  Tokens, page ids and lengths as in
 * fpv2_decode_attention.  The results' strides are multiples of 8, their pointers
 * 16-byte aligned; batch * kv_heads is at most 65535.
 */
int fpv2_dequantize_pages(const void* k_codes, const float* k_scales, const void* v_codes,
                          const float* v_scales, const int32_t* page_table,
                          const int32_t* lengths, void* k_out, void* v_out, int dtype,
                          const fpv2_dequantize_params* params, void* stream);

/* Attention over a cache of codes. */
typedef struct fpv2_quantized_decode_params {
  fpv2_decode_params attention;  /* strides of k and v in bytes of codes      */
  int64_t ks_page_stride, ks_head_stride, ks_row_stride;
  int64_t vs_page_stride, vs_head_stride, vs_row_stride;
} fpv2_quantized_decode_params;

/*
 * fpv2_decode_attention over the values codes[j] scale.  The codes are whole numbers and
 * exact in the products; the queries are multiplied as float16 of 11 bits, relative to a
 * power of two by their greatest, a key's scale in float32 with its score; a value's scale
 * with its weight, which is then rounded to float16, relative to 2^-15 of the greatest such
 * product of 32 keys.  Products below 2^-111, where the greatest score's weight is 1, may
 * count as 0.  The codes' strides are multiples of 16, their pointers 16-byte aligned.
 */
int64_t fpv2_quantized_decode_attention_workspace_bytes(const fpv2_quantized_decode_params* params);
int fpv2_quantized_decode_attention(const void* q, const void* k_codes, const float* k_scales,
                                    const void* v_codes, const float* v_scales,
                                    const int32_t* page_table, const int32_t* lengths, void* out,
                                    int dtype, const fpv2_quantized_decode_params* params,
                                    void* workspace, int64_t workspace_bytes, void* stream);

/* Most alternatives of fpv2_token_logprobs. */
#define FPV2_MAX_TOP 32

typedef struct fpv2_logprobs_params {
  int64_t rows;
  int64_t vocab;            /* 1 .. FPV2_MAX_VOCAB                            */
  int64_t logits_stride;    /* elements between rows                          */
  int64_t token_bytes;      /* 4 or 8: type of tokens                         */
  int64_t top;              /* alternatives of a row: 0 .. FPV2_MAX_TOP       */
} fpv2_logprobs_params;

/*
 * For each row of logits [rows, vocab] (float32, bf16 or f16), with p = softmax(row):
 *   logprobs[r] = log p[tokens[r]], -inf for a token outside the vocabulary
 *   entropy[r] = -sum p log p, in nats
 *   top_tokens[r][i], top_logprobs[r][i]: the i-th greatest logit's token, of equal ones
 *   the first, and log p of it; -1 and -inf where there is none above -inf
 * A NaN logit counts as -inf, magnitudes beyond 2^126 as 2^126 (in p; the alternatives are in the order of
 * the logits as given); a row of nothing but -inf has logprob -inf and entropy 0.  float32 arithmetic.  workspace:
 * fpv2_token_logprobs_workspace_bytes bytes for the current device (0: none), 16-byte
 * aligned, not kept between calls; calls that share one on different streams race.
 */
int64_t fpv2_token_logprobs_workspace_bytes(const fpv2_logprobs_params* params);
int fpv2_token_logprobs(const void* logits, const void* tokens, int dtype,
                        const fpv2_logprobs_params* params, float* logprobs, float* entropy,
                        int64_t* top_tokens, float* top_logprobs, void* workspace,
                        int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FPV2_BATCH_H_ */
