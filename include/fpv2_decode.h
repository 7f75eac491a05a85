/*
 * fpv2_decode.h — operators of a decode step (one new token per sequence
 * after the FPV2 prefill), exported by libfpv2_hip.so.
 *
 * The reference ends where the prompt is prefilled (fpv2/generate.py:97-130
 * hands the caches to mlx-lm, an external dependency, whose models decode
 * over the cache with 4-bit weights and sample the tokens).  These are the
 * gfx950 operators of that step: attention of single tokens over a paged or
 * contiguous cache, norms and rotation with the cache write, products with
 * 4-bit weights, and sampling.
 *
 * Conventions as in fpv2.h: device pointers, element strides, a hipStream_t
 * passed as void*, work enqueued on that stream on the current device, no
 * allocation, no host synchronisation, FPV2_OK or a negative fpv2_status with
 * fpv2_last_error() set.  Lengths, page ids, positions and slots are read on
 * the device; the ones out of range are clipped or skipped as stated.
 * Outputs are apart from one another and from all inputs, and no two of an output's
 * rows share memory (not checked here); only the queries' result may be the queries
 * themselves (`out` of the attention, `q_out` in the rows of `qkv`), element for element.
 */
#ifndef FPV2_DECODE_H_
#define FPV2_DECODE_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of one new token per sequence over a cache in pages. */
typedef struct fpv2_decode_params {
  int64_t batch;
  int64_t query_heads;
  int64_t kv_heads;      /* divides query_heads                               */
  int64_t head_dim;      /* 64, 96, 128 or 256                                */
  int64_t pages;         /* pages of k_pages / v_pages                        */
  int64_t page_size;     /* tokens of a page                                  */
  int64_t table_width;   /* pages of a sequence (columns of page_table)       */
  int64_t table_stride;  /* elements between its rows                         */
  int64_t length;        /* every sequence's length where `lengths` is NULL   */
  int64_t window_tokens; /* keys at the end that are visible; 0: all          */
  int64_t sink_tokens;   /* keys at the start that stay visible               */
  double scale;
  int64_t q_batch_stride, q_head_stride;
  int64_t k_page_stride, k_head_stride, k_row_stride;
  int64_t v_page_stride, v_head_stride, v_row_stride;
  int64_t o_batch_stride, o_head_stride;
} fpv2_decode_params;

/*
 * out[b][h] = sum_t softmax_t(scale q[b][h].k_t) v_t over the visible keys t of
 * sequence b: t < length, and t < sink_tokens or t >= length - window_tokens
 * where a window is given.  Token t of sequence b is row t % page_size of page
 * page_table[b][t / page_size] (int32; without page_table of page b).  Page ids
 * are clipped to [0, pages) and lengths to [0, table_width * page_size]; a
 * sequence of length 0 gives zeros.  Rows behind a length are not used.
 * The weights are rounded to the inputs' type for their product with v (f16: relative
 * to 2^-15 of the greatest of 32 keys), their sum is not; everything else is float32.
 * bf16 or f16; the strides of q, k and v multiples of 8 and their pointers
 * 16-byte aligned.  workspace: fpv2_decode_attention_workspace_bytes bytes for
 * the current device (0: none), 16-byte aligned, not kept between calls; calls
 * that share one on different streams race.  Deterministic.
 */
int64_t fpv2_decode_attention_workspace_bytes(const fpv2_decode_params* params);
int fpv2_decode_attention(const void* q, const void* k_pages, const void* v_pages,
                          const int32_t* page_table, const int32_t* lengths, void* out, int dtype,
                          const fpv2_decode_params* params, void* workspace,
                          int64_t workspace_bytes, void* stream);

/* Norms and rotation of fused projection rows, K and V into pages. */
typedef struct fpv2_rope_pages_params {
  int64_t tokens;
  int64_t query_heads;
  int64_t kv_heads;
  int64_t head_dim;       /* a multiple of 16, at most 512                     */
  int64_t rotary_half;    /* columns of cos / sin: a multiple of 8, at most
                             head_dim / 2                                      */
  int64_t table_rows;     /* positions that cos / sin hold                     */
  int64_t interleaved;    /* 0: pairs (j, j + rotary_half); 1: (2j, 2j + 1)    */
  int64_t pages, page_size;
  int64_t position_bytes; /* 4 or 8: type of positions[t]; 0: first_position + t */
  int64_t slot_bytes;     /* 4 or 8: type of slots[t]; 0: first_slot + t       */
  int64_t first_position, first_slot;
  int64_t qkv_row_stride;
  int64_t q_token_stride, q_head_stride;
  int64_t k_page_stride, k_head_stride, k_row_stride;
  int64_t v_page_stride, v_head_stride, v_row_stride;
  double eps;
} fpv2_rope_pages_params;

/*
 * Per-head RMSNorm (skipped for a NULL weight) and rotary embedding of the
 * query and key heads of fused projection rows qkv[t] = [q | k | v heads]:
 *   n = x rsqrt(mean(x^2) + eps) weight
 *   (n_a, n_b) -> (n_a cos - n_b sin, n_b cos + n_a sin), the pair's angle
 *   from row positions[t] (clipped to the table) of cos / sin
 * in float32, rounded once.  Query heads go to q_out, key heads and the
 * unchanged value heads to row slots[t] % page_size of page slots[t] / page_size;
 * a token whose slot lies outside the pages is padding: its K and V are not
 * written.  Slots must be distinct.  Dimensions from 2 rotary_half on are not
 * rotated.  bf16 or f16; cos / sin float32 [table_rows, rotary_half]
 * contiguous; strides multiples of 8 and pointers 16-byte aligned
 * (positions / slots by their type).
 * Counterpart of mlx-lm's q_norm / k_norm, nn.RoPE and cache update.
 */
int fpv2_rope_to_pages(const void* qkv, const void* q_weight, const void* k_weight,
                       const float* cos, const float* sin, const void* positions,
                       const void* slots, void* q_out, void* k_pages, void* v_pages, int dtype,
                       const fpv2_rope_pages_params* params, void* stream);

/*
 * out[m][n] = sum_k x[m][k] w[n][k] with 4-bit weights in groups along k:
 *   w[n][k] = scales[n][k / group] q[n][k] + biases[n][k / group]
 * q[n][k] is bits 4 (k % 8) .. + 3 of 32-bit word packed[n][k / 8] (the layout of
 * MLX's affine quantization).  group 32, 64 or 128 divides cols.  x, scales
 * and biases share dtype (bf16 or f16), out has it too or float32 (out_dtype);
 * products and sums in float32.  Row strides in elements (packed: in words);
 * x_row_stride a multiple of 8, packed_row_stride of 4; x and packed 16-byte
 * aligned; scales / biases rows contiguous, scale_row_stride elements apart.
 */
int fpv2_quantized_linear(const void* x, const void* packed, const void* scales,
                          const void* biases, void* out, int dtype, int out_dtype, int64_t rows,
                          int64_t out_cols, int64_t cols, int64_t group, int64_t x_row_stride,
                          int64_t packed_row_stride, int64_t scale_row_stride,
                          int64_t out_row_stride, void* stream);

/* Largest vocabulary of fpv2_sample_tokens (its sums are integers of 64 bits). */
#define FPV2_MAX_VOCAB (1 << 19)

/* Sampling.  A NULL array takes the value beside it for every row. */
typedef struct fpv2_sample_params {
  int64_t batch;
  int64_t vocab;
  int64_t logits_stride;    /* elements between rows                          */
  const float* temperatures;
  const int32_t* top_ks;
  const float* top_ps;
  const float* min_ps;
  double temperature;       /* 0 or less: the greatest logit; at most 1e30     */
  int64_t top_k;            /* 0 or less: no limit                            */
  double top_p;             /* 1 or more: no limit                            */
  double min_p;
} fpv2_sample_params;

/*
 * One token per row of logits [batch, vocab] (float32, bf16 or f16) by the row's
 * number uniforms[b] in [0, 1):
 *   weights w_i = exp((logit_i - max) / temperature), tokens ordered by logit,
 *   equal ones by index, and kept: the first top_k; of these the ones whose
 *   weight before them is less than top_p of the weight of all of these; of
 *   these the ones with w_i >= min_p (clipped to 1).  The first is always kept.
 *   token = the first one in index order whose running kept weight exceeds
 *   uniforms[b] (clipped to [0, 1]) times all kept weight (the last kept one of
 *   any weight where none does).
 * Weights are computed in float64 and rounded to 2^-44, sums are exact, so the
 * result does not depend on any order.  A NaN logit counts as -inf; a row of
 * nothing but -inf gives token -1.  logprobs (NULL: not written): log of the
 * token's share of the kept weight, 0 for a greedy row, -inf for token -1.
 * workspace: fpv2_sample_tokens_workspace_bytes bytes for the current device (0:
 * none), 16-byte aligned, not kept between calls; calls that share one on
 * different streams race.
 */
int64_t fpv2_sample_tokens_workspace_bytes(const fpv2_sample_params* params);
int fpv2_sample_tokens(const void* logits, const float* uniforms, int dtype,
                       const fpv2_sample_params* params, int64_t* tokens, float* logprobs,
                       void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* FPV2_DECODE_H_ */
