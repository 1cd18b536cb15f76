/*
 * Serving operators between a decoder's matrix products (libtgm_mi355x.so): rotary positions, a
 * quantised paged key/value cache (write, read, attention over it, attention of a batch that
 * shares a prefix), token sampling and log probabilities.
 *
 * The reference has no model code; these are what a serving loop around its packed matmul
 * (alexandreteles/tinygrad-dx12 src/tinygrad_dx12/codegen/decomp/dx12.py:108-112) needs next
 * to the products.
 *
 * A cache holds pages of page_size positions.  For keys and for values alike:
 *   codes   [pages, kv_heads, page_size, head_dim]      fp8_e4m3 one a byte, fp4_e2m1 two a byte
 *                                                       (lower nibble first)
 *   scales  [pages, kv_heads, head_dim / 32, page_size] E8M0: a power of two per 32 values of a
 *                                                       head, its exponent plus 127
 * Row b of a page table (int32, row stride ld_table) names the pages of sequence b: position p
 * lies in page table[b, p / page_size], slot p % page_size.  Kernels check every table entry
 * against the page count: a position whose entry names no page, or that lies outside the table,
 * is not stored, reads as zeros and is not attended to.
 *
 * Strides count elements; the innermost dimension of every tensor is contiguous.  Types are
 * F32, F16 or BF16 (enum tgm_dtype).  Every function returns TGM_OK or a negative tgm_status
 * (message in tgm_last_error()); none allocates memory or issues a memset.
 */
#ifndef TGM_SERVING_H
#define TGM_SERVING_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum tgm_kv_format { TGM_KV_FP8_E4M3 = 0, TGM_KV_FP4_E2M1 = 1 };
enum tgm_rotary_layout { TGM_ROTARY_HALF = 0, TGM_ROTARY_INTERLEAVED = 1 };

/* head_dim is 64 or 128, page_size a power of two from 16 to 1024; the four stores 16-byte aligned. */
typedef struct tgm_kv_cache {
  void* k_data;
  void* k_scales;
  void* v_data;
  void* v_scales;
  int64_t pages;
  int64_t kv_heads;
  int64_t head_dim;
  int64_t page_size;
  int64_t k_format; /* tgm_kv_format */
  int64_t v_format;
} tgm_kv_cache;

/* Rotated pairs of a head: freq (device, float64 [rotary_dim / 2]) in radians per position; the
 * rotated values are multiplied by gain.  Pair i is (i, i + rotary_dim / 2) in the half layout
 * and (2 i, 2 i + 1) in the interleaved one; values from rotary_dim on stay as they are. */
typedef struct tgm_rotary {
  const double* freq;
  double gain;
  int64_t rotary_dim; /* even, at most head_dim */
  int64_t layout;     /* tgm_rotary_layout */
} tgm_rotary;

/* The layout of a tensor [batch, tokens, heads, head_dim]; its address goes beside it. */
typedef struct tgm_heads {
  int64_t stride_b, stride_t, stride_h;
  int64_t heads;
  int64_t dtype;
} tgm_heads;

/* out = x rotated, token t of sequence b at position start[b] + t.  Angles, sines and products
 * are computed in 64 bits and rounded once to 32 and once to the output's type.  out may be x;
 * any other memory that the two share, or that elements of out share, is a race. */
int tgm_rotate(const tgm_rotary* rotary, const tgm_heads* x, const void* x_data, const tgm_heads* out, void* out_data,
               const int32_t* start, int64_t batch, int64_t tokens, int64_t head_dim, void* stream);

/* The cache write of new tokens: k (rotated by `rotary` unless that is NULL) and v are quantised
 * to the cache's formats at positions start[b] + t, in blocks of 32 values: the scale is
 * 2^(floor(log2 max|x|) - e), e the exponent of the format's largest value (8 for fp8_e4m3, 2 for
 * fp4_e2m1), at least 2^-127 and 2^0 for a block of zeros; codes round to the nearest, ties to
 * even, and saturate.  NaN is stored as 0; infinities as the largest finite value.
 * q (may be NULL) is rotated into q_out.  seen (may be NULL) is the layout of k_seen and v_seen,
 * which receive what the cache now holds for the new tokens.  All of q, k and v have k's type. */
int tgm_kv_append(const tgm_kv_cache* cache, const tgm_rotary* rotary, const tgm_heads* q, const void* q_data,
                  const tgm_heads* q_out, void* q_out_data, const tgm_heads* k, const void* k_data, const tgm_heads* v,
                  const void* v_data, const tgm_heads* seen, void* k_seen, void* v_seen, const int32_t* table,
                  int64_t ld_table, int64_t table_cols, const int32_t* start, int64_t batch, int64_t tokens,
                  void* stream);

/* Positions first[b] .. first[b] + count - 1 of every sequence, [batch, count, kv_heads, head_dim]
 * contiguous of type dtype (rounded once from the exact value), 16-byte aligned. */
int tgm_kv_read(const tgm_kv_cache* cache, const int32_t* table, int64_t ld_table, int64_t table_cols,
                const int32_t* first, int64_t batch, int64_t count, void* k_out, void* v_out, int dtype, void* stream);

/* Grouped-query attention of `tokens` new tokens per sequence over the cache.  lengths[b] counts
 * the cached positions of sequence b, the new tokens among them: token t sees the positions up to
 * lengths[b] - tokens + t; one that sees none gives zeros, one with a NaN among its scores or with
 * one of +infinity (a query that is not finite, a product beyond 32 bits) gives NaN.
 * out [batch, tokens, heads, head_dim] contiguous, of q's type, and q itself or memory that the two
 * do not share; scores are multiplied by scale, softmax and sums are held in 32 bits.
 * shared > 0 (a multiple of page_size): positions below it lie in the same pages for every
 * sequence (those of row 0 of the table) and are read once for the whole batch.
 * workspace: tgm_kv_attend_workspace() bytes, 16-byte aligned. */
int64_t tgm_kv_attend_workspace(const tgm_kv_cache* cache, int64_t q_dtype, int64_t heads, int64_t batch, int64_t tokens,
                                int64_t table_cols, int64_t shared);
int tgm_kv_attend(const tgm_kv_cache* cache, const tgm_heads* q, const void* q_data, const int32_t* table,
                  int64_t ld_table, int64_t table_cols, const int32_t* lengths, int64_t batch, int64_t tokens,
                  int64_t shared, double scale, void* workspace, int64_t workspace_bytes, void* out, void* stream);

/* One token per row of logits [rows, vocab] (row stride ld) by inversion: with
 * w_i = exp((logit_i - max) / temperature) in 64 bits, the kept set is cut to the top_k largest
 * (0 and less: all), then to the shortest descending run whose mass reaches top_p of what is
 * left (1 and more: all; the first always stays), then to w >= min_p; ties rank by index.  The
 * token is the first kept index whose running sum, in the vocabulary's order, exceeds u times
 * the kept mass, u in [0, 1).  temperature <= 0 takes the first maximum.  -inf and NaN logits are
 * never taken; a row that holds nothing else gives 0.
 * Parameters are per-row arrays on the device (float32; top_k int32); top_k, top_p and min_p may be
 * NULL (no cut).  workspace: tgm_sample_workspace() bytes, 16-byte aligned (NULL when 0). */
int64_t tgm_sample_workspace(int64_t rows, int64_t vocab, int64_t dtype);
int tgm_sample(const void* logits, int64_t dtype, int64_t rows, int64_t vocab, int64_t ld, const float* u,
               const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, int32_t* tokens,
               void* workspace, int64_t workspace_bytes, void* stream);

/* Log probabilities of one given token per row of logits [rows, vocab] (row stride ld), natural logarithms in 32 bits:
 *   logprobs[r]  of tokens[r];  ranks[r]  how many tokens come before it by falling logit, equal ones by index
 *   entropy[r]   of the row's distribution;  top_ids, top_logprobs [rows, top]  the likeliest tokens, the first first
 * top is 0 to 64 (top_ids and top_logprobs may be NULL for 0), at most vocab.  A token outside the vocabulary names none: its
 * logprob is 0 and its rank -1.  A row with a NaN or +infinity, or of -infinities alone, has NaN probabilities and
 * entropy; NaN ranks behind everything.
 * workspace: tgm_log_probs_workspace() bytes, 16-byte aligned (NULL when 0). */
int64_t tgm_log_probs_workspace(int64_t rows, int64_t vocab, int64_t dtype, int64_t top);
int tgm_log_probs(const void* logits, int64_t dtype, int64_t rows, int64_t vocab, int64_t ld, const int32_t* tokens,
                  int64_t top, float* logprobs, int32_t* ranks, float* entropy, int32_t* top_ids, float* top_logprobs,
                  void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TGM_SERVING_H */
