/*
 * bz_paged_cache.h - C ABI of libbz_gqa_decode.so for a KV cache held in pages: rotary positions, storing a step's new
 * keys and values, reading them back, and the attention of the new tokens of every row over its pages.
 *
 * Conventions are those of bz_gqa_decode.h (device pointers on the current device, strides in elements unless stated,
 * no allocation, no host decision from device data, bz_status return values, nothing launched when a check fails).
 *
 * Rows and tokens. A batch has `batch` rows and `tokens` new tokens, those of one row behind those of the row before:
 * row b's are q_start[b] .. q_start[b + 1] - 1 (int32 [batch + 1], not decreasing, from 0 to `tokens`; NULL: one token a
 * row, tokens == batch). They are the last positions of a row of seq_lens[b] (int32 [batch]): token n is its position
 * seq_lens[b] - (q_start[b + 1] - n). Tokens of no row (behind q_start[batch], a batch's padding) are neither read nor
 * written. Position p of row b lies in page page_table[b, p / page_size], at place p % page_size. A page number outside
 * [0, pages), and positions below 0 or past the table, hold nothing: what would be stored there is dropped, loads give
 * zeros, and nothing attends them. A page may stand in several rows, or twice in one, and is then read for each; where two
 * tokens of one call are stored at the same place, what that place holds afterwards is undefined (and nothing else is).
 */
#ifndef BZ_PAGED_CACHE_H
#define BZ_PAGED_CACHE_H

#include "bz_gqa_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The cache and the batch's rows. K and V [pages, num_kv_heads, page_size, head_dim], sharing strides, the last dimension
   contiguous: bf16 (bits 16) or e4m3 codes (bits 8) with one scale byte E for each vector of head_dim, which stands for
   2^(E - 127) (10 to 247 as the stores make them; 255: NaN, every value of the vector), in k_scale and v_scale uint8
   [pages, num_kv_heads, page_size], sharing
   strides, the last dimension contiguous. Strides are in bytes; K, V and their strides are multiples of 16, scales and
   theirs of 4. page_size is a power of two from 16 to 1024, head_dim 64 or 128; a page of a head spans less than 2^30 bytes.
   page_table int32 [batch, max_pages], table_stride elements from row to row; max_pages * page_size at most 2^30. */
typedef struct bz_paged_cache {
  void *k, *v;
  int64_t stride_page, stride_h, stride_s;
  void *k_scale, *v_scale;
  int64_t scale_stride_page, scale_stride_h;
  int32_t pages, num_kv_heads, page_size, head_dim, bits;
  const int32_t* page_table;
  int64_t table_stride;
  int32_t batch, max_pages;
  const int32_t* seq_lens;
  const int32_t* q_start;
  int32_t tokens;
} bz_paged_cache;

/* A rotation. Pair i of the first rotary_dim dims of a head (a multiple of 16 up to head_dim) is turned by the angle
   position * inv_freq[i] (float64 [rotary_dim / 2]) and multiplied by `factor`; the pair is dims i and i + rotary_dim / 2, or, if
   interleaved, 2 i and 2 i + 1. The other dims stay. Angles are worked out in 64 bits and reduced to one turn there; cos, sin
   and the products are fp32, rounded once. */
typedef struct bz_rope {
  const double* inv_freq;
  int32_t rotary_dim, interleaved;
  float factor;
} bz_rope;

/* out[n, h] = x[n, h] turned by positions[n] (int32, or int64 with positions_64); inverse: turned back (by -position, divided by
   factor). x, out bf16 [tokens, heads, head_dim], 16-byte aligned with strides of multiples of 8 elements; out may be x itself
   (with its strides), else must not overlap it. */
typedef struct bz_rope_args {
  bz_rope rope;
  const void* x;
  int64_t x_stride_t, x_stride_h;
  void* out;
  int64_t out_stride_t, out_stride_h;
  const void* positions;
  int32_t positions_64, inverse;
  int32_t tokens, heads, head_dim;
} bz_rope_args;
int bz_rope_apply(const bz_rope_args* args, hipStream_t stream);

/* Stores the new tokens' k and v (bf16 [tokens, num_kv_heads, head_dim], aligned as x above) into the pages. With
   rope.inv_freq, k is turned first, and q (bf16 [tokens, num_q_heads, head_dim]) into q_out (which may be q itself), by the token's
   position in its row, or positions[n] if given; with q_norm_weight / k_norm_weight (bf16 [head_dim]) q / k are normed before
   that: x * rsqrt(mean(x^2) + eps) * weight. All of this is fp32, rounded once, to bf16 or into the 8-bit cache: the scale of a vector
   is the smallest power of two, from 2^-117, with max |x| <= 448 scale, its codes are x / scale rounded to the nearest e4m3 value
   (ties to even; a value of 2^128 - 2^123 or more, under the largest scale, becomes 2^128, which reads as an infinity); a vector
   that holds NaN or an infinity gets scale byte 255. Without rope, q must be NULL and the norms too. */
typedef struct bz_paged_store_args {
  bz_paged_cache cache;
  const void *k, *v;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  bz_rope rope;
  const void* q;
  int64_t q_stride_t, q_stride_h;
  void* q_out;
  int64_t q_out_stride_t, q_out_stride_h;
  int32_t num_q_heads;
  const void *q_norm_weight, *k_norm_weight;
  float eps;
  const void* positions;
  int32_t positions_64;
} bz_paged_store_args;
int bz_paged_store(const bz_paged_store_args* args, hipStream_t stream);

/* The bf16 values of positions starts[b] .. starts[b] + count - 1 of each row, into k and v (bf16 [batch, num_kv_heads, count,
   head_dim], sharing strides, aligned as above; they share no memory), exactly as bz_gqa_paged reads them. seq_lens, q_start and
   tokens of the cache are not used: what a page holds behind a row's length comes back too. */
int bz_paged_load(const bz_paged_cache* cache, const int32_t* starts, int32_t count, void* k, void* v, int64_t x_stride_b,
                  int64_t x_stride_h, int64_t x_stride_t, hipStream_t stream);

/* Arguments of bz_gqa_paged. q, out bf16 [tokens, num_q_heads, head_dim], q 16-byte aligned with strides of multiples of 8
   elements; q head h reads kv head h / G, G = num_q_heads / num_kv_heads of 1, 2, 4 or 8. max_tokens (0: unknown) and max_seq_len
   (0: max_pages * page_size): about the most new tokens and positions of a row, right or wrong. They steer the launch: they change
   the order of a result's sums and, for rows of more than 16 / G tokens, whether softmax terms meet V as two bf16 terms or as one
   (below). workspace: bz_paged_workspace_size bytes, 256-byte aligned, zero-filled once; it serves every later call
   of any sizes that needs no more, and two calls that share one must be ordered on one stream. */
typedef struct bz_gqa_paged_args {
  bz_paged_cache cache;
  const void* q;
  int64_t q_stride_t, q_stride_h;
  void* out;
  int64_t out_stride_t, out_stride_h;
  float scale;
  int32_t num_q_heads, max_tokens, max_seq_len;
  void* workspace;
  size_t workspace_bytes;
} bz_gqa_paged_args;

/* Causal attention of the new tokens: out[n, h] = sum_p softmax_p(scale q[n, h] . k[p]) v[p] over the positions p of the token's
   row up to its own. A token that attends nothing, or whose scores are all -inf, yields zeros; what is stored at positions that a
   token does not attend (NaN and infinities among it) does not reach its output. Sums are fp32 (sum |V| over a token's positions
   below 2^119, as in bz_long_cache.h); softmax terms meet V as two bf16 terms each in rows of up to 16 / G tokens (off by at most
   2^-17 of themselves), in longer ones as two or as one (2^-8, as the output's own rounding), by the batch's sizes and the hints;
   max_tokens of up to 64 / G makes it two in all rows. */
int bz_gqa_paged(const bz_gqa_paged_args* args, hipStream_t stream);

/* Workspace bytes of bz_gqa_paged calls with this head_dim whose rows have up to max_tokens new tokens (0: any): at head_dim 128 and
   256 CUs 8.8 MB with max_tokens * group <= 16, 17 MB up to 64, else 77 MB; at head_dim 64 half of that. */
int bz_paged_workspace_size(int32_t head_dim, int32_t group, int32_t max_tokens, size_t* bytes);

#ifdef __cplusplus
}
#endif

#endif /* BZ_PAGED_CACHE_H */
