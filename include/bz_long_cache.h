/*
 * bz_long_cache.h - C ABI of libbz_gqa_decode.so for keeping a long KV cache small and reading it: attention with a
 * sliding window and sinks, a KV cache held in 4 bits, and eviction by accumulated attention weight.
 *
 * Conventions are those of bz_gqa_decode.h (device pointers on the current device, strides in elements unless stated,
 * no allocation, no host decision from device data, bz_status return values, nothing launched when a check fails).
 *
 * Range rule. Row b holds positions [kv_start[b], seq_lens[b]) (clamped as in bz_gqa_decode). With T query tokens per
 * row, token t is the row's position seq_lens[b] - T + t and ends at e_t = max(kv_start[b], seq_lens[b] - (T - 1 - t)).
 * It attends the positions p of [kv_start[b], e_t) with window == 0, p >= e_t - window, or p < kv_start[b] + sinks: the
 * last `window` positions up to its own, and the row's first `sinks`. A token that attends nothing, or whose scores are all
 * -inf, yields zeros, as in bz_gqa_decode. What is stored at positions a token does not attend (NaN and infinities among it)
 * does not reach its output. Outputs are sums in fp32 of terms of up to 2^8 times V, divided by the terms' sum at the end: the sum
 * of |V| over the positions a token attends must stay below 2^119.
 */
#ifndef BZ_LONG_CACHE_H
#define BZ_LONG_CACHE_H

#include "bz_gqa_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Arguments of bz_gqa_window. base: as for bz_gqa_decode, with mask NULL and mask_dtype 0; tokens_per_row T may be one or
   a whole prompt; num_splits 0 picks the default; combine is ignored; workspace of at least bz_long_workspace_size(..)
   bytes where that is not 0.
   Two kernels, by the units of the call (batch * num_kv_heads * the tiles of 16 (token, q head) columns a row has, at most 16
   / group tokens each). With one tile a row, or fewer units than the device has CUs, the split kernel, unless num_splits is 0,
   a row has at least 128 columns and the positions are long enough to half fill the device with shares of 128 columns; else the
   chunk kernel. Softmax terms meet V as two bf16 terms in the split kernel (each off by at most 2^-17 of itself), as
   one in the chunk kernel (at most 2^-8, as the output's own rounding), where the products are the bound. The chunk kernel
   takes at most 65535 tiles of 128 columns, times splits, a row (BZ_ERR_SHAPE beyond): about a million tokens with a group of 8. */
typedef struct bz_gqa_window_args {
  bz_gqa_decode_args base;
  int32_t window;             /* >= 0; 0: no window (plain causal attention) */
  int32_t sinks;              /* >= 0; first positions of the row that stay visible */
} bz_gqa_window_args;

/* Causal attention of the row's last T positions over a bf16 cache, by the range rule above. */
int bz_gqa_window(const bz_gqa_window_args* args, hipStream_t stream);

/* A KV cache in 4 bits, for each of K and V: codes uint8 [batch, num_kv_heads, capacity, head_dim / 2], the even dim of
   each pair in the low four bits, and scales uint8 [batch, num_kv_heads, capacity, head_dim / 32], one for each 32
   consecutive dims. A code holds a sign, two exponent bits and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6); a scale
   byte E stands for 2^(E - 127), 255 for NaN (every value of its block). K and V share strides. The last dimension of
   codes and the last two of scales are contiguous. Strides are in bytes; code pointers and strides are multiples of 8
   (16 with head_dim 128), scale pointers and strides multiples of head_dim / 32. */
typedef struct bz_kv4_cache {
  void *k, *v;
  int64_t stride_b, stride_h, stride_s;
  void *k_scale, *v_scale;
  int64_t scale_stride_b, scale_stride_h;
  int32_t batch, num_kv_heads, capacity, head_dim;
} bz_kv4_cache;

/* Rounds k and v (bf16 [batch, num_kv_heads, tokens, head_dim], 16-byte aligned with strides of multiples of 8 elements)
   into the slots slots[b] .. slots[b] + tokens - 1 of row b. The scale of a block is the smallest power of two (from
   2^-126) with max |x| / scale <= 7, codes are x / scale rounded to nearest even and saturated at 6; a block that holds NaN
   or an infinity gets scale byte 255. (Values from 1.75 * 2^127 on become 4 * 2^126, which bf16 reads as infinity.) counts,
   optional int32 [batch]: only the first counts[b] tokens of row b are stored. Slots outside [0, capacity) are skipped. k and
   v share strides; the cache's four tensors share no memory. */
int bz_kv4_store(const void* k, const void* v, int64_t x_stride_b, int64_t x_stride_h, int64_t x_stride_t, int32_t tokens,
                 const int32_t* slots, const int32_t* counts, const bz_kv4_cache* cache, hipStream_t stream);

/* The bf16 values of slots slots[b] .. slots[b] + tokens - 1 of row b, into k and v (layout as in bz_kv4_store; they
   share no memory); zeros for slots outside [0, capacity). */
int bz_kv4_load(const bz_kv4_cache* cache, const int32_t* slots, int32_t tokens, void* k, void* v, int64_t x_stride_b,
                int64_t x_stride_h, int64_t x_stride_t, hipStream_t stream);

/* Arguments of bz_gqa_decode_kv4. base: as for bz_gqa_window, but k_cache, v_cache, kv_stride_*, batch, num_kv_heads,
   capacity and head_dim are taken from cache; at most 16 tokens per row. */
typedef struct bz_gqa_kv4_args {
  bz_gqa_decode_args base;
  bz_kv4_cache cache;
  int32_t window, sinks;
} bz_gqa_kv4_args;

/* Decode attention over a 4-bit cache, by the range rule above. */
int bz_gqa_decode_kv4(const bz_gqa_kv4_args* args, hipStream_t stream);

/* Arguments of bz_gqa_decode_tracked. base: as for bz_gqa_decode with one token per row and no mask. */
typedef struct bz_gqa_tracked_args {
  bz_gqa_decode_args base;
  const float* weights;       /* [batch, num_kv_heads, capacity], last dimension contiguous */
  int64_t w_stride_b, w_stride_h;
  float* weights_out;         /* as weights; may be weights itself, else must not overlap it */
  int64_t wo_stride_b, wo_stride_h;
  float decay;
} bz_gqa_tracked_args;

/* bz_gqa_decode, and for every position p of the row's range
   weights_out[b, h, p] = decay * weights[b, h, p] + the sum over the q heads of kv head h of their softmax probability of
   p (decay 0: weights is not read). Other positions of weights_out are left as they were. */
int bz_gqa_decode_tracked(const bz_gqa_tracked_args* args, hipStream_t stream);

/* Workspace bytes of the three attention entry points above (0 where none is needed); a workspace is zero-filled once,
   256-byte aligned, and serves every later call of any of them that it is large enough for and that has as many units once
   those are rounded up to a power of two, at least BZ_LONG_SHARED_UNITS (units: batch * num_kv_heads * the column tiles of
   a row, tokens_per_row over 16 / group, at most tokens_per_row, rounded up). Two calls that share one must be ordered on
   one stream. */
#define BZ_LONG_SHARED_UNITS 512
typedef enum bz_long_kind { BZ_LONG_WINDOW = 0, BZ_LONG_KV4 = 1, BZ_LONG_TRACKED = 2 } bz_long_kind;
int bz_long_workspace_size(int32_t kind, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                           int32_t capacity, int32_t tokens_per_row, int32_t window, int32_t sinks, int32_t num_splits,
                           int32_t max_seq_len, size_t* bytes);

/* Which positions of each (row, kv head) stay when at most `keep` may. A row of n = seq_lens - kv_start positions with
   n <= keep keeps all; else its first `sinks` and last `recent` positions and the keep - sinks - recent of the others with
   the largest weight, of equal ones the lower position (NaN counts as the largest, -0 as 0). index [batch, num_kv_heads,
   keep] int32, contiguous: the positions kept, ascending, then -1; lens [batch] int32: how many (may be seq_lens or kv_start
   itself, not shifted over them).
   weights_out (optional; may be weights itself, else must not overlap it): the kept positions' weights from slot 0 on,
   then zeros up to the row's old end; slots from the old end on are left as they were. sinks + recent <= keep <= capacity. */
typedef struct bz_kv_select_args {
  const float* weights;       /* [batch, num_kv_heads, capacity], last dimension contiguous */
  int64_t w_stride_b, w_stride_h;
  const int32_t* seq_lens;
  const int32_t* kv_start;    /* may be NULL */
  int32_t* index;
  int32_t* lens;
  float* weights_out;         /* may be NULL */
  int64_t wo_stride_b, wo_stride_h;
  int32_t batch, num_kv_heads, capacity, keep, sinks, recent;
} bz_kv_select_args;
int bz_kv_select(const bz_kv_select_args* args, hipStream_t stream);

/* One tensor of bz_kv_compact: [batch, num_kv_heads, capacity] rows of row_bytes contiguous bytes; strides in bytes. dst
   is src with the same strides (in place), or does not overlap it. */
typedef struct bz_kv_tensor {
  const void* src;
  void* dst;
  int64_t src_stride_b, src_stride_h, src_stride_s;
  int64_t dst_stride_b, dst_stride_h, dst_stride_s;
  int32_t row_bytes;
} bz_kv_tensor;

/* For each of up to BZ_KV_TENSORS tensors, (row, kv head) and d < min(lens[b], keep): row d of dst is row index[b, h, d] of
   src. Other rows of dst are left as they were, and so is row d where index[b, h, d] lies outside [0, capacity). In place
   index[b, h, :lens[b]] must ascend strictly (bz_kv_select's does). */
#define BZ_KV_TENSORS 4
int bz_kv_compact(const bz_kv_tensor* tensors, int32_t num_tensors, const int32_t* index, const int32_t* lens,
                  int32_t batch, int32_t num_kv_heads, int32_t capacity, int32_t keep, hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* BZ_LONG_CACHE_H */
