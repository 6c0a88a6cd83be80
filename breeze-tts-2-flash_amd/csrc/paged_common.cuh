// What the kernels of the paged cache share (include/bz_paged_cache.h): a batch's rows and tokens, the page of a position, and the
// values of 8-bit codes.
#pragma once

#include "bz_paged_cache.h"
#include "device_common.cuh"

constexpr int64_t kMaxGrid = (1 << 24) - 1;  // of 256 threads: HIP takes fewer than 2^32 in a dimension
constexpr int64_t kMaxPositions = 1 << 30;  // sums of positions, tokens and tile sizes stay in 32 bits

namespace bz {

struct PagedRows {
  const int32_t* table;
  int64_t table_st;
  const int32_t *seq_lens, *q_start;
  int B, tokens, max_pages, pages, pshift;
};

int check_paged(const bz_paged_cache* c, bool rows);  // paged_store.hip
PagedRows paged_rows(const bz_paged_cache* c);

// The row of token n and its position there; false for a token of no row, and where the position passes 32 bits. (A binary search;
// with a q_start that decreases it ends all the same, at a row that is checked to hold n.)
__device__ __forceinline__ bool row_of(const PagedRows& r, int n, int& row, int& pos) {
  int b = n, end = n + 1;
  if (r.q_start != nullptr) {
    int lo = 0, hi = r.B;  // the first row that ends behind n
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (r.q_start[mid + 1] <= n) lo = mid + 1;
      else hi = mid;
    }
    if (lo >= r.B || r.q_start[lo] > n) return false;
    b = lo, end = r.q_start[lo + 1];
  }
  const int64_t at = (int64_t)r.seq_lens[b] - ((int64_t)end - n);
  row = b, pos = (int)at;
  return at == pos;
}

// The page of position pos of a row, -1 where there is none.
__device__ __forceinline__ int page_of(const PagedRows& r, int row, int pos) {
  if (pos < 0 || (pos >> r.pshift) >= r.max_pages) return -1;
  const int page = r.table[row * r.table_st + (pos >> r.pshift)];
  return (uint32_t)page < (uint32_t)r.pages ? page : -1;
}

// Two e4m3 codes (half HI of w) times 2^(E - 127) as a bf16 pair: exact (three mantissa bits, and from E = 10 on no value
// below 2^-126), and NaN for E = 255 (v_cvt_scalef32_pk_bf16_fp8 takes the exponent of its fp32 scale operand).
template <bool HI>
__device__ __forceinline__ uint32_t f8_pair(uint32_t w, uint32_t e) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, __uint_as_float(e << 23), HI));
}
__device__ __forceinline__ uint4 f8_values(uint2 w, uint32_t e) {
  return make_uint4(f8_pair<false>(w.x, e), f8_pair<true>(w.x, e), f8_pair<false>(w.y, e), f8_pair<true>(w.y, e));
}

}  // namespace bz
