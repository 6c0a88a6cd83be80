// Device code of the attention over a long cache (include/bz_long_cache.h): a sliding window with sinks over a bf16 cache,
// the same over a 4-bit cache, and the decode step that records its scores for the accumulated weights.
//
//   out = sum_p softmax_p(scale q . k_p) v_p over the positions a token attends: [kv_start, e_t) from e_t - window on, and
//   the row's first `sinks`.
//
// The (token, q head) pairs that share a kv head are the columns of one product: 16 columns a workgroup (tokens
// t0 .. t0 + 16 / G - 1 of a row times the G heads of the group), so K and V are read once for all of them. The positions
// any of the columns attends are at most two intervals, the sinks and the window; they are cut into wave tiles of 16
// (bf16) or 32 (4-bit) positions, aligned to their size, numbered through, and dealt to the splits and waves, so the work
// follows the attended positions however long the row is. Each column masks what it does not attend.
#pragma once

#include "bz_long_cache.h"
#include "gqa_kernels.cuh"

namespace bz {

struct LongParams {
  const uint16_t* q;
  int64_t q_sb, q_sh, q_st;
  const char *k, *v;            // bf16 rows, or 4-bit codes
  int64_t kv_sb, kv_sh, kv_ss;  // bytes
  const uint8_t *k_scale, *v_scale;
  int64_t sc_sb, sc_sh;         // bytes; head_dim / 32 bytes a position
  int window, sinks;            // window INT32_MAX: none
  float scale_log2;             // scale * log2(e)
  uint16_t* out;
  int64_t o_sb, o_sh, o_st;
  int out_wide;                 // out and its strides are multiples of 8 bytes
  int NKV, G, gshift, T, cap;   // G = 1 << gshift q heads per kv head
  int tiles, tpt;               // column tiles per row, tokens per column tile (16 / G)
  int rows;                     // balanced: rows * column tiles, at most 64
  float inv_splits;             // 1 / splits; balanced: 1 / (splits * rows)
  int splits, min_tiles, one_split;  // a split takes at least min_tiles wave tiles; up to one_split in all are not split
  float* part_acc;              // [row * tile, kv head, split, column, D] unnormalised sums; balanced: [kv head, workgroup, ..]
  float2* part_ml;              // [row * tile, kv head, split, column] (max, sum); the same
  int* counters;                // [row * tile, kv head] x kCounterStride
  float* scores;                // tracked: [row, q head, score_stride] scores times log2(e)
  int score_stride;
  float2* head_ml;              // tracked: [row, q head] (max, 1 / sum)
  const float* weights;         // tracked
  float* weights_out;
  int64_t w_sb, w_sh, wo_sb, wo_sh;
  float decay;
  int fuse;                     // tracked: the merging workgroup adds the row's weights too (no second launch)
};

}  // namespace bz

namespace {

using bz::LongParams;

constexpr int kApplyThreads = 256;
constexpr int kLongCols = 16, kMaxGroup = 8;
constexpr int kBf16 = 0, kKv4 = 1, kKv4Packed = 2;  // cache formats of the split kernel

__device__ __forceinline__ int clamp_int(int x, int lo, int hi) { return min(max(x, lo), hi); }

// [start, end) of row b, clamped to the cache as clamp_range does.
__device__ __forceinline__ void long_range(int e_raw, int s_raw, bool has_start, int cap, int& start, int& end) {
  end = wave_uniform(clamp_int(e_raw, 0, cap));
  start = has_start ? wave_uniform(clamp_int(s_raw, 0, end)) : 0;
}

// What one column (query token) attends: [lo, lo + len) and [s, s + sink).
struct Reach {
  int lo, len, sink;
};
__device__ __forceinline__ Reach reach_of(int s, int token_end, int window, int sinks) {
  const int lo = max(s, token_end - window);
  return {lo, token_end - lo, min(sinks, token_end - s)};
}
__device__ __forceinline__ bool attends(const Reach& c, int s, int pos) {
  return (uint32_t)(pos - c.lo) < (uint32_t)c.len || (uint32_t)(pos - s) < (uint32_t)c.sink;
}

// The wave tiles (P positions each, aligned) that hold every position some column of a workgroup attends: na tiles from
// position fa on (sinks) and nb tiles from fb on (window). e0 and e1: the ends of its first and last token.
struct TileRange {
  int fa, na, fb, nb;
};
template <int P>
__device__ __forceinline__ TileRange tile_range(int s, int e0, int e1, int window, int sinks) {
  TileRange t{s & ~(P - 1), 0, 0, 0};
  if (e1 <= s) return t;
  t.fb = max(s, e0 - window) & ~(P - 1);
  const int a1 = s + min(sinks, e1 - s);
  if (a1 > s) t.na = (a1 - t.fa + P - 1) / P;
  if (t.na > 0 && t.fa + t.na * P > t.fb) t.na = 0, t.fb = t.fa;  // they touch: one interval
  t.nb = (e1 - t.fb + P - 1) / P;
  return t;
}

// ------------------------------------------------------------------------------------------------ wave tiles

// With r = lane % 16 and g = lane / 16, a lane scores the positions pos0 + 16 s + 4 g + i (s < P / 16, i < 4) of column r,
// and holds V of the same positions, so P goes from K . q^T to V^T . P^T without leaving its lane.

// 32 positions of 4-bit codes. K: lane (r, g) holds the D / 4 dims from (D / 4) g on of rows r and 16 + r, one load each
// (64 lanes read 16 whole rows); the products take dims in any order as long as q's operand has the same, so product j
// of a row takes dims (D / 4) g + 8 j .. + 7, and all of a lane's codes lie in one block of 32: one scale. V: dims (D / 16) r
// .. of its 8 positions.
template <int D>
struct Kv4Tile {
  static constexpr int P = 32;
  uint32_t k[2][D / 32];
  uint32_t ks[2];
  uint32_t v[8];
  uint32_t vs[8];  // the scale byte of this lane's dims
};

struct Kv4Spans {
  Rsrc k, v, ks, vs;
  uint32_t row_bytes;
};

// PACKED: the rows lie one behind the other, so the loads of a tile differ by constants, which the instructions hold: about 30
// vector instructions a tile fewer (one workgroup over 32768 positions, head_dim 128: 169 us; with the row's stride 177).
template <int D, bool PACKED>
__device__ __forceinline__ void load_kv4_tile(Kv4Tile<D>& t, const Kv4Spans& sp, int pos0, int r, int g) {
  constexpr int SB = D / 32;  // scale bytes of a position
  const uint32_t row_bytes = PACKED ? D / 2 : sp.row_bytes;
  uint32_t ko = (pos0 + r) * row_bytes + (D / 8) * g, kso = (pos0 + r) * SB + (D == 128 ? g : g / 2);
  uint32_t vo = (pos0 + 4 * g) * row_bytes + (D / 32) * r, vso = (pos0 + 4 * g) * SB + r / (D == 128 ? 4 : 8);
  asm("" : "+v"(ko), "+v"(kso), "+v"(vo), "+v"(vso));  // sums as they stand here: not as ors, which no instruction holds
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const uint32_t off = ko + 16 * s * row_bytes;
    if constexpr (D == 128) {
      const uint4 w = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(sp.k, off, 0, kStream));
      t.k[s][0] = w.x, t.k[s][1] = w.y, t.k[s][2] = w.z, t.k[s][3] = w.w;
    } else {
      const uint2 w = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(sp.k, off, 0, kStream));
      t.k[s][0] = w.x, t.k[s][1] = w.y;
    }
    t.ks[s] = __builtin_amdgcn_raw_buffer_load_b8(sp.ks, kso + 16 * s * SB, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int step = 16 * (i / 4) + i % 4;
    const uint32_t off = vo + step * row_bytes;
    if constexpr (D == 128) t.v[i] = __builtin_amdgcn_raw_buffer_load_b32(sp.v, off, 0, kStream);
    else t.v[i] = __builtin_amdgcn_raw_buffer_load_b16(sp.v, off, 0, kStream);
    t.vs[i] = __builtin_amdgcn_raw_buffer_load_b8(sp.vs, vso + step * SB, 0, 0);
  }
}

// Two 4-bit codes (byte SEL of w) times 2^(E - 127) as a bf16 pair: exact, and NaN for E = 255 (v_cvt_scalef32_pk_bf16_fp4
// takes the exponent of its fp32 scale operand).
template <int SEL>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, uint32_t e) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, __uint_as_float(e << 23), SEL));
}

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
// Whether a packed bf16 pair, its signs cleared, holds an infinity or NaN in either half, from the halves' maxima.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
__device__ __forceinline__ bool pair_not_finite(uint32_t m) { return (m & 0xffffu) >= 0x7f80u || (m >> 16) >= 0x7f80u; }
// The pair with non-finite halves replaced by 0.
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  const uint32_t lo = (w & 0x7fffu) >= 0x7f80u ? 0u : w & 0xffffu, hi = (w & 0x7fff0000u) >= 0x7f800000u ? 0u : w & 0xffff0000u;
  return lo | hi;
}

// Scores are taken times a positive scale, which a maximum may be taken before; the query carries the sign. (1e-30 stands for
// a scale of 0, whose product with an excluded position's -inf would be NaN; for a scale that is NaN as well, and the query is
// NaN then: so are the scores of the positions a token attends, and no others.)
__device__ __forceinline__ float positive_scale(float scale_log2) { return fmaxf(fabsf(scale_log2), 1e-30f); }
__device__ __forceinline__ bf16x8_t signed_q(uint4 q, float scale_log2) {
  const uint32_t flip = scale_log2 < 0.f ? 0x80008000u : 0u;
  q.x ^= flip, q.y ^= flip, q.z ^= flip, q.w ^= flip;
  if (scale_log2 != scale_log2) q.x = q.y = q.z = q.w = 0x7fff7fffu;
  return __builtin_bit_cast(bf16x8_t, q);
}

// The running state of one wave: column r's max (the same in the column's four lanes) and sum (over the lane's own
// positions), and acc[n][i]: dim (D / 16)(4 g + i) + n of column r.
template <int D>
struct LongState {
  float m, l;
  f32x4_t acc[D / 16];
};

// One wave tile's products x (q . k times a positive scale is the score in base 2; -inf where not attended) folded into the
// running max and sum; x becomes the softmax terms 2^(scale x - m). The running maximum moves only when a column's has grown
// by more than 2^8, so that the accumulators are rarely rescaled: until then its terms stay below 2^8, and what rounds them
// is relative.
template <int D, int N>
__device__ __forceinline__ void fold_scores(LongState<D>& st, float (&x)[N], float scale) {
  float mt[1] = {x[0]};
#pragma unroll
  for (int i = 1; i < N; ++i) mt[0] = fmaxf(mt[0], x[i]);
  rows_max<1>(mt);
  const float top = mt[0] * scale;
  if (__ballot(top > st.m + 8.f) != 0) {
    const float mn = fmaxf(st.m, top), mu = (mn == -INFINITY) ? 0.f : mn, alpha = fast_exp2(st.m - mu);
    st.m = mn;
    st.l *= alpha;
#pragma unroll
    for (int n = 0; n < D / 16; ++n) st.acc[n] *= alpha;
  }
  const float base = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = fast_exp2(fmaf(x[i], scale, -base));
    st.l += x[i];
  }
}

// The softmax terms as two bf16 terms each, hi + lo (16 bits of each p: an error of 2^-17 at most, below the 2^-8 that the
// output's own rounding to bf16 costs at most; one term alone would add as much error again as that rounding).
template <int N>
__device__ __forceinline__ void split_terms(const float (&p)[N], uint32_t (&hi)[N / 2], uint32_t (&lo)[N / 2]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    hi[i] = pack_bf16x2(p[2 * i], p[2 * i + 1]);
    lo[i] = pack_bf16x2(p[2 * i] - bf16_lo(hi[i]), p[2 * i + 1] - bf16_hi(hi[i]));
  }
}

// acc += V^T P for operands of N positions a lane (4: 16 positions a wave, 8: 32).
template <int N>
__device__ __forceinline__ f32x4_t mfma_pv(const uint32_t (&v)[N / 2], const uint32_t (&p)[N / 2], f32x4_t acc) {
  if constexpr (N == 4)
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4_t, make_uint2(v[0], v[1])),
                                                     __builtin_bit_cast(s16x4_t, make_uint2(p[0], p[1])), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, make_uint4(v[0], v[1], v[2], v[3])),
                                                   __builtin_bit_cast(bf16x8_t, make_uint4(p[0], p[1], p[2], p[3])), acc, 0, 0, 0);
}

// The pair with finite halves replaced by 0.
__device__ __forceinline__ uint32_t odd_pair(uint32_t w) { return w & ~finite_pair(w); }

// st.acc += V^T P. v[i][m]: bf16 dims 2 m and 2 m + 1 of this lane's dims at its i-th position; pos(i): that position.
// Where V holds an infinity or NaN (bad, any lane of the wave), 0 times it must not reach the columns that do not attend
// its position: each column then takes a product of its own with the non-finite values of the positions it attends (in the
// higher terms alone: p times an infinity is the infinity), and the product of all columns what is left.
template <int D, int N, class Pos>
__device__ __forceinline__ void accumulate(LongState<D>& st, uint32_t (&v)[N][D / 32], const float (&p)[N], bool bad,
                                           int col, int ncol, const Reach& mine, int s, Pos pos) {
  uint32_t hi[N / 2], lo[N / 2];
  split_terms(p, hi, lo);
  auto operand = [](const uint32_t (&x)[N][D / 32], int n, uint32_t (&vt)[N / 2]) {
#pragma unroll
    for (int a = 0; a < N / 2; ++a)
      vt[a] = n % 2 ? pair_hi(x[2 * a][n / 2], x[2 * a + 1][n / 2]) : pair_lo(x[2 * a][n / 2], x[2 * a + 1][n / 2]);
  };
  if (__builtin_expect(__ballot(bad) != 0, 0)) {
    for (int c = 0; c < ncol; ++c) {
      const Reach rc{__builtin_amdgcn_readlane(mine.lo, c), __builtin_amdgcn_readlane(mine.len, c),
                     __builtin_amdgcn_readlane(mine.sink, c)};
      uint32_t keep[N / 2];  // the halves of each operand word whose positions the column attends
#pragma unroll
      for (int a = 0; a < N / 2; ++a)
        keep[a] = (attends(rc, s, pos(2 * a)) ? 0xffffu : 0u) | (attends(rc, s, pos(2 * a + 1)) ? 0xffff0000u : 0u);
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t vt[N / 2];
        operand(v, n, vt);
#pragma unroll
        for (int a = 0; a < N / 2; ++a) {
          vt[a] = odd_pair(vt[a]) & keep[a];
          asm volatile("" : "+v"(vt[a]));  // worked out here, not for all columns before the loop (registers)
        }
        const f32x4_t t = mfma_pv<N>(vt, hi, f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int i = 0; i < 4; ++i) st.acc[n][i] += col == c ? t[i] : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int m = 0; m < D / 32; ++m) v[i][m] = finite_pair(v[i][m]);
  }
#pragma unroll
  for (int n = 0; n < D / 16; ++n) {
    uint32_t vt[N / 2];
    operand(v, n, vt);
    st.acc[n] = mfma_pv<N>(vt, hi, st.acc[n]);
    st.acc[n] = mfma_pv<N>(vt, lo, st.acc[n]);
  }
}

// Merges nact partials of ncol columns in split order and writes out (and, tracked, each head's max and 1 / sum). Each
// thread owns 4 consecutive values of one column; the weights of 16 splits at a time are worked out by the lanes of a
// 16-lane row and handed round by DPP, as in merge_many. write(column, dim, values, max, sum).
template <int D, int NT, class Write>
__device__ __forceinline__ void merge_columns(const float* part_acc, const float2* part_ml, int ncols_max, int ncol, int nact,
                                              Write write) {
  const Rsrc racc = span_rsrc(part_acc, nact * ncols_max * D * 4), rml = span_rsrc(part_ml, nact * ncols_max * 8);
  const int lane16 = threadIdx.x % 16;
  for (int o = threadIdx.x; o < ncol * D / 4; o += NT) {
    const int c = o / (D / 4);
    float m = -INFINITY, l = 0.f;
    f32x4_t a = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < nact; s0 += 16) {
      const uint2 ml = __builtin_bit_cast(
          uint2, __builtin_amdgcn_raw_buffer_load_b64(rml, ((s0 + lane16) * ncols_max + c) * 8, 0, kSc1));
      f32x4_t v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u)
        v[u] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                               racc, ((s0 + u) * ncols_max * (D / 4) + o) * 16, 0, kSc1));
      const float ms = s0 + lane16 < nact ? __uint_as_float(ml.x) : -INFINITY;  // sums and values are 0 past nact
      const float mn = fmaxf(m, row_max16(ms));
      const float mu = (mn == -INFINITY) ? 0.f : mn;
      const float alpha = fast_exp2(m - mu), e = fast_exp2(ms - mu);
      m = mn;
      l = fmaf(l, alpha, row_sum<16>(e * __uint_as_float(ml.y)));
      a *= alpha;
      row_lanes(e, [&](int u, float w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = fmaf(w, v[u][i], a[i]);
      });
    }
    write(c, 4 * (o % (D / 4)), a, m, l);
  }
}

// weights_out[b, h, pos] = decay * weights[b, h, pos] + sum_g 2^(score - max_g) / sum_g over the row's range [s, e): four consecutive
// positions a thread and turn, their scores (16-byte loads, coherent with the other workgroups' stores) and old weights loaded by
// load_turn and added by add_turn. ml(g): (max, 1 / sum) of the group's q head g.
struct WeightTurn {
  f32x4_t x[kMaxGroup], old;
};
__device__ __forceinline__ WeightTurn load_turn(const LongParams& p, int b, int h, int s, int e, int pos0) {
  WeightTurn t;
  t.old = f32x4_t{0.f, 0.f, 0.f, 0.f};
  if (pos0 >= e) return t;
  const int row = p.score_stride * 4;  // bytes; below 2^27 (host), so those of a group below 2^30
  const Rsrc rs = span_rsrc(wave_uniform(p.scores + ((int64_t)b * p.NKV + h) * p.G * p.score_stride), p.G * row);
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g) {
    if (g >= p.G) break;
    t.x[g] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, 4 * pos0, g * row, kSc1));
  }
  if (p.decay != 0.f) {
    const float* const wi = p.weights + (int64_t)b * p.w_sb + (int64_t)h * p.w_sh;
#pragma unroll
    for (int i = 0; i < 4; ++i) t.old[i] = wi[clamp_int(pos0 + i, s, e - 1)];  // outside the range: unused
  }
  return t;
}
template <class Ml>
__device__ __forceinline__ void add_turn(const LongParams& p, int b, int h, int s, int e, int pos0, const WeightTurn& t, Ml ml) {
  float* const wo = p.weights_out + (int64_t)b * p.wo_sb + (int64_t)h * p.wo_sh;
  if (pos0 >= e) return;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < kMaxGroup; ++g) {
    if (g >= p.G) break;
    const float2 y = ml(g);
    const float mu = y.x == -INFINITY ? 0.f : y.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(fast_exp2(t.x[g][i] - mu), y.y, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (pos0 + i >= s && pos0 + i < e) wo[pos0 + i] = p.decay == 0.f ? acc[i] : fmaf(p.decay, t.old[i], acc[i]);
}

// ------------------------------------------------------------------------------------------------ split kernel

// What a workgroup takes: (row, column tile) z; balanced, also the first workgroup of z and the wave tiles of a split.
struct Share {
  int z, first, per;
};
// Balanced: lane i works out how many wave tiles (row, column tile) i has, and the wave the tiles a split takes, the same for all
// rows (every workgroup streams at about the same rate, so the longest share is what the launch takes), in steps of the
// waves. First what all rows have together over the grid, which fits where lengths are equal; then the same with as many
// workgroups set aside as rounding up took; then what fits for certain: sum max(1, ceil(n / c)) <= sum n / c + rows <= grid, or
// the longest row in as many splits as each has on average.
// At most 64 splits of a row to merge.
template <int P, int NW, bool BAL>
__device__ __forceinline__ Share deal_splits(const int32_t* lens, const int32_t* starts, const LongParams& p) {
  if constexpr (!BAL) return {(int)blockIdx.z, 0, 0};
  const int lane = threadIdx.x % kWave, zl = min(lane, p.rows - 1);
  const int b = p.tiles == 1 ? zl : zl / p.tiles, t0 = (zl - b * p.tiles) * p.tpt;
  const int e_raw = lens[b], s_raw = (starts ? starts : lens)[b];
  const int e = clamp_int(e_raw, 0, p.cap), s = starts ? clamp_int(s_raw, 0, e) : 0;
  auto token_end = [&](int t) { return max(s, e - (p.T - 1 - t)); };
  const TileRange tr = tile_range<P>(s, token_end(t0), token_end(min(t0 + p.tpt, p.T) - 1), p.window, p.sinks);
  const int n = lane < p.rows ? tr.na + tr.nb : 0;
  const float all = 1.000001f * (float)__builtin_amdgcn_readlane((int)wave_scan((uint32_t)n), kWave - 1);
  const int most = wave_uniform((int)wave_max((float)n)), least = max(p.min_tiles, (most + 63) / 64);
  const int grid = p.splits * p.rows;
  const float certain = fminf(all / (float)(grid - p.rows), 1.000001f * (float)most / (float)p.splits);
  float share = all * p.inv_splits;
  int per, k, last;
  for (int i = 0; i < 3; ++i) {
    per = (max(least, (int)share + 1) + NW - 1) & ~(NW - 1);
    const float inv = __builtin_amdgcn_rcpf((float)per);
    k = lane >= p.rows ? 0 : n <= p.one_split ? 1 : max(1, ceil_div_est(n, per, inv));
    last = (int)wave_scan((uint32_t)k);
    const int need = __builtin_amdgcn_readlane(last, kWave - 1);
    if (need <= grid) break;
    share = i == 0 ? fminf(all / fmaxf((float)grid - ((float)need - all * inv), 1.f), certain) : certain;
  }
  const uint64_t mine = __ballot((int)blockIdx.x < last && (int)blockIdx.x >= last - k);
  if (mine == 0) return {-1, 0, 0};
  const int z = __builtin_ctzll(mine);
  return {z, __builtin_amdgcn_readlane(last - k, z), per};
}

// FMT: the cache's format. TRACK: also writes the scores (one token per row). Grid (splits, kv heads, rows * column tiles), each
// row cut into as many splits; BAL: (splits * rows * column tiles, kv heads), dealt to the rows by their lengths (deal_splits).
//
// Four waves take every fourth wave tile of their split; a tile's loads are issued two tiles ahead, into registers, and the
// product's columns are complete within a wave, so the waves meet once, at the end (LDS), and the workgroups once (the
// counters). What bounds it (us): a bf16 cache over long rows the stream (16 rows of 500..16384 behind a window of 4096, 8 kv
// heads, head_dim 128: 269 MB in 38.4, 7.0 TB/s, a plain read's rate); few rows the launch, two round trips of loads and the
// merge across workgroups (2 rows, window 1024: 6.3, 8.4 MB); a 4-bit cache both its stream and the vector instructions, about
// 160 a tile of 32 positions, 64 of them conversions and 32 the transposition of V's pairs (4 rows of 20001..32768, 4 kv
// heads of 8 q: 61 MB in 17.7; a copy of the kernel with the loads alone 17.4 where this took 18.9, with tiles from the L2 17.1).
// V's scales as two 16-byte loads and a bit field each, in place of eight byte loads: no faster.
template <int D, int FMT, bool TRACK, bool BAL, int NT>
__global__ void __launch_bounds__(NT, 2)
    long_split_kernel(const int32_t* lens, const int32_t* starts, const LongParams p) {
  constexpr bool KV4 = FMT != kBf16;
  constexpr int NW = NT / kWave, P = KV4 ? 32 : 16, NS = P / 16, N = 4 * NS, NJ = D / 32;
  const int h = blockIdx.y;
  const Share share = deal_splits<P, NW, BAL>(lens, starts, p);
  if (BAL && share.z < 0) return;  // more workgroups than splits
  const int z = share.z, split = BAL ? (int)blockIdx.x - share.first : (int)blockIdx.x;
  const int b = p.tiles == 1 ? z : z / p.tiles, t0 = (z - b * p.tiles) * p.tpt;
  const int e_raw = lens[b], s_raw = (starts ? starts : lens)[b];
  const int tid = threadIdx.x, lane = tid % kWave, w = wave_uniform(tid / kWave), r = lane % 16, g = lane / 16;

  const int ntok = min(p.tpt, p.T - t0), ncol = ntok << p.gshift;
  const int col = p.T == 1 ? r & (p.G - 1) : r % ncol;  // columns past the last repeat earlier ones
  const int tok = t0 + (col >> p.gshift), hq = (h << p.gshift) + (col & (p.G - 1));

  // the B operand of K . q^T: this lane's column, dims as the tile's K has them; loaded now, used after the first tiles' loads
  // are on their way
  uint4 qr[NJ];
  {
    const uint16_t* qsrc = p.q + (int64_t)b * p.q_sb + (int64_t)tok * p.q_st + (int64_t)hq * p.q_sh;
#pragma unroll
    for (int j = 0; j < NJ; ++j) qr[j] = *reinterpret_cast<const uint4*>(qsrc + (KV4 ? (D / 4) * g + 8 * j : 32 * j + 8 * g));
  }

  int s, e;
  long_range(e_raw, s_raw, starts != nullptr, p.cap, s, e);
  auto token_end = [&](int t) { return max(s, e - (p.T - 1 - t)); };
  const Reach mine = reach_of(s, token_end(tok), p.window, p.sinks);
  const TileRange tr = tile_range<P>(s, token_end(t0), token_end(t0 + ntok - 1), p.window, p.sinks);
  const int n = tr.na + tr.nb;
  // tiles per split, a multiple of the waves (no integer division: about 30 dependent instructions before the first load)
  const int least = n <= p.one_split ? n : BAL ? share.per : max(p.min_tiles, ceil_div_est(n, p.splits, p.inv_splits));
  const int per = max(NW, (least + NW - 1) & ~(NW - 1));
  if (split > 0 && split * per >= n) return;  // past the row's last tile (split 0 always stays)
  const int j0 = split * per, j1 = min(n, j0 + per);
  const int e1 = token_end(t0 + ntok - 1);
  // every column attends the whole of [whole_lo, whole_end)
  const int whole_end = token_end(t0), whole_lo = max(s, e1 - p.window);
  const int past = (e1 + P - 1) & ~(P - 1);  // a tile here lies outside the spans: its loads touch no memory
  auto pos_of = [&](int j) { return j >= j1 ? past : j < tr.na ? tr.fa + P * j : tr.fb + P * (j - tr.na); };

  std::conditional_t<KV4, Kv4Tile<D>, WaveTile<D>> ta, tb;
  [[maybe_unused]] Spans sp;
  [[maybe_unused]] Kv4Spans sp4;
  {
    const int64_t head = (int64_t)b * p.kv_sb + (int64_t)h * p.kv_sh;
    const int span = e1 * (int)p.kv_ss;  // < 2^31 (host)
    if constexpr (KV4) {
      const int64_t sc = (int64_t)b * p.sc_sb + (int64_t)h * p.sc_sh;
      sp4.row_bytes = (uint32_t)p.kv_ss;
      sp4.k = span_rsrc(p.k + head, span);
      sp4.v = span_rsrc(p.v + head, span);
      sp4.ks = span_rsrc(p.k_scale + sc, e1 * (D / 32));
      sp4.vs = span_rsrc(p.v_scale + sc, e1 * (D / 32));
    } else {
      sp.row_bytes = (uint32_t)p.kv_ss;
      sp.lane_off = 0;
      sp.k = span_rsrc(p.k + head, span);
      sp.v = span_rsrc(p.v + head, span);
    }
  }
  auto load = [&](auto& t, int j) {
    if constexpr (KV4) load_kv4_tile<D, FMT == kKv4Packed>(t, sp4, pos_of(j), r, g);
    else load_wave_tile<D, BZ_MASK_NONE>(t, sp, pos_of(j), r, g);
  };

  LongState<D> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) st.acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  int j = j0 + w;
  load(ta, j);
  load(tb, j + NW);
  __builtin_amdgcn_sched_barrier(0);  // q's conversion waits for q: not before the tiles' loads
  const int nact = ceil_div_est(max(n, 1), per, __builtin_amdgcn_rcpf((float)per));  // splits with tiles
  const float scale = positive_scale(p.scale_log2);
  bf16x8_t qf[NJ];
#pragma unroll
  for (int i = 0; i < NJ; ++i) qf[i] = signed_q(qr[i], p.scale_log2);
  auto consume = [&](auto& t, int j) {
    const int pos0 = pos_of(j);
    auto pos = [&](int i) { return pos0 + 16 * (i / 4) + 4 * g + i % 4; };
    float x[N];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      f32x4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NJ; ++k) {
        bf16x8_t kf;
        if constexpr (KV4) {
          const uint32_t c = t.k[u][k], sc = t.ks[u];
          kf = __builtin_bit_cast(bf16x8_t, make_uint4(fp4_pair<0>(c, sc), fp4_pair<1>(c, sc), fp4_pair<2>(c, sc), fp4_pair<3>(c, sc)));
        } else {
          kf = k_operand<D>(t, k);
        }
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[k], d, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * u + i] = d[i];
    }
    if (!(pos0 + P <= whole_end && pos0 >= whole_lo)) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = attends(mine, s, pos(i)) ? x[i] : -INFINITY;
    }
    if constexpr (TRACK) {
      if (r < ncol) {
        float* const row = p.scores + ((int64_t)b * p.NKV * p.G + hq) * p.score_stride;
        const Rsrc rs = span_rsrc(row, p.score_stride * 4);
        using U4 = decltype(__builtin_amdgcn_raw_buffer_load_b128(rs, 0, 0, 0));
        const U4 y = __builtin_bit_cast(U4, f32x4_t{x[0], x[1], x[2], x[3]} * scale);
        // coherent where another workgroup of this launch may read them (for 4 rows of 9000..16384 such stores cost 3 us)
        if (p.fuse) __builtin_amdgcn_raw_buffer_store_b128(y, rs, 4 * (pos0 + 4 * g), 0, kSc1);
        else __builtin_amdgcn_raw_buffer_store_b128(y, rs, 4 * (pos0 + 4 * g), 0, 0);
      }
    }
    fold_scores<D, N>(st, x, scale);
    if constexpr (KV4) {
      uint32_t v[N][NJ];
      uint32_t emax = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t c = t.v[i], sc = t.vs[i];
        v[i][0] = fp4_pair<0>(c, sc), v[i][1] = fp4_pair<1>(c, sc);
        if constexpr (D == 128) v[i][2] = fp4_pair<2>(c, sc), v[i][3] = fp4_pair<3>(c, sc);
        emax = max(emax, sc);
      }
      accumulate<D, N>(st, v, x, emax >= 253, col, ncol, mine, s, pos);  // 2^126 times 4 is past bf16
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int m = 0; m < NJ; ++m) top = max_u16x2(top, t.v[i][m] & 0x7fff7fffu);
      accumulate<D, N>(st, t.v, x, pair_not_finite(top), col, ncol, mine, s, pos);
    }
  };

  for (; j < j1; j += 2 * NW) {
    consume(ta, j);
    if (j + NW >= j1) break;
    load(ta, j + 2 * NW);
    consume(tb, j + NW);
    load(tb, j + 3 * NW);
  }

  // the columns are complete over the wave's positions; only the sums are still one per lane group
  float y = st.l;
  swap16(st.l, y);
  st.l += y;
  y = st.l;
  swap32(st.l, y);
  st.l += y;

  constexpr int PD = D + 4;  // keeps the 16-byte stores free of bank conflicts
  __shared__ __align__(16) float s_acc[NW][kLongCols][PD];
  __shared__ float s_m[NW][kLongCols], s_l[NW][kLongCols];
  if (r < ncol) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < D / 16; q += 4)
        *reinterpret_cast<f32x4_t*>(&s_acc[w][r][D / 16 * (4 * g + i) + q]) =
            f32x4_t{st.acc[q][i], st.acc[q + 1][i], st.acc[q + 2][i], st.acc[q + 3][i]};
    if (g == 0) {
      s_m[w][r] = st.m;
      s_l[w][r] = st.l;
    }
  }
  __syncthreads();

  __shared__ float2 s_head[TRACK ? kLongCols : 1];
  auto write = [&](int c, int d, const f32x4_t& a, float m, float l) {
    const int ot = t0 + (c >> p.gshift), oh = (h << p.gshift) + (c & (p.G - 1));
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN sum stays one
    uint16_t* const o = p.out + (int64_t)b * p.o_sb + (int64_t)ot * p.o_st + (int64_t)oh * p.o_sh + d;
    const uint2 y = make_uint2(pack_bf16x2(a[0] * inv, a[1] * inv), pack_bf16x2(a[2] * inv, a[3] * inv));  // l == 0: a is 0
    if (p.out_wide) {
      *reinterpret_cast<uint2*>(o) = y;
    } else {
      o[0] = (uint16_t)y.x, o[1] = (uint16_t)(y.x >> 16), o[2] = (uint16_t)y.y, o[3] = (uint16_t)(y.y >> 16);
    }
    if (TRACK && d == 0) {
      if (p.fuse) s_head[c] = make_float2(m, inv);
      else p.head_ml[(int64_t)b * p.NKV * p.G + oh] = make_float2(m, inv);
    }
  };
  // tracked: the row's weights, once every score of it is written and its heads' sums are in s_head. The first two turns (all
  // there are up to 2048 positions) may have been loaded before.
  const int turn0 = (s & ~3) + 4 * tid;
  auto turn = [&](int u) { return load_turn(p, b, h, s, e, turn0 + 4 * NT * u); };
  auto add = [&](int u, const WeightTurn& t) {
    add_turn(p, b, h, s, e, turn0 + 4 * NT * u, t, [&](int q) { return s_head[q]; });
  };

  const int ncols_max = p.tpt << p.gshift;
  const int64_t unit = (int64_t)z * p.NKV + h;
  const int64_t part0 = BAL ? (int64_t)h * gridDim.x + share.first : unit * p.splits;  // its first partials
  for (int o = tid; o < ncol * D / 4; o += NT) {
    const int c = o / (D / 4), d = 4 * (o % (D / 4));
    float M = s_m[0][c];
#pragma unroll
    for (int u = 1; u < NW; ++u) M = fmaxf(M, s_m[u][c]);
    const float mu = (M == -INFINITY) ? 0.f : M;
    float L = 0.f;
    f32x4_t A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float f = fast_exp2(s_m[u][c] - mu);
      L = fmaf(f, s_l[u][c], L);
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(&s_acc[u][c][d]);
#pragma unroll
      for (int i = 0; i < 4; ++i) A[i] = fmaf(f, a[i], A[i]);
    }
    if (nact == 1) {
      write(c, d, A, M, L);
    } else {
      const int64_t ps = (part0 + split) * ncols_max;
      const Rsrc rp = span_rsrc(p.part_acc + ps * D, ncols_max * D * 4);
      using U4 = decltype(__builtin_amdgcn_raw_buffer_load_b128(rp, 0, 0, 0));
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(U4, A), rp, 16 * o, 0, kSc1);
      if (d == 0) {
        st_agent(reinterpret_cast<float*>(p.part_ml + ps + c), M);
        st_agent(reinterpret_cast<float*>(p.part_ml + ps + c) + 1, L);
      }
    }
  }
  if (nact == 1) {
    if (TRACK && p.fuse) {
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
      for (int u = 0; turn0 + 4 * NT * u < e; ++u) add(u, turn(u));
    }
    return;
  }

  // the last workgroup of this (row, tile, kv head) to count in merges, as in gqa_split_kernel
  __shared__ int s_last;
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
  if (tid == 0) {
    int* cnt = p.counters + unit * kCounterStride;
    const int prev = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = (prev == nact - 1);
    if (s_last) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  const auto merge = [&]() {
    merge_columns<D, NT>(p.part_acc + part0 * ncols_max * D, p.part_ml + part0 * ncols_max, ncols_max, ncol, nact, write);
  };
  if (TRACK && p.fuse) {
    const WeightTurn a = turn(0), c = turn(1);  // with the partials, not after them
    merge();
    __syncthreads();
    add(0, a);
    add(1, c);
    for (int u = 2; turn0 + 4 * NT * u < e; ++u) add(u, turn(u));
  } else {
    merge();
  }
}

// The weights in a launch of their own, after the split kernel that wrote the scores: grid (chunks of kApplyThreads * 4 positions,
// kv heads, rows). Memory bound: 4 rows x 8 kv heads of 9000..16384, groups of 4: 5.0 us for 15 MB of scores and weights, most
// of them in the L2.
__global__ void __launch_bounds__(kApplyThreads)
    track_apply_kernel(const int32_t* lens, const int32_t* starts, const LongParams p) {
  const int h = blockIdx.y, b = blockIdx.z;
  int s, e;
  long_range(lens[b], (starts ? starts : lens)[b], starts != nullptr, p.cap, s, e);
  for (int pos0 = (s & ~3) + 4 * (blockIdx.x * kApplyThreads + threadIdx.x); pos0 < e; pos0 += 4 * gridDim.x * kApplyThreads)
    add_turn(p, b, h, s, e, pos0, load_turn(p, b, h, s, e, pos0),
             [&](int g) { return p.head_ml[((int64_t)b * p.NKV + h) * p.G + g]; });
}

}  // namespace
