// Device code of bz_gqa_window over a chunk of many query tokens (include/bz_long_cache.h).
//
// The (token, q head) pairs of one kv head are the columns of two products, 32 a wave. The four waves of a workgroup are CG
// column groups times PG = 4 / CG position groups: 4 x 1 fetches K and V once for 128 columns (128 / G tokens of a row times
// its G heads); with 2 x 2 and 1 x 4 a small chunk has more workgroups and fewer steps, each position group taking every
// PG-th tile, and the groups' accumulators are merged through LDS at the end by the log-sum-exp rule.
//
// A workgroup walks the positions any of its tokens attends (the sinks' tiles, then the window's; pre_range) in tiles of 64
// (PG = 1) or 32 positions staged in LDS, two buffers each of K and V per position group, the next loads in flight while a
// tile is worked on.
//   S^T = K Q^T   mfma 32x32x16: A = K rows, B = Q^T (registers, loaded once). A lane then holds 32 scores of one column, the
//                 rows 8 (v / 4) + 4 half + v % 4 of each block of 32 positions, so the softmax is within a lane but for one
//                 swap with lane ^ 32.
//   O^T += V^T P^T: the same 32 scores, as terms rounded to bf16, are the B operand as they stand when the contraction takes
//                 the positions in the order 16 s + 8 a + 4 half + i; A = V^T by ds_read_b64_tr_b16 (four rows of 16 dims,
//                 transposed on the way), which reads them in that order.
// The terms are rounded to one bf16 each (sums are fp32): at most 2^-8 of each term, as the output's own rounding, and less over
// many terms, whose errors differ in sign (against 64 bits 0.00162 and 0.00167 of the output's norm on 333 tokens and on
// 8192, with float32 terms 0.00161 and 0.00162); a second term would cost half as many products again, and here the products are
// the bound.
//
// What bounds it: the matrix and vector instructions of two waves a SIMD, which overlap only partly (8192 tokens, 16 q / 8 kv
// heads, head_dim 128, window 4096: 207 GFLOP in 223 us, 925 TFLOP/s; matrix units busy 42% of the cycles, vector units 42%,
// LDS 43%; 32768 tokens 1030; a large library product reaches 1308). The 8192-token grid is 1.75 rounds of workgroups that
// take two. 64 columns a wave in place of 32 (half the LDS reads a product, accumulators in the second half of the register
// file) measured 637 TFLOP/s against 1024: one wave a SIMD.
#pragma once

#include "long_cache.cuh"

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_lds __attribute__((ext_vector_type(4)));

constexpr int kPreThreads = 256, kPreWaveCols = 32;
constexpr int kPreMinSteps = 8;  // of a split: below, its sums' way through memory costs more than the steps

// LDS of one tile of K or V: TP rows of D bf16, in 16-byte chunks. Chunk c of row r lies in slot c ^ swizzle(r), so that the
// lanes of one read, which take the same chunk of different rows, fall into different banks.
template <int D, int TP>
struct PreLds {
  static constexpr int kRow = 2 * D, kBytes = TP * kRow;
  static __device__ __forceinline__ int k_swz(int r) { return r & (D / 8 - 1); }
  static __device__ __forceinline__ int v_swz(int r) { return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); }
};

// The tiles of TP positions that hold every position some column of a workgroup attends: na from position fa on, of the sinks,
// [fa, a1), and nb from fb on, of the window, up to e1; where sinks and window touch, nb of both. They begin with what is attended,
// aligned to nothing, and their rows past a1 or e1 are not read (stage_tile): what no column attends, such as NaN or infinities
// in memory that nothing has written or that was given up between the sinks and the window, would as a factor of 0 send every
// column to careful_column (1024 tokens, 8 kv heads, G 2, window 1000 behind 5 sinks with NaN between them: 5749 us, 41
// without). e0 and e1: the ends of the workgroup's first and last token.
struct PreRange {
  int fa, a1, na, fb, nb;
};
template <int TP>
__device__ __forceinline__ PreRange pre_range(int s, int e0, int e1, int window, int sinks) {
  if (e1 <= s) return {s, s, 0, s, 0};
  PreRange t{s, s + min(sinks, e1 - s), 0, max(s, e0 - window), 0};
  if (t.a1 >= t.fb) t.fb = s;
  else t.na = (t.a1 - s + TP - 1) / TP;
  t.nb = (e1 - t.fb + TP - 1) / TP;
  return t;
}

// Loads the TP rows from pos0 on (a row past `last` holds a copy of that one, and no column attends it) into
// LDS at base, by CG waves (this one is cg): 64 lanes write 1 KB in lane order, so the swizzle is in which chunk each lane
// fetches.
template <int D, int TP, int CG, bool V>
__device__ __forceinline__ void stage_tile(char* base, const Rsrc& rsrc, int pos0, int last, uint32_t row_bytes, int cg, int lane) {
  using L = PreLds<D, TP>;
  constexpr int RPI = 1024 / L::kRow, CH = D / 8;  // rows an instruction, chunks a row
#pragma unroll
  for (int u = 0; u < L::kBytes / 1024 / CG; ++u) {
    const int row0 = RPI * (cg * (L::kBytes / 1024 / CG) + u), row = row0 + lane / CH, c = lane % CH;
    const uint32_t off = (uint32_t)min(pos0 + row, last) * row_bytes + 16 * (c ^ (V ? L::v_swz(row) : L::k_swz(row)));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(base + row0 * L::kRow), 16, off, 0, 0,
                                             0);
  }
}

// One column, by one wave, in fp32 and without any product of a position that the column does not attend: where a result is
// not finite, which is right where the column attends an infinity or NaN and wrong where a tile held one that it does not (0
// times it). The lanes score 64 positions, then each accumulates D / 64 dims over them.
template <int D>
__device__ __forceinline__ void careful_column(const LongParams& p, int b, int h, int s, int e, int tok, int hq) {
  constexpr int DV = D / 64;
  const int lane = threadIdx.x % kWave;
  const char* const kb = p.k + (int64_t)b * p.kv_sb + (int64_t)h * p.kv_sh;
  const char* const vb = p.v + (int64_t)b * p.kv_sb + (int64_t)h * p.kv_sh;
  const int end = max(s, e - (p.T - 1 - tok));
  const Reach r = reach_of(s, end, p.window, p.sinks);
  const uint16_t* const q = p.q + (int64_t)b * p.q_sb + (int64_t)tok * p.q_st + (int64_t)hq * p.q_sh;
  float m = -INFINITY, l = 0.f, acc[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i) acc[i] = 0.f;
  for (int p0 = s; p0 < end; p0 += kWave) {
    if (p0 >= s + r.sink && p0 + kWave <= r.lo) {  // between the sinks and the window
      p0 += (r.lo - p0) / kWave * kWave - kWave;
      continue;
    }
    const int pos = p0 + lane;
    float x = -INFINITY;
    if (pos < end && attends(r, s, pos)) {
      const uint16_t* const kr = reinterpret_cast<const uint16_t*>(kb + (int64_t)pos * p.kv_ss);
      float d = 0.f;
      for (int i = 0; i < D; ++i) d = fmaf(bf16_to_f32(q[i]), bf16_to_f32(kr[i]), d);
      x = d * p.scale_log2;
    }
    const float mn = fmaxf(m, wave_max(x)), mu = mn == -INFINITY ? 0.f : mn, alpha = fast_exp2(m - mu);
    m = mn;
    const float t = fast_exp2(x - mu);
    l = l * alpha + wave_sum(t);
    if (l != l) break;  // a score that is NaN or +inf: all of the output is NaN
#pragma unroll
    for (int i = 0; i < DV; ++i) acc[i] *= alpha;
    for (int j = 0; j < min(kWave, end - p0); ++j) {
      if (!attends(r, s, p0 + j)) continue;
      const float tj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(t), j));
      const uint16_t* const vr = reinterpret_cast<const uint16_t*>(vb + (int64_t)(p0 + j) * p.kv_ss);
#pragma unroll
      for (int i = 0; i < DV; ++i) acc[i] = fmaf(tj, bf16_to_f32(vr[DV * lane + i]), acc[i]);
    }
  }
  uint16_t* const o = p.out + (int64_t)b * p.o_sb + (int64_t)tok * p.o_st + (int64_t)hq * p.o_sh;
#pragma unroll
  for (int i = 0; i < DV; ++i) o[DV * lane + i] = f32_to_bf16(l == 0.f ? 0.f : acc[i] / l);
}

// The columns of a wave.
template <int D>
__device__ __forceinline__ void prefill_careful(const LongParams& p, int b, int h, int s, int e, int t0, int ntok, int cg) {
  for (int c = 0; c < kPreWaveCols; ++c) {
    const int m0 = kPreWaveCols * cg + c, tok = t0 + (m0 >> p.gshift);
    if (tok >= t0 + ntok) break;
    careful_column<D>(p, b, h, s, e, tok, (h << p.gshift) + (m0 & (p.G - 1)));
  }
}

// The positions a column tile attends, in steps, and how they are cut: splits of `per` steps, nact of them.
struct PreCut {
  int n, per, nact;
};
template <int TP, int PG>
__device__ __forceinline__ PreCut cut_steps(const PreRange& tr, int splits) {
  const int n = (tr.na + tr.nb + PG - 1) / PG, per = splits == 1 ? max(n, 1) : max((n + splits - 1) / splits, kPreMinSteps);
  return {n, per, max((n + per - 1) / per, 1)};
}

// grid (kv heads, column tiles, rows): workgroups go to the XCDs in turn, so with a multiple of 8 kv heads each head's K and V
// pass through one XCD's L2 alone. The last tiles, which attend most, start first.
// SPLIT: grid (kv heads, column tiles * splits, rows), each workgroup a share of the positions; its sums go to the workspace,
// and window_merge_kernel adds them up.
template <int D, int CG, bool SPLIT>
__global__ void __launch_bounds__(kPreThreads, 2)
    window_prefill_kernel(const int32_t* lens, const int32_t* starts, const LongParams p) {
  constexpr int PG = 4 / CG, TP = PG == 1 ? 64 : 32, NB = TP / 32, NQ = D / 16, ND = D / 32, kCols = CG * kPreWaveCols;
  using L = PreLds<D, TP>;
  const int y = gridDim.y - 1 - blockIdx.y, tile = SPLIT ? y / p.splits : y, split = SPLIT ? y - tile * p.splits : 0;
  const int h = blockIdx.x, b = blockIdx.z;
  const int e_raw = lens[b], s_raw = (starts ? starts : lens)[b];
  const int lane = threadIdx.x % kWave, w = wave_uniform((int)threadIdx.x / kWave), c = lane % 32, half = lane / 32;
  const int cg = w % CG, pg = w / CG;

  const int t0 = tile * (kCols >> p.gshift), ntok = min(kCols >> p.gshift, p.T - t0);
  const int mine = kPreWaveCols * cg + c, tok = t0 + min(mine >> p.gshift, ntok - 1), hq = (h << p.gshift) + (mine & (p.G - 1));

  const float scale = positive_scale(p.scale_log2);
  bf16x8_t qf[NQ];
  {
    const uint16_t* src = p.q + (int64_t)b * p.q_sb + (int64_t)tok * p.q_st + (int64_t)hq * p.q_sh + 8 * half;
#pragma unroll
    for (int j = 0; j < NQ; ++j) qf[j] = signed_q(*reinterpret_cast<const uint4*>(src + 16 * j), p.scale_log2);
  }

  int s, e;
  long_range(e_raw, s_raw, starts != nullptr, p.cap, s, e);
  auto token_end = [&](int t) { return max(s, e - (p.T - 1 - t)); };
  const Reach me = reach_of(s, token_end(tok), p.window, p.sinks);
  const int e1 = token_end(t0 + ntok - 1);
  const PreRange tr = pre_range<TP>(s, token_end(t0), e1, p.window, p.sinks);
  const PreCut cut = cut_steps<TP, PG>(tr, SPLIT ? p.splits : 1);
  const int j0 = SPLIT ? split * cut.per : 0;
  if (SPLIT && split > 0 && j0 >= cut.n) return;
  const int n = SPLIT ? min(cut.per, cut.n - j0) : cut.n;  // steps; position group pg takes tile PG (j0 + j) + pg in step j
  auto of_sinks = [&](int j) { return PG * (j0 + j) + pg < tr.na; };
  auto pos_of = [&](int j) {  // (a tile past the last begins at or past e1: nothing there is attended)
    const int i = PG * (j0 + j) + pg;
    return i < tr.na ? tr.fa + TP * i : tr.fb + TP * (i - tr.na);
  };
  auto last_of = [&](int j) { return (of_sinks(j) ? tr.a1 : e1) - 1; };
  // every column of the wave attends the whole of [whole_lo, whole_end)
  const int whole_end = token_end(t0 + min((kPreWaveCols * cg) >> p.gshift, ntok - 1));
  const int whole_lo = max(s, token_end(t0 + min((kPreWaveCols * cg + kPreWaveCols - 1) >> p.gshift, ntok - 1)) - p.window);

  // arrays of their own, and the tiles' parity known at compile time: the compiler then sees that the reads of one do not
  // depend on the loads in flight to another (it would wait for all of them)
  __shared__ __align__(16) char k_even[PG * L::kBytes], k_odd[PG * L::kBytes], v_even[PG * L::kBytes], v_odd[PG * L::kBytes];
  const int64_t head = (int64_t)b * p.kv_sb + (int64_t)h * p.kv_sh;
  const uint32_t row_bytes = (uint32_t)p.kv_ss;
  const Rsrc rk = span_rsrc(p.k + head, e1 * (int)p.kv_ss), rv = span_rsrc(p.v + head, e1 * (int)p.kv_ss);

  // this lane's LDS addresses: K chunk 2 j + half of row c; V, transposed: the four rows and 16 dims of its group of 16 lanes
  const int group = pg * L::kBytes, k_addr = group + c * L::kRow, k_sw = L::k_swz(c);
  const int l16 = lane % 16, v_row = 4 * half + l16 / 4;
  int v_addr[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
    v_addr[d] = group + v_row * L::kRow + 16 * ((4 * d + 2 * ((lane / 16) % 2) + (l16 % 4) / 2) ^ L::v_swz(v_row)) + 8 * (l16 % 2);

  float m = -INFINITY, l = 0.f;
  f32x16_t acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

  // K operand i of the tile in buf: positions 32 (i % NB) .., contraction step i / NB (the two blocks' products alternate,
  // since one that adds to the product before it waits for it)
  auto k_read = [&](const char* buf, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const bf16x8_t*>(buf + k_addr + 32 * (i % NB) * L::kRow + 16 * ((2 * (i / NB) + half) ^ k_sw));
  };
  // V^T operand d of 16 positions: the lane's 8, in two reads
  auto v_read = [&](const char* buf, int ut, int d) __attribute__((always_inline)) {
    using Tr = __attribute__((address_space(3))) s16x4_lds*;
    const char* const at = buf + v_addr[d] + 16 * ut * L::kRow;
    const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(at)));
    const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(at + 8 * L::kRow)));
    return __builtin_bit_cast(bf16x8_t, make_uint4(a.x, a.y, b.x, b.y));
  };
  constexpr int NK = NB * NQ, PT = 8 * NB / NK, KA = NK < 8 ? NK : 8;  // products of K q, pairs of terms beside each, reads ahead
  // Tile j: its scores x into the running maximum, sum and accumulators, and the scores of tile j + 1 (next; unused after the
  // last). A wave has the matrix unit, the vector unit and LDS at work at once only if its instructions alternate, and an
  // operand read just before its product costs the LDS latency each time: so the first KA K operands are read before the
  // maximum is taken, each product of K q is followed by the read KA products ahead (or of V) and a share of the
  // exponentials, and each product of V p by the read 4 ahead. The scheduling barriers keep that order.
  auto step = [&](auto odd, int j, f32x16_t (&x)[NB], f32x16_t (&next)[NB]) __attribute__((always_inline)) {
    constexpr bool kOdd = decltype(odd)::value;
    const char *const kbuf = kOdd ? k_even : k_odd, *const vbuf = kOdd ? v_odd : v_even;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // this wave's loads of K j + 1 and V j are in LDS
    // everyone's are, and nobody reads K j or V j - 1 any more (a wave with tiles of its own has just used what it read of them)
    if constexpr (CG > 1) __syncthreads();
    bf16x8_t kf[KA], vf[2][ND];
#pragma unroll
    for (int i = 0; i < KA; ++i) kf[i] = k_read(kbuf, i);
    __builtin_amdgcn_sched_barrier(0);
    if (j + 2 < n) stage_tile<D, TP, CG, false>((kOdd ? k_odd : k_even) + group, rk, pos_of(j + 2), last_of(j + 2), row_bytes, cg, lane);
    if (j + 1 < n) stage_tile<D, TP, CG, true>((kOdd ? v_even : v_odd) + group, rv, pos_of(j + 1), last_of(j + 1), row_bytes, cg, lane);
    const int p0 = pos_of(j);
    if (!(p0 + TP <= whole_end && p0 >= whole_lo)) {
      const Reach part{me.lo, of_sinks(j) ? 0 : me.len, me.sink};  // a sinks' tile may end in the window, whose tiles have that
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          x[u][i] = attends(part, s, p0 + 32 * u + 8 * (i / 4) + 4 * half + i % 4) ? x[u][i] : -INFINITY;
    }
    float top = x[0][0];
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, x[u][i]);
    float other = top;
    swap32(top, other);
    top = fmaxf(top, other) * scale;
    // the running maximum moves only when a column's has grown by more than 2^8: until then its terms stay below 2^8, and a
    // term's rounding is relative
    if (__ballot(top > m + 8.f) != 0) {
      const float mn = fmaxf(m, top), mu = mn == -INFINITY ? 0.f : mn, alpha = fast_exp2(m - mu);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[d] *= alpha;
    }
    const float base = m == -INFINITY ? 0.f : m;
    uint32_t pk[NB][8];
    const f32x16_t zero = {};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      next[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i % KA], qf[i / NB], i < NB ? zero : next[i % NB], 0, 0, 0);
      if (i + KA < NK) kf[i % KA] = k_read(kbuf, i + KA);
      else if (i - (NK - KA) < ND) vf[0][i - (NK - KA)] = v_read(vbuf, 0, i - (NK - KA));
#pragma unroll
      for (int g = PT * i; g < PT * (i + 1); ++g) {
        const int u = g / 8, v = 2 * (g % 8);
        pk[u][g % 8] = pack_bf16x2(fast_exp2(fmaf(x[u][v], scale, -base)), fast_exp2(fmaf(x[u][v + 1], scale, -base)));
        l = dot2_bf16(pk[u][g % 8], 0x3f803f80u, l);  // the sum of the rounded terms, the ones that meet V
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int ut = 0; ut < 2 * NB; ++ut) {
      const uint32_t* const q = &pk[ut / 2][4 * (ut % 2)];
      const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, make_uint4(q[0], q[1], q[2], q[3]));
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[ut % 2][d], pf, acc[d], 0, 0, 0);
        if (ut + 1 < 2 * NB) vf[(ut + 1) % 2][d] = v_read(vbuf, ut + 1, d);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  if (n > 0) {
    stage_tile<D, TP, CG, false>(k_even + group, rk, pos_of(0), last_of(0), row_bytes, cg, lane);
    __builtin_amdgcn_s_waitcnt(0x0f70);
    if constexpr (CG > 1) __syncthreads();
    if (n > 1) stage_tile<D, TP, CG, false>(k_odd + group, rk, pos_of(1), last_of(1), row_bytes, cg, lane);
    stage_tile<D, TP, CG, true>(v_even + group, rv, pos_of(0), last_of(0), row_bytes, cg, lane);
    f32x16_t xa[NB], xb[NB];
#pragma unroll
    for (int i = 0; i < NK; ++i)
      xa[i % NB] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_read(k_even, i), qf[i / NB], i < NB ? f32x16_t{} : xa[i % NB], 0, 0, 0);
    for (int j = 0; j < n; j += 2) {
      step(std::false_type{}, j, xa, xb);
      if (j + 1 < n) step(std::true_type{}, j + 1, xb, xa);
    }
  }

  float other = l;
  swap32(l, other);
  l += other;
  if constexpr (PG > 1) {
    // the position groups' accumulators through the tiles' LDS: for PG = 4 groups 2 and 3 to 0 and 1, then (as for PG = 2)
    // group 1 to 0
    __shared__ float s_m[4][kPreWaveCols], s_l[4][kPreWaveCols];
#pragma unroll
    for (int from = PG / 2; from > 0; from /= 2) {
      __syncthreads();  // the tiles, or the round before, have been read
      const bool gives = pg >= from && pg < 2 * from, takes = pg < from;
      const int giver = gives ? w : w + from * CG;  // its wave
      char* const at = (giver % 2 ? k_odd : k_even) + 16 * lane;  // 16 ND registers of a wave: 4 KB ND, half an array's least
      if (gives) {
        if (half == 0) s_m[w][c] = m, s_l[w][c] = l;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<f32x4_t*>(at + 4096 * d + 256 * i) = f32x4_t{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
      }
      __syncthreads();
      if (takes) {
        const float mo = s_m[giver][c], mn = fmaxf(m, mo), mu = mn == -INFINITY ? 0.f : mn;
        const float f0 = fast_exp2(m - mu), f1 = fast_exp2(mo - mu);
        m = mn;
        l = l * f0 + s_l[giver][c] * f1;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f32x4_t y = *reinterpret_cast<const f32x4_t*>(at + 4096 * d + 256 * i);
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[d][i + k] = acc[d][i + k] * f0 + y[k] * f1;
          }
      }
    }
    if (pg > 0) return;
  }
  if (SPLIT && cut.nact > 1) {
    const int64_t part = ((((int64_t)b * p.tiles + tile) * p.NKV + h) * p.splits + split) * kCols + mine;
    if (half == 0) p.part_ml[part] = make_float2(m, l);
    float* const at = p.part_acc + part * D + 4 * half;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<f32x4_t*>(at + 32 * d + 2 * i) = f32x4_t{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float worst = 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) worst += fabsf(acc[d][i]) * 0x1p-8f;
  if (__builtin_expect(__ballot(!(worst < INFINITY) || !(l < INFINITY)) != 0, 0)) {
    prefill_careful<D>(p, b, h, s, e, t0, ntok, cg);
    return;
  }
  if ((mine >> p.gshift) >= ntok) return;
  uint16_t* const o = p.out + (int64_t)b * p.o_sb + (int64_t)tok * p.o_st + (int64_t)hq * p.o_sh + 4 * half;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const uint2 y = make_uint2(pack_bf16x2(acc[d][i] * inv, acc[d][i + 1] * inv), pack_bf16x2(acc[d][i + 2] * inv, acc[d][i + 3] * inv));
      uint16_t* const at = o + 32 * d + 2 * i;
      if (p.out_wide) {
        *reinterpret_cast<uint2*>(at) = y;
      } else {
        at[0] = (uint16_t)y.x, at[1] = (uint16_t)(y.x >> 16), at[2] = (uint16_t)y.y, at[3] = (uint16_t)(y.y >> 16);
      }
    }
}

// Adds up the splits of window_prefill_kernel<D, 4, true> and writes the outputs: a wave a column, grid (columns / 4, kv heads,
// rows).
template <int D>
__global__ void __launch_bounds__(kPreThreads) window_merge_kernel(const int32_t* lens, const int32_t* starts, const LongParams p) {
  constexpr int DV = D / 64, kCols = 4 * kPreWaveCols, TP = 64;
  const int h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x % kWave;
  const int col = wave_uniform((int)(blockIdx.x * (kPreThreads / kWave) + threadIdx.x / kWave));
  const int tok = col >> p.gshift, hq = (h << p.gshift) + (col & (p.G - 1));
  if (tok >= p.T) return;
  int s, e;
  long_range(lens[b], (starts ? starts : lens)[b], starts != nullptr, p.cap, s, e);
  auto token_end = [&](int t) { return max(s, e - (p.T - 1 - t)); };
  const int tile = col / kCols, t0 = tile * (kCols >> p.gshift), last = min(t0 + (kCols >> p.gshift), p.T) - 1;
  const PreCut cut = cut_steps<TP, 1>(pre_range<TP>(s, token_end(t0), token_end(last), p.window, p.sinks), p.splits);
  if (cut.nact == 1) return;  // its one split has written them
  const int64_t part = (((int64_t)b * p.tiles + tile) * p.NKV + h) * p.splits * kCols + col % kCols;
  float m = -INFINITY, l = 0.f, acc[DV] = {};
  for (int k0 = 0; k0 < cut.nact; k0 += 8) {
    float2 ml[8];
    float x[8][DV];
#pragma unroll
    for (int k = 0; k < 8; ++k) {  // past the last: the last again, with no weight
      const int64_t at = part + (int64_t)min(k0 + k, cut.nact - 1) * kCols;
      ml[k] = p.part_ml[at];
#pragma unroll
      for (int i = 0; i < DV; ++i) x[k][i] = p.part_acc[at * D + DV * lane + i];
    }
    float mn = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) mn = fmaxf(mn, ml[k].x);
    const float mu = mn == -INFINITY ? 0.f : mn, alpha = fast_exp2(m - mu);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < DV; ++i) acc[i] *= alpha;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k0 + k >= cut.nact) break;
      const float f = fast_exp2(ml[k].x - mu);
      l = fmaf(f, ml[k].y, l);
#pragma unroll
      for (int i = 0; i < DV; ++i) acc[i] = fmaf(f, x[k][i], acc[i]);
    }
  }
  float worst = fabsf(l) * 0x1p-8f;
#pragma unroll
  for (int i = 0; i < DV; ++i) worst += fabsf(acc[i]) * 0x1p-8f;
  if (__builtin_expect(__ballot(!(worst < INFINITY)) != 0, 0)) {
    careful_column<D>(p, b, h, s, e, tok, hq);
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* const o = p.out + (int64_t)b * p.o_sb + (int64_t)tok * p.o_st + (int64_t)hq * p.o_sh + DV * lane;
#pragma unroll
  for (int i = 0; i < DV; ++i) o[i] = f32_to_bf16(acc[i] * inv);
}

}  // namespace
