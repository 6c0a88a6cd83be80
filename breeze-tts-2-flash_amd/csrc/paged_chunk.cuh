// Device code of bz_gqa_paged (include/bz_paged_cache.h) for rows of many new tokens.
//
// The (token, q head) pairs of one kv head are the columns of two products, 128 a workgroup and 32 a wave: 128 / G tokens of a row
// times its G heads. A workgroup walks the positions its tokens attend in steps staged in LDS, two buffers each of K and V, as
// window_prefill.cuh does: S^T = K Q^T (mfma 32x32x16), the softmax within a lane but for one swap, O^T += V^T P^T with V^T by
// ds_read_b64_tr_b16 and each term rounded to one bf16. What differs is where a step's rows come from: they are staged in blocks of 16,
// each in one page (block and page are powers of two). With four column groups (4 x 1) a step is BL = 4 blocks, of which each wave stages
// one for all four waves; with 2 x 2 and 1 x 4 a tile is BL = 2 blocks, of which a wave stages one (for two waves) or both (for itself
// alone, maybe from two pages, and without a barrier). The page numbers of 64 / BL steps are held one a lane. bf16 rows go from memory to
// LDS directly; rows of 8 bits through registers, a step earlier, where they become bf16 with their scale (exactly).
//
// One term of bf16 (at most 2^-8 of itself; the sum is of the rounded terms, so the weights add up to 1) adds 2 to 3% to the error against
// 64 bits (0.00163 to 0.00165 .. 0.00168 of the output's norm, most of which is the output's own rounding). Two terms, as rows of few
// tokens have, take half as many products again and registers that are not there (us, one / two, 16 q and 8 kv heads of 128 dims: 2048
// tokens alone 36 / 42, 8192 275 / 404, 8192 of 8 bits 303 / 620, 512 behind 15872 of 8 bits 88.5 / 214, 256 behind 8192 36.7 / 46.7;
// head_dim 64, 1500 of 8 and 4 heads 12.6 / 14.4).
//
// Rows differ in length and in tokens, so the work is dealt on the device (deal_paged): every (column tile, split) about as many
// steps. The sums of a tile that is split go through the workspace, and paged_merge_kernel adds them up.
#pragma once

#include "paged_split.cuh"
#include "window_prefill.cuh"

namespace {

constexpr int kChunkCols = 128, kChunkStep = 64;

// One column, by one wave, in fp32 and without any product of a position that the column does not attend (careful_column's case).
template <int D, bool F8>
__device__ __forceinline__ void paged_careful(const PagedParams& p, int h, int row, int token, int hq, int end) {
  constexpr int DV = D / 64;
  const int lane = threadIdx.x % kWave;
  const uint16_t* const q = p.q + (int64_t)token * p.q_st + (int64_t)hq * p.q_sh;
  // the value of dim i at place `at` of a page
  auto value = [&](const char* kv, const uint8_t* scales, int page, int at, int i) {
    const char* const src = kv + page * p.kv_sp + h * p.kv_sh + (int64_t)at * p.kv_ss;
    if constexpr (F8) {
      const uint32_t e = scales[page * p.sc_sp + h * p.sc_sh + at];
      return bf16_lo(bz::f8_pair<false>((uint32_t)(uint8_t)src[i], e));
    } else {
      return bf16_to_f32(reinterpret_cast<const uint16_t*>(src)[i]);
    }
  };
  const int pmask = (1 << p.rows.pshift) - 1;
  float m = -INFINITY, l = 0.f, acc[DV] = {};
  for (int p0 = 0; p0 < end; p0 += kWave) {
    const int pos = p0 + lane, page = pos < end ? bz::page_of(p.rows, row, pos) : -1;
    float x = -INFINITY;
    if (page >= 0) {
      float d = 0.f;
      for (int i = 0; i < D; ++i) d = fmaf(bf16_to_f32(q[i]), value(p.k, p.ks, page, pos & pmask, i), d);
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
      const int pj = __builtin_amdgcn_readlane(page, j);
      if (pj < 0) continue;
      const float tj = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(t), j));
#pragma unroll
      for (int i = 0; i < DV; ++i) acc[i] = fmaf(tj, value(p.v, p.vs, pj, (p0 + j) & pmask, DV * lane + i), acc[i]);
    }
  }
  uint16_t* const o = p.out + (int64_t)token * p.o_st + (int64_t)hq * p.o_sh;
#pragma unroll
  for (int i = 0; i < DV; ++i) o[DV * lane + i] = f32_to_bf16(l == 0.f ? 0.f : acc[i] / l);
}

// LDS of one tile of K or V: TP rows of D bf16, in 16-byte chunks. Chunk c of row r lies in slot c ^ swizzle(r): the 16 lanes of a cycle of
// a K read take the same chunk of 16 rows, the 32 of a transposing V read four chunks each of four rows, and either way they fall
// into all 64 banks, as do the 16 lanes that write rows of 8 bits, four rows of the same chunks in each quarter (with V swizzled for
// reads of 16 lanes, as window_prefill.cuh does, a third of the LDS cycles were conflicts).
template <int D, int TP>
struct ChunkLds {
  static constexpr int kRow = 2 * D, kBytes = TP * kRow;
  static __device__ __forceinline__ int k_swz(int r) { return r & (D / 8 - 1); }
  static __device__ __forceinline__ int v_swz(int r) { return D == 128 ? 5 * (r & 3) : 5 * ((r >> 1) & 1); }
};

// How a column tile of n steps is cut: `per` steps a split, nact of them.
struct ChunkCut {
  int per, nact;
};
__device__ __forceinline__ ChunkCut cut_chunk(int n, int k) {
  const int per = k <= 1 ? max(n, 1) : max((n + k - 1) / k, kPreMinSteps);
  return {per, max((n + per - 1) / per, 1)};
}

// 16 rows of 8-bit codes on their way to LDS: lane l holds the D / 4 dims from (D / 4) (l % 4) on of row l / 4, and its scale.
template <int D>
struct F8Rows {
  uint2 c[D / 32];
  uint32_t e;
};

// Grid (p.slots + few.slots) * kv heads, a slot's heads side by side (workgroups go to the XCDs in turn, so with a multiple of 8 kv heads each
// head's K and V pass through one XCD's L2 alone). p.slots are the chunks'; the others, behind them or (few_first) ahead, do the split
// kernel's work on rows of few tokens, with the parameters `few`: in a launch of its own that work began when the last chunk had ended.
// CG column groups, one a wave, times PG = 4 / CG position groups: 4 x 1 in steps of 64; with 2 x 2 and 1 x 4 a small chunk has
// more workgroups and fewer steps, each position group taking every PG-th tile of 32, and the groups' accumulators meet in LDS. Only
// 4 x 1 is split.
//
// Matrix and vector instructions of two waves a SIMD, which overlap in part, bound it: 8192 tokens alone, 16 q and 8 kv heads, head_dim
// 128, 281 us, 978 TFLOP/s, matrix units busy 45%, vector units 44%; 512 tokens behind 16384 of 8 bits 79 us and 11 of merge, 860 TFLOP/s.
template <int D, bool F8, int CG>
__global__ void __launch_bounds__(kPreThreads, 2) paged_chunk_kernel(const PagedParams p, const PagedParams few, const int few_first) {
  constexpr int PG = 4 / CG, TP = PG == 1 ? kChunkStep : 32, NB = TP / 32, NQ = D / 16, ND = D / 32, COLS = CG * kPreWaveCols;
  constexpr int BL = TP / 16, UB = BL / CG;         // blocks of 16 positions of a tile, and those that a wave stages
  constexpr int WS = kWave / BL;                    // steps whose pages a wave holds
  using L = ChunkLds<D, TP>;
  static_assert(split_floats<D, 1>() * 4 <= PG * L::kBytes, "the rows of few tokens use the same LDS");
  // arrays of their own, and the steps' parity known at compile time: the compiler then sees that the reads of one do not
  // depend on the loads in flight to another (it would wait for all of them)
  __shared__ __align__(16) char k_even[PG * L::kBytes], k_odd[PG * L::kBytes], v_even[PG * L::kBytes], v_odd[PG * L::kBytes];
  int at = (int)(blockIdx.x / (uint32_t)p.NKV);
  const int h = (int)blockIdx.x - at * p.NKV, before = few_first ? few.slots : 0;
  if (few_first ? at < before : at >= p.slots) {
    paged_split<D, F8, true, 1, kPreThreads>(few, few_first ? at : at - p.slots, h, [&](int u) {
      return reinterpret_cast<float*>(u == 0 ? k_even : u == 1 ? k_odd : u == 2 ? v_even : v_odd);
    });
    return;
  }
  at -= before;
  const PagedShare share = deal_paged<true, false, kChunkStep, 1>(p, COLS, at);
  if (share.b < 0) return;
  const PagedRow& row = share.row;
  const int lane = threadIdx.x % kWave, w = wave_uniform((int)threadIdx.x / kWave), c = lane % 32, half = lane / 32;
  const int cg = PG == 1 ? w : w % CG, pg = PG == 1 ? 0 : w / CG;
  const int tpt = COLS >> p.gshift, tiles = (row.T + tpt - 1) / tpt, tile = tiles - 1 - share.tile;  // the longest first
  const int t0 = tile * tpt, ntok = min(tpt, row.T - t0);
  const int mine = kPreWaveCols * cg + c, tok = t0 + min(mine >> p.gshift, ntok - 1), hq = (h << p.gshift) + (mine & (p.G - 1));

  const float scale = positive_scale(p.scale_log2);
  auto token_end = [&](int t) { return paged_end(p.rows, row, t); };
  const int my_end = token_end(tok), e1 = wave_uniform(token_end(t0 + ntok - 1)), last = e1 - 1;
  const int whole_end = wave_uniform(token_end(t0 + min((kPreWaveCols * cg) >> p.gshift, ntok - 1)));  // of the wave's columns
  const int steps = (e1 + TP * PG - 1) / (TP * PG);
  const ChunkCut cut = cut_chunk(steps, PG == 1 ? share.k : 1);
  const int j0 = PG == 1 ? share.split * cut.per : 0;
  if (PG == 1 && share.split > 0 && j0 >= steps) return;
  const int n = min(cut.per, steps - j0);  // steps of this split
  auto pos_of = [&](int j) { return TP * (PG * (j0 + j) + pg); };

  const int64_t khead = (int64_t)h * p.kv_sh, shead = (int64_t)h * p.sc_sh;
  const int pshift = p.rows.pshift, pmask = (1 << pshift) - 1;
  const Rsrc table = span_rsrc(p.rows.table + share.b * p.rows.table_st, p.rows.max_pages * 4);

  // Lane i holds the page of block i of 16 positions, of the 64 blocks (WS steps) of this wave's tiles at hand: that of the block's
  // first position, or of the last attended one where the block lies behind it. odd: the blocks without one (-1); they are staged
  // as zeros, through a span of no bytes, and attended by nobody (read from some page instead, a NaN there would send every column to
  // paged_careful: 300 tokens behind 700 of 64 heads, a hole and page 0 not yet written, 6414 us in place of 24.5).
  int ids = 0;
  uint64_t odd = 0;
  auto fetch = [&](int j) __attribute__((always_inline)) {
    ids = page_ids(table, p.rows.max_pages, min(pos_of(j + lane / BL) + 16 * (lane % BL), max(last, 0)) >> pshift);
  };
  auto settle = [&]() __attribute__((always_inline)) {
    const bool there = (uint32_t)ids < (uint32_t)p.rows.pages;
    odd = __ballot(!there);
    ids = there ? ids : -1;
  };
  struct Pages {
    int id[UB];  // of the blocks that this wave stages
  };
  auto page_at = [&](int j) __attribute__((always_inline)) {
    Pages x;
#pragma unroll
    for (int u = 0; u < UB; ++u) x.id[u] = __builtin_amdgcn_readlane(ids, BL * (j & (WS - 1)) + cg * UB + u);
    return x;
  };
  auto odd_at = [&](int j) __attribute__((always_inline)) { return (uint32_t)(odd >> (BL * (j & (WS - 1)))) & ((1u << BL) - 1); };
  // the place in its page of position x, behind the last attended one that one's
  auto place = [&](int x) __attribute__((always_inline)) { return min(x, last) & pmask; };

  // This wave's rows of step j of K or V into LDS. 64 lanes write 1 KB in lane order, so the swizzle is in which chunk each fetches.
  const int group = pg * L::kBytes;
  auto stage = [&](auto isv, char* buf, int j, const Pages& pages) __attribute__((always_inline)) {
    constexpr bool V = decltype(isv)::value;
    constexpr int RPI = 1024 / L::kRow, CH = D / 8;  // rows an instruction, chunks a row
    const int p0 = pos_of(j);
#pragma unroll
    for (int b = 0; b < UB; ++b) {
      const Rsrc rsrc = span_rsrc((V ? p.v : p.k) + max(pages.id[b], 0) * p.kv_sp + khead, pages.id[b] < 0 ? 0 : p.page_bytes);
#pragma unroll
      for (int u = 0; u < 16 / RPI; ++u) {
        const int row0 = 16 * (cg * UB + b) + RPI * u, rw = row0 + lane / CH, ch = lane % CH;
        const uint32_t off = (uint32_t)place(p0 + rw) * p.kv_ss + 16 * (ch ^ (V ? L::v_swz(rw) : L::k_swz(rw)));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(buf + group + row0 * L::kRow), 16, off,
                                                 0, 0, 0);
      }
    }
  };
  auto load8 = [&](auto isv, F8Rows<D> (&x)[UB], int j, const Pages& pages) __attribute__((always_inline)) {
    constexpr bool V = decltype(isv)::value;
#pragma unroll
    for (int b = 0; b < UB; ++b) {
      const int64_t page = max(pages.id[b], 0);
      const bool there = pages.id[b] >= 0;
      const Rsrc rsrc = span_rsrc((V ? p.v : p.k) + page * p.kv_sp + khead, there ? p.page_bytes : 0);
      const Rsrc rs = span_rsrc((V ? p.vs : p.ks) + page * p.sc_sp + shead, there ? pmask + 1 : 0);
      const int at = place(pos_of(j) + 16 * (cg * UB + b) + lane / 4);
#pragma unroll
      for (int i = 0; i < D / 32; i += 2) {
        const uint4 y = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(
                                                      rsrc, (uint32_t)at * p.kv_ss + (D / 4) * (lane % 4) + 8 * i, 0, 0));
        x[b].c[i] = make_uint2(y.x, y.y), x[b].c[i + 1] = make_uint2(y.z, y.w);
      }
      x[b].e = __builtin_amdgcn_raw_buffer_load_b8(rs, at, 0, 0);
    }
  };
  auto put8 = [&](auto isv, char* buf, const F8Rows<D> (&x)[UB]) __attribute__((always_inline)) {
    constexpr bool V = decltype(isv)::value;
#pragma unroll
    for (int b = 0; b < UB; ++b) {
      const int rw = 16 * (cg * UB + b) + lane / 4, swz = V ? L::v_swz(rw) : L::k_swz(rw);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const int ch = (D / 32) * (lane % 4) + i;
        *reinterpret_cast<uint4*>(buf + group + rw * L::kRow + 16 * (ch ^ swz)) = bz::f8_values(x[b].c[i], x[b].e);
      }
    }
  };
  constexpr std::false_type isk{};
  constexpr std::true_type isv{};

  // this lane's LDS addresses: K chunk 2 j + half of row c; V, transposed: the four rows and 16 dims of its group of 16 lanes
  const int k_addr = group + c * L::kRow, k_sw = L::k_swz(c), l16 = lane % 16, v_row = 4 * half + l16 / 4;
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

  auto k_read = [&](const char* buf, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const bf16x8_t*>(buf + k_addr + 32 * (i % NB) * L::kRow + 16 * ((2 * (i / NB) + half) ^ k_sw));
  };
  auto v_read = [&](const char* buf, int ut, int d) __attribute__((always_inline)) {
    using Tr = __attribute__((address_space(3))) s16x4_lds*;
    const char* const src = buf + v_addr[d] + 16 * ut * L::kRow;
    const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(src)));
    const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(src + 8 * L::kRow)));
    return __builtin_bit_cast(bf16x8_t, make_uint4(a.x, a.y, b.x, b.y));
  };

  // In step j K of step j + AHEAD is asked for and V of the step before that: bf16 straight into LDS, where the next steps read
  // them; 8 bits into kr and vr, which go to LDS one step later. vpage: the page of that V. holes: the blocks without a page of
  // the steps from j on, BL bits each.
  constexpr int AHEAD = F8 ? 3 : 2;
  Pages vpage{};
  uint32_t holes = 0;
  bf16x8_t qf[NQ];
  F8Rows<D> kr[UB], vr[UB];
  // products of K q, pairs of terms beside each, reads ahead (8 bits, D 128: fewer, for the registers)
  constexpr int NK = NB * NQ, PT = 8 * NB / NK, AH = F8 && D == 128 && CG == 4 ? 4 : 8, KA = NK < AH ? NK : AH;

  // Step j: its scores x into the running maximum, sum and accumulators, and the scores of step j + 1 (next; unused after the
  // last), in window_prefill_kernel's order.
  auto step = [&](auto odd_step, int j, f32x16_t (&x)[NB], f32x16_t (&next)[NB]) __attribute__((always_inline)) {
    constexpr bool kOdd = decltype(odd_step)::value;
    const char *const kbuf = kOdd ? k_even : k_odd, *const vbuf = kOdd ? v_odd : v_even;
    char *const knew = kOdd ? k_odd : k_even, *const vnew = kOdd ? v_even : v_odd;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // this wave's loads have arrived: of K j + 1 and V j, or (8 bits) of K j + 2 and V j + 1
    // K j + 1 and V j are in LDS, and nobody reads K j or V j - 1 any more (a wave with tiles of its own has just used what it read)
    if constexpr (CG > 1) __syncthreads();
    else asm volatile("" ::: "memory");
    bf16x8_t kf[KA], vf[2][ND];
#pragma unroll
    for (int i = 0; i < KA; ++i) kf[i] = k_read(kbuf, i);
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t hole = holes & ((1u << BL) - 1);
    holes >>= BL;
    const int jk = j + AHEAD;
    if ((jk & (WS - 1)) == 0 && jk < n) settle();
    if constexpr (F8) {
      if (j + 2 < n) put8(isk, knew, kr);
      if (j + 1 < n) put8(isv, vnew, vr);
    }
    Pages kpage{};
    if (jk < n) {
      kpage = page_at(jk);
      holes |= odd_at(jk) << (BL * (AHEAD - 1));
      if constexpr (F8) load8(isk, kr, jk, kpage);
      else stage(isk, knew, jk, kpage);
    }
    if (jk - 1 < n) {
      if constexpr (F8) load8(isv, vr, jk - 1, vpage);
      else stage(isv, vnew, jk - 1, vpage);
    }
    vpage = kpage;
    if ((jk & (WS - 1)) == WS - 1 && jk + 1 < n) fetch(jk + 1);  // (there with the next step's wait)
    const int p0 = pos_of(j);
    if (p0 + TP > whole_end || hole != 0) {
#pragma unroll
      for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          x[u][i] = p0 + 32 * u + 8 * (i / 4) + 4 * half + i % 4 < my_end && !(hole >> (2 * u + i / 8) & 1u) ? x[u][i] : -INFINITY;
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
    // the table's entries, q and the first tiles are asked for one behind the other, and waited for as they are needed
    fetch(0);
    uint4 qr[NQ];
    {
      const uint16_t* src = p.q + (int64_t)(row.q0 + tok) * p.q_st + (int64_t)hq * p.q_sh + 8 * half;
#pragma unroll
      for (int j = 0; j < NQ; ++j) qr[j] = *reinterpret_cast<const uint4*>(src + 16 * j);
    }
    settle();
    const Pages page0 = page_at(0), page1 = page_at(1);  // (behind the last step: any page, unused)
    holes = odd_at(0) | odd_at(1) << BL;
    f32x16_t xa[NB], xb[NB];
    if constexpr (F8) {
      F8Rows<D> k0[UB];
      load8(isk, k0, 0, page0);
      if (n > 1) load8(isk, kr, 1, page1);
      load8(isv, vr, 0, page0);
      put8(isk, k_even, k0);
      if (n > 1) put8(isk, k_odd, kr);
      put8(isv, v_even, vr);
      vpage = page_at(2);
      holes |= odd_at(2) << (2 * BL);
      if (n > 2) load8(isk, kr, 2, vpage);
      if (n > 1) load8(isv, vr, 1, page1);
    } else {
      constexpr int LOADS = UB * 16 * L::kRow / 1024;  // of a wave for a tile
      auto all_but = [](int n) { return 0x0f70 | (n & 15) | (n >> 4) << 14; };
      stage(isk, k_even, 0, page0);
      if (n > 1) stage(isk, k_odd, 1, page1);
      stage(isv, v_even, 0, page0);
      vpage = page1;
      if (n > 1) __builtin_amdgcn_s_waitcnt(all_but(2 * LOADS));  // q and K 0 are there
      else __builtin_amdgcn_s_waitcnt(all_but(LOADS));
    }
    if constexpr (CG > 1) __syncthreads();
    else asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < NQ; ++j) qf[j] = signed_q(qr[j], p.scale_log2);
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
      char* const to = (giver % 2 ? k_odd : k_even) + 16 * lane;  // 16 ND registers of a wave: 4 KB ND, half an array's least
      if (gives) {
        if (half == 0) s_m[w][c] = m, s_l[w][c] = l;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<f32x4_t*>(to + 4096 * d + 256 * i) = f32x4_t{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
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
            const f32x4_t y = *reinterpret_cast<const f32x4_t*>(to + 4096 * d + 256 * i);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[d][i + q] = acc[d][i + q] * f0 + y[q] * f1;
          }
      }
    }
    if (pg > 0) return;
  }
  if (PG == 1 && cut.nact > 1) {
    const int64_t part = ((int64_t)h * p.part_slots + share.first + share.split) * kChunkCols + mine;
    if (half == 0) p.part_ml[part] = make_float2(m, l);
    float* const to = p.part_acc + part * D + 4 * half;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<f32x4_t*>(to + 32 * d + 2 * i) = f32x4_t{acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float worst = 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) worst += fabsf(acc[d][i]) * 0x1p-8f;
  if (__builtin_expect(__ballot(!(worst < INFINITY) || !(l < INFINITY)) != 0, 0)) {
    for (int i = 0; i < kPreWaveCols; ++i) {
      const int col = kPreWaveCols * cg + i, t = t0 + (col >> p.gshift);
      if (t >= t0 + ntok) break;
      paged_careful<D, F8>(p, h, share.b, row.q0 + t, (h << p.gshift) + (col & (p.G - 1)), wave_uniform(token_end(t)));
    }
    return;
  }
  if ((mine >> p.gshift) >= ntok) return;
  uint16_t* const o = p.out + (int64_t)(row.q0 + tok) * p.o_st + (int64_t)hq * p.o_sh + 4 * half;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const uint2 y = make_uint2(pack_bf16x2(acc[d][i] * inv, acc[d][i + 1] * inv), pack_bf16x2(acc[d][i + 2] * inv, acc[d][i + 3] * inv));
      uint16_t* const to = o + 32 * d + 2 * i;
      if (p.out_wide) {
        *reinterpret_cast<uint2*>(to) = y;
      } else {
        to[0] = (uint16_t)y.x, to[1] = (uint16_t)(y.x >> 16), to[2] = (uint16_t)y.y, to[3] = (uint16_t)(y.y >> 16);
      }
    }
}

// Adds up the splits of paged_chunk_kernel's tiles and writes their outputs, four dims a lane. Grid column tiles * kv heads * (128 /
// p.merge_cols), a tile's heads side by side.
template <int D, bool F8>
__global__ void __launch_bounds__(kPreThreads) paged_merge_kernel(const PagedParams p) {
  constexpr int LPC = D / 4, CPW = kWave / LPC;  // lanes a column, columns a wave at a time
  const int groups = kChunkCols / p.merge_cols;
  const int u = (int)(blockIdx.x / (uint32_t)(p.NKV * groups)), rest = (int)blockIdx.x - u * p.NKV * groups;
  const int h = rest / groups, c0 = p.merge_cols * (rest - h * groups);
  const PagedShare share = deal_paged<true, true, kChunkStep, 1>(p, kChunkCols, u);
  if (share.b < 0 || share.k <= 1) return;
  const PagedRow& row = share.row;
  const int lane = threadIdx.x % kWave, w = wave_uniform((int)threadIdx.x / kWave);
  const int tpt = kChunkCols >> p.gshift, tiles = (row.T + tpt - 1) / tpt, tile = tiles - 1 - share.tile;
  const int t0 = tile * tpt, ntok = min(tpt, row.T - t0);
  const ChunkCut cut = cut_chunk((paged_end(p.rows, row, t0 + ntok - 1) + kChunkStep - 1) / kChunkStep, share.k);
  if (cut.nact == 1) return;  // its one split has written them
  const int64_t slot = (int64_t)h * p.part_slots + share.first;
  for (int c1 = c0 + CPW * w; c1 < c0 + p.merge_cols; c1 += CPW * (kPreThreads / kWave)) {
    const int col = c1 + lane / LPC, d = 4 * (lane % LPC);
    if ((c1 >> p.gshift) >= ntok) return;  // (uniform: a wave's columns lie side by side)
    float m = -INFINITY, l = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < cut.nact; k0 += 8) {
      float2 ml[8];
      f32x4_t x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // past the last: the last again, with no weight
        const int64_t at = (slot + min(k0 + k, cut.nact - 1)) * kChunkCols + col;
        ml[k] = p.part_ml[at];
        x[k] = *reinterpret_cast<const f32x4_t*>(p.part_acc + at * D + d);
      }
      float mn = m;
#pragma unroll
      for (int k = 0; k < 8; ++k) mn = fmaxf(mn, ml[k].x);
      const float mu = mn == -INFINITY ? 0.f : mn, alpha = fast_exp2(m - mu);
      m = mn;
      l *= alpha;
      acc *= alpha;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k0 + k >= cut.nact) break;
        const float f = fast_exp2(ml[k].x - mu);
        l = fmaf(f, ml[k].y, l);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = fmaf(f, x[k][i], acc[i]);
      }
    }
    float worst = fabsf(l) * 0x1p-8f;
#pragma unroll
    for (int i = 0; i < 4; ++i) worst += fabsf(acc[i]) * 0x1p-8f;
    const bool mine = col < kChunkCols && (col >> p.gshift) < ntok;
    const uint64_t off = __ballot(mine && !(worst < INFINITY));
    if (__builtin_expect(off != 0, 0)) {
      for (int i = 0; i < CPW; ++i) {
        const int cc = c1 + i, t = t0 + (cc >> p.gshift);
        if (!(off >> (LPC * i) & (LPC == 64 ? ~0ull : (1ull << LPC) - 1))) continue;
        paged_careful<D, F8>(p, h, share.b, row.q0 + t, (h << p.gshift) + (cc & (p.G - 1)), wave_uniform(paged_end(p.rows, row, t)));
      }
    }
    if (!mine || (off >> (lane / LPC * LPC) & ((1ull << LPC) - 1))) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* const o = p.out + (int64_t)(row.q0 + t0 + (col >> p.gshift)) * p.o_st + (int64_t)((h << p.gshift) + (col & (p.G - 1))) * p.o_sh + d;
    const uint2 y = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
    if (p.out_wide) {
      *reinterpret_cast<uint2*>(o) = y;
    } else {
      o[0] = (uint16_t)y.x, o[1] = (uint16_t)(y.x >> 16), o[2] = (uint16_t)y.y, o[3] = (uint16_t)(y.y >> 16);
    }
  }
}

}  // namespace
