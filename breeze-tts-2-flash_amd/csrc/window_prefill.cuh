// Device code of bz_gqa_window over a chunk of many query tokens (include/bz_long_cache.h).
//
// A workgroup of four waves takes 128 columns: (token, q head) pairs of one kv head, 128 / G tokens of a row times its G
// heads, 32 a wave, so K and V are fetched once for the whole group. It walks the positions any of its tokens attends (the
// sinks' tiles, then the window's; tile_range) in tiles of 64 staged in LDS, two buffers each of K and V, the next loads in
// flight while a tile is worked on.
//   S^T = K Q^T   mfma 32x32x16: A = K rows, B = Q^T (registers, loaded once). A lane then holds 32 scores of one column, the
//                 rows 8 (v / 4) + 4 half + v % 4 of each block of 32 positions, so the softmax is within a lane but for one
//                 swap with lane ^ 32.
//   O^T += V^T P^T: the same 32 scores, as terms rounded to bf16, are the B operand as they stand when the contraction takes
//                 the positions in the order 16 s + 8 a + 4 half + i; A = V^T by ds_read_b64_tr_b16 (four rows of 16 dims,
//                 transposed on the way), which reads them in that order.
// The terms are rounded to one bf16 each (sums are fp32): 2^-9 rms of each term, about as much again as the output's own
// rounding; a second term would cost half as many products again, and here the products are the bound.
#pragma once

#include "long_cache.cuh"

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short s16x4_lds __attribute__((ext_vector_type(4)));

constexpr int kPreThreads = 256, kPreCols = 128, kPreTile = 64, kPreRows = kPreTile / 4;

// LDS of one buffer: K, then V, 64 rows of D bf16 each, in 16-byte chunks. Chunk c of row r lies in slot c ^ swizzle(r), so
// that the lanes of one read, which take the same chunk of different rows, fall into different banks.
template <int D>
struct PreLds {
  static constexpr int kRow = 2 * D, kBytes = kPreTile * kRow;
  static __device__ __forceinline__ int k_swz(int r) { return r & (D / 8 - 1); }
  static __device__ __forceinline__ int v_swz(int r) { return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); }
};

// Loads the 64 rows from pos0 on (clamped to `last`: a row past it holds a copy of that one, and no column attends it) into
// LDS at base: 64 lanes write 1 KB in lane order, so the swizzle is in which chunk each lane fetches.
template <int D, bool V>
__device__ __forceinline__ void stage_tile(char* base, const Rsrc& rsrc, int pos0, int last, uint32_t row_bytes, int w, int lane) {
  using L = PreLds<D>;
  constexpr int RPI = 1024 / L::kRow, CH = D / 8;  // rows an instruction, chunks a row
#pragma unroll
  for (int u = 0; u < kPreRows / RPI; ++u) {
    const int row = kPreRows * w + RPI * u + lane / CH, c = lane % CH;
    const uint32_t off = (uint32_t)min(pos0 + row, last) * row_bytes + 16 * (c ^ (V ? L::v_swz(row) : L::k_swz(row)));
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rsrc, (__attribute__((address_space(3))) void*)(base + (kPreRows * w + RPI * u) * L::kRow), 16, off, 0, 0, 0);
  }
}

// One column at a time, in fp32 and without any product of a position that the column does not attend: for a wave whose
// result is not finite, which is right where the column attends an infinity or NaN and wrong where a tile held one that it
// does not (0 times it). The lanes score 64 positions, then each accumulates D / 64 dims over them.
template <int D>
__device__ __forceinline__ void prefill_careful(const LongParams& p, int b, int h, int s, int e, int t0, int ntok, int w) {
  constexpr int DV = D / 64;
  const int lane = threadIdx.x % kWave;
  const char* const kb = p.k + (int64_t)b * p.kv_sb + (int64_t)h * p.kv_sh;
  const char* const vb = p.v + (int64_t)b * p.kv_sb + (int64_t)h * p.kv_sh;
  for (int c = 0; c < 32; ++c) {
    const int m0 = 32 * w + c, tok = t0 + (m0 >> p.gshift), hq = (h << p.gshift) + (m0 & (p.G - 1));
    if (tok >= t0 + ntok) break;
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
}

// grid (kv heads, column tiles, rows): workgroups go to the XCDs in turn, so with a multiple of 8 kv heads each head's K and V
// pass through one XCD's L2 alone. The last tiles, which attend most, start first.
template <int D>
__global__ void __launch_bounds__(kPreThreads, 2)
    window_prefill_kernel(const int32_t* lens, const int32_t* starts, const LongParams p) {
  using L = PreLds<D>;
  constexpr int NQ = D / 16, ND = D / 32;
  const int h = blockIdx.x, tile = gridDim.y - 1 - blockIdx.y, b = blockIdx.z;
  const int e_raw = lens[b], s_raw = (starts ? starts : lens)[b];
  const int lane = threadIdx.x % kWave, w = wave_uniform((int)threadIdx.x / kWave), c = lane % 32, half = lane / 32;

  const int t0 = tile * (kPreCols >> p.gshift), ntok = min(kPreCols >> p.gshift, p.T - t0);
  const int mine = 32 * w + c, tok = t0 + min(mine >> p.gshift, ntok - 1), hq = (h << p.gshift) + (mine & (p.G - 1));

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
  const TileRange tr = tile_range<kPreTile>(s, token_end(t0), e1, p.window, p.sinks);
  const int n = tr.na + tr.nb;
  auto pos_of = [&](int j) { return j < tr.na ? tr.fa + kPreTile * j : tr.fb + kPreTile * (j - tr.na); };
  // of this wave's tokens: the first one's end, and the last one's window start and end
  const int wt0 = t0 + min((32 * w) >> p.gshift, ntok - 1), wt1 = t0 + min((32 * w + 31) >> p.gshift, ntok - 1);
  const int we0 = token_end(wt0), we1 = token_end(wt1);
  const int wlo1 = max(s, we1 - p.window);

  // arrays of their own, and the tiles' parity known at compile time: the compiler then sees that the reads of one do not
  // depend on the loads in flight to another (it would wait for all of them)
  __shared__ __align__(16) char k_even[L::kBytes], k_odd[L::kBytes], v_even[L::kBytes], v_odd[L::kBytes];
  const int64_t head = (int64_t)b * p.kv_sb + (int64_t)h * p.kv_sh;
  const uint32_t row_bytes = (uint32_t)p.kv_ss;
  const Rsrc rk = span_rsrc(p.k + head, e1 * (int)p.kv_ss), rv = span_rsrc(p.v + head, e1 * (int)p.kv_ss);

  // this lane's LDS addresses: K chunk 2 j + half of row c; V, transposed: the four rows and 16 dims of its group of 16 lanes
  const int k_addr = c * L::kRow, k_sw = L::k_swz(c);
  const int l16 = lane % 16, v_row = 4 * half + l16 / 4;
  int v_addr[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
    v_addr[d] = v_row * L::kRow + 16 * ((4 * d + 2 * ((lane / 16) % 2) + (l16 % 4) / 2) ^ L::v_swz(v_row)) + 8 * (l16 % 2);

  float m = -INFINITY, l = 0.f;
  f32x16_t acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

  // K operand i of the tile in buf: positions 32 (i % 2) .., contraction step i / 2 (the two blocks' products alternate, since
  // one that adds to the product before it waits for it)
  auto k_read = [&](const char* buf, int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const bf16x8_t*>(buf + k_addr + 32 * (i % 2) * L::kRow + 16 * ((2 * (i / 2) + half) ^ k_sw));
  };
  // V^T operand d of 16 positions: the lane's 8, in two reads
  auto v_read = [&](const char* buf, int ut, int d) __attribute__((always_inline)) {
    using Tr = __attribute__((address_space(3))) s16x4_lds*;
    const char* const at = buf + v_addr[d] + 16 * ut * L::kRow;
    const uint2 a = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(at)));
    const uint2 b = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(at + 8 * L::kRow)));
    return __builtin_bit_cast(bf16x8_t, make_uint4(a.x, a.y, b.x, b.y));
  };
  constexpr int NK = 2 * NQ, PG = 16 / NK;  // products of K q, and pairs of terms worked out beside each
  // Tile j: its scores x into the running maximum, sum and accumulators, and the scores of tile j + 1 (next; unused after the
  // last). A wave has the matrix unit, the vector unit and LDS at work at once only if its instructions alternate, and an
  // operand read just before its product costs the LDS latency each time: so the first 8 K operands are read before the
  // maximum is taken, each product of K q is followed by the read 8 products ahead (or of V) and a share of the
  // exponentials, and each product of V p by the read 4 ahead. The scheduling barriers keep that order.
  auto step = [&](auto odd, int j, f32x16_t (&x)[2], f32x16_t (&next)[2]) __attribute__((always_inline)) {
    constexpr bool kOdd = decltype(odd)::value;
    const char *const kbuf = kOdd ? k_even : k_odd, *const vbuf = kOdd ? v_odd : v_even;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // this wave's loads of K j + 1 and V j are in LDS
    __syncthreads();                     // everyone's are, and nobody reads K j or V j - 1 any more
    bf16x8_t kf[8], vf[2][ND];
#pragma unroll
    for (int i = 0; i < 8; ++i) kf[i] = k_read(kbuf, i);
    __builtin_amdgcn_sched_barrier(0);
    if (j + 2 < n) stage_tile<D, false>(kOdd ? k_odd : k_even, rk, pos_of(j + 2), e1 - 1, row_bytes, w, lane);
    if (j + 1 < n) stage_tile<D, true>(kOdd ? v_even : v_odd, rv, pos_of(j + 1), e1 - 1, row_bytes, w, lane);
    const int p0 = pos_of(j);
    if (!(p0 + kPreTile <= we0 && p0 >= wlo1)) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          x[u][i] = attends(me, s, p0 + 32 * u + 8 * (i / 4) + 4 * half + i % 4) ? x[u][i] : -INFINITY;
    }
    float top = x[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
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
    uint32_t pk[2][8];
    const f32x16_t zero = {};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      next[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[i % 8], qf[i / 2], i < 2 ? zero : next[i % 2], 0, 0, 0);
      if (i + 8 < NK) kf[i % 8] = k_read(kbuf, i + 8);
      else if (i - (NK - 8) < ND) vf[0][i - (NK - 8)] = v_read(vbuf, 0, i - (NK - 8));
#pragma unroll
      for (int g = PG * i; g < PG * (i + 1); ++g) {
        const int u = g / 8, v = 2 * (g % 8);
        pk[u][g % 8] = pack_bf16x2(fast_exp2(fmaf(x[u][v], scale, -base)), fast_exp2(fmaf(x[u][v + 1], scale, -base)));
        l = dot2_bf16(pk[u][g % 8], 0x3f803f80u, l);  // the sum of the rounded terms, the ones that meet V
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int ut = 0; ut < 4; ++ut) {
      const uint32_t* const q = &pk[ut / 2][4 * (ut % 2)];
      const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, make_uint4(q[0], q[1], q[2], q[3]));
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[ut % 2][d], pf, acc[d], 0, 0, 0);
        if (ut < 3) vf[(ut + 1) % 2][d] = v_read(vbuf, ut + 1, d);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  if (n > 0) {
    stage_tile<D, false>(k_even, rk, pos_of(0), e1 - 1, row_bytes, w, lane);
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
    if (n > 1) stage_tile<D, false>(k_odd, rk, pos_of(1), e1 - 1, row_bytes, w, lane);
    stage_tile<D, true>(v_even, rv, pos_of(0), e1 - 1, row_bytes, w, lane);
    f32x16_t xa[2], xb[2];
#pragma unroll
    for (int i = 0; i < NK; ++i)
      xa[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_read(k_even, i), qf[i / 2], i < 2 ? f32x16_t{} : xa[i % 2], 0, 0, 0);
    for (int j = 0; j < n; j += 2) {
      step(std::false_type{}, j, xa, xb);
      if (j + 1 < n) step(std::true_type{}, j + 1, xb, xa);
    }
  }

  float other = l;
  swap32(l, other);
  l += other;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float worst = 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) worst += fabsf(acc[d][i]) * 0x1p-8f;
  if (__builtin_expect(__ballot(!(worst < INFINITY) || !(l < INFINITY)) != 0, 0)) {
    prefill_careful<D>(p, b, h, s, e, t0, ntok, w);
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

}  // namespace
