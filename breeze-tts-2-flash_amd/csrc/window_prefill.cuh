// Device code of bz_gqa_window over a chunk of many query tokens (include/bz_long_cache.h).
//
// A workgroup of four waves takes 128 columns: (token, q head) pairs of one kv head, 128 / G tokens of a row times its G
// heads, 32 a wave, so K and V are fetched once for the whole group. It walks the positions any of its tokens attends (the
// sinks' tiles, then the window's; tile_range) in tiles of 64 staged in LDS, two buffers, the next tile's loads in flight
// while one is worked on.
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

constexpr int kPreThreads = 256, kPreCols = 128, kPreTile = 64;

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
template <int D>
__device__ __forceinline__ void stage_tile(char* base, const Rsrc& rk, const Rsrc& rv, int pos0, int last, uint32_t row_bytes,
                                           int w, int lane) {
  using L = PreLds<D>;
  constexpr int RPI = 1024 / L::kRow, CH = D / 8;  // rows an instruction, chunks a row
#pragma unroll
  for (int u = 0; u < 16 / RPI; ++u) {
    const int row = 16 * w + RPI * u + lane / CH, c = lane % CH;
    const uint32_t off = (uint32_t)min(pos0 + row, last) * row_bytes;
    char* const to = base + (16 * w + RPI * u) * L::kRow;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (__attribute__((address_space(3))) void*)to, 16,
                                             off + 16 * (c ^ L::k_swz(row)), 0, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (__attribute__((address_space(3))) void*)(to + L::kBytes), 16,
                                             off + 16 * (c ^ L::v_swz(row)), 0, 0, 0);
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

  const float scale = fmaxf(fabsf(p.scale_log2), 1e-30f);  // scores are taken times a positive scale: q carries the sign
  const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
  bf16x8_t qf[NQ];
  {
    const uint16_t* src = p.q + (int64_t)b * p.q_sb + (int64_t)tok * p.q_st + (int64_t)hq * p.q_sh + 8 * half;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      uint4 x = *reinterpret_cast<const uint4*>(src + 16 * j);
      x.x ^= flip, x.y ^= flip, x.z ^= flip, x.w ^= flip;
      qf[j] = __builtin_bit_cast(bf16x8_t, x);
    }
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
  const int wlo0 = max(s, we0 - p.window), wlo1 = max(s, we1 - p.window), wsink = s + min(p.sinks, we1 - s);

  __shared__ __align__(16) char lds[2][2 * L::kBytes];
  const int64_t head = (int64_t)b * p.kv_sb + (int64_t)h * p.kv_sh;
  const uint32_t row_bytes = (uint32_t)p.kv_ss;
  const Rsrc rk = span_rsrc(p.k + head, e1 * (int)p.kv_ss), rv = span_rsrc(p.v + head, e1 * (int)p.kv_ss);

  // this lane's LDS addresses: K chunk 2 j + half of row c; V, transposed: the four rows and 16 dims of its group of 16 lanes
  const int k_addr = c * L::kRow, k_sw = L::k_swz(c);
  const int l16 = lane % 16, v_row = 4 * half + l16 / 4;
  int v_addr[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
    v_addr[d] = L::kBytes + v_row * L::kRow + 16 * ((4 * d + 2 * ((lane / 16) % 2) + (l16 % 4) / 2) ^ L::v_swz(v_row)) + 8 * (l16 % 2);

  float m = -INFINITY, l = 0.f;
  f32x16_t acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;

  if (n > 0) stage_tile<D>(lds[0], rk, rv, pos_of(0), e1 - 1, row_bytes, w, lane);
  for (int j = 0; j < n; ++j) {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // this wave's loads of tile j are in LDS
    __syncthreads();                     // everyone's are, and nobody reads the other buffer any more
    if (j + 1 < n) stage_tile<D>(lds[(j + 1) & 1], rk, rv, pos_of(j + 1), e1 - 1, row_bytes, w, lane);
    const int p0 = pos_of(j);
    if (p0 >= we1 || (p0 + kPreTile <= wlo0 && p0 >= wsink)) continue;  // this wave attends nothing here
    const char* const buf = lds[j & 1];

    f32x16_t x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[u][i] = 0.f;
#pragma unroll
      for (int k = 0; k < NQ; ++k) {
        const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(buf + k_addr + 32 * u * L::kRow + 16 * ((2 * k + half) ^ k_sw));
        x[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[k], x[u], 0, 0, 0);
      }
    }
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
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float a = fast_exp2(fmaf(x[u][i], scale, -base)), a1 = fast_exp2(fmaf(x[u][i + 1], scale, -base));
        l += a + a1;
        pk[u][i / 2] = pack_bf16x2(a, a1);
      }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8_t pf =
            __builtin_bit_cast(bf16x8_t, make_uint4(pk[u][4 * t], pk[u][4 * t + 1], pk[u][4 * t + 2], pk[u][4 * t + 3]));
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          using Tr = __attribute__((address_space(3))) s16x4_lds*;
          const char* const at = buf + v_addr[d] + (32 * u + 16 * t) * L::kRow;
          const auto v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(at));
          const auto v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Tr)(at + 8 * L::kRow));
          const uint2 a = __builtin_bit_cast(uint2, v0), a1 = __builtin_bit_cast(uint2, v1);
          acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, make_uint4(a.x, a.y, a1.x, a1.y)), pf,
                                                           acc[d], 0, 0, 0);
        }
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
