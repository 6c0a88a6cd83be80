// The paged cache of include/bz_paged_cache.h: rotary positions, storing new keys and values, reading them back.
//
// A head vector is worked on by D / 16 lanes of 16 values each, as two 16-byte chunks that hold whole pairs: chunks j and
// j + R / 16 of the R rotated dims (both halves of eight pairs in the half layout, eight pairs of neighbours in the
// interleaved one), then the chunks behind R two by two. So no value crosses lanes but for the norm's sum and the 8-bit
// scale's maximum (DPP).
//
// Angles: position * inv_freq in turns in fp64, less its nearest integer, then v_sin / v_cos, which take turns. fp32 products would
// be off by position * 2^-24 (0.008 rad at 131072, eight bf16 roundings); fp64 costs 8 multiplies and 8 roundings a lane.
//
// Memory bound: every byte is read and written once (4097 tokens of 40 heads, 64 of 128 dims turned: 84 MB in 15.8 us, 5.3 TB/s, where a
// large copy moves 5.1; rope_store of 6000 tokens, 16 q and 8 kv heads, normed: 98 MB in 20.7; paged_load of 4 rows of 2047: 67 MB in 12.9).
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "bz_paged_cache.h"
#include "paged_common.cuh"

namespace {

constexpr int kPagedThreads = 256;
// Head vectors (of q, k and v, all tokens) from which on a thread of rope_store takes four, with one turn's cosines for all (us, 16 q and
// 8 kv heads of 128 dims, normed, one / four a thread: 6000 tokens 22.9 / 20.7, 2048 11.9 / 11.1, 512 6.3 / 6.6; without a rotation one,
// 6000 10.6 / 23.6).
constexpr int64_t kManyHeads = 1 << 15;

struct TurnParams {
  const double* inv_freq;
  int R, interleaved;
  float factor;  // inverse: 1 / factor
  double sign;   // 1 / 2 pi, negative for the inverse
};

struct RopeParams {
  const uint16_t* x;
  int64_t x_st, x_sh;
  uint16_t* out;
  int64_t o_st, o_sh;
  const void* positions;
  int positions_64;
  int64_t tokens;
  int heads;
  TurnParams turn;
};

struct PagedStoreParams {
  bz::PagedRows rows;
  char *k, *v;
  int64_t kv_sp, kv_sh, kv_ss;
  uint8_t *ks, *vs;
  int64_t sc_sp, sc_sh;
  const uint16_t *xk, *xv, *xq;
  int64_t k_st, k_sh, v_st, v_sh, q_st, q_sh;
  uint16_t* q_out;
  int64_t o_st, o_sh;
  int NH, NKV;
  const uint16_t *qw, *kw;
  float eps;
  const void* positions;
  int positions_64;
  TurnParams turn;
};

// The lane's two chunks of a head, j of its D / 16 lanes.
struct Chunks {
  int a, b;
  bool turned;
};
__device__ __forceinline__ Chunks chunks_of(int j, int R) {
  const int n = R / 16;
  return j < n ? Chunks{j, j + n, true} : Chunks{2 * j, 2 * j + 1, false};
}

// cos and sin (times factor) of the lane's eight pairs at a position.
__device__ __forceinline__ void turn_of(const TurnParams& t, int j, double pos, float (&cs)[8], float (&sn)[8]) {
  const double turns = pos * t.sign;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int f = !t.interleaved ? 8 * j + i : i < 4 ? 4 * j + i : 4 * (j + t.R / 16) + i - 4;
    const double a = turns * t.inv_freq[f];
    const float r = (float)(a - __builtin_rint(a));
    cs[i] = t.factor * __builtin_amdgcn_cosf(r);
    sn[i] = t.factor * __builtin_amdgcn_sinf(r);
  }
}

// x: the lane's 16 values, chunk a then chunk b.
__device__ __forceinline__ void apply_turn(float (&x)[16], bool interleaved, const float (&cs)[8], const float (&sn)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x0 = interleaved ? x[2 * i] : x[i], x1 = interleaved ? x[2 * i + 1] : x[i + 8];
    const float y0 = fmaf(x0, cs[i], -(x1 * sn[i])), y1 = fmaf(x1, cs[i], x0 * sn[i]);
    (interleaved ? x[2 * i] : x[i]) = y0;
    (interleaved ? x[2 * i + 1] : x[i + 8]) = y1;
  }
}

__device__ __forceinline__ void load16(const uint16_t* src, const Chunks& c, uint4& a, uint4& b) {
  a = *reinterpret_cast<const uint4*>(src + 8 * c.a);
  b = *reinterpret_cast<const uint4*>(src + 8 * c.b);
}
__device__ __forceinline__ void unpack16(const uint4& a, const uint4& b, float (&x)[16]) {
  float y[8];
  unpack8(a, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = y[i];
  unpack8(b, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[8 + i] = y[i];
}
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

__device__ __forceinline__ double position_at(const void* positions, int is64, int64_t n) {
  return is64 ? (double)static_cast<const int64_t*>(positions)[n] : (double)static_cast<const int32_t*>(positions)[n];
}

// One head vector by D / 16 lanes.
template <int D>
__global__ void __launch_bounds__(kPagedThreads) rope_kernel(const RopeParams p) {
  constexpr int LPH = D / 16;
  const int64_t item = (int64_t)blockIdx.x * (kPagedThreads / LPH) + threadIdx.x / LPH;
  const int j = threadIdx.x % LPH;
  if (item >= p.tokens * p.heads) return;
  const int64_t n = item / p.heads;
  const int h = (int)(item - n * p.heads);
  const Chunks c = chunks_of(j, p.turn.R);
  uint4 a, b;
  load16(p.x + n * p.x_st + h * p.x_sh, c, a, b);
  if (c.turned) {
    float x[16], cs[8], sn[8];
    turn_of(p.turn, j, position_at(p.positions, p.positions_64, n), cs, sn);
    unpack16(a, b, x);
    apply_turn(x, p.turn.interleaved, cs, sn);
    a = pack8(x), b = pack8(x + 8);
  }
  uint16_t* const o = p.out + n * p.o_st + h * p.o_sh;
  *reinterpret_cast<uint4*>(o + 8 * c.a) = a;
  *reinterpret_cast<uint4*>(o + 8 * c.b) = b;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_bits(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}

// The head vectors hg, hg + HG, .. (HP of them, HG = heads / HP) of a token's q, k and v, by D / 16 lanes: the token's row, its angles and
// their cosines are worked out once for all of them.
template <int D, bool F8, bool ROPE, int HP>
__global__ void __launch_bounds__(kPagedThreads) paged_store_kernel(const PagedStoreParams p) {
  constexpr int LPH = D / 16;
  const int64_t item = (int64_t)blockIdx.x * (kPagedThreads / LPH) + threadIdx.x / LPH;
  const int j = threadIdx.x % LPH, heads = p.NH + 2 * p.NKV, HG = (heads + HP - 1) / HP;
  // (a wave's lanes may leave here: the lanes of one head leave together, and those are all that meet below)
  if (item >= (int64_t)p.rows.tokens * HG) return;
  const int n = (int)(item / HG), hg = (int)(item - (int64_t)n * HG);
  int row, pos;
  if (!bz::row_of(p.rows, n, row, pos)) return;
  const Chunks c = chunks_of(j, ROPE ? p.turn.R : D);
  uint4 a[HP], b[HP];
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    const int hh = min(hg + i * HG, heads - 1), h = hh < p.NH ? hh : hh < p.NH + p.NKV ? hh - p.NH : hh - p.NH - p.NKV;
    load16(hh < p.NH             ? p.xq + n * p.q_st + h * p.q_sh
           : hh < p.NH + p.NKV ? p.xk + n * p.k_st + h * p.k_sh
                               : p.xv + n * p.v_st + h * p.v_sh,
           c, a[i], b[i]);
  }
  const int page = bz::page_of(p.rows, row, pos), at = pos & ((1 << p.rows.pshift) - 1);
  float cs[8], sn[8];
  if (ROPE && c.turned && hg < p.NH + p.NKV)
    turn_of(p.turn, j, p.positions ? position_at(p.positions, p.positions_64, n) : (double)pos, cs, sn);
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    const int hh = hg + i * HG;
    if (hh >= heads) return;
    const bool isq = hh < p.NH, isv = hh >= p.NH + p.NKV;
    const int h = isq ? hh : isv ? hh - p.NH - p.NKV : hh - p.NH;
    if (!isq && page < 0) continue;
    const uint16_t* const w = isq ? p.qw : p.kw;
    const bool changed = ROPE && !isv && (c.turned || w != nullptr);
    float x[16];
    if (F8 || (ROPE && !isv)) unpack16(a[i], b[i], x);
    if (ROPE && !isv) {
      if (w != nullptr) {
        uint4 wa, wb;
        load16(w, c, wa, wb);
        float y[16];
        unpack16(wa, wb, y);
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < 16; ++u) s = fmaf(x[u], x[u], s);
        s += dpp<0xb1>(s);  // over the lanes of the head
        s += dpp<0x4e>(s);
        if (LPH == 8) s += dpp<0x141>(s);
        // (correctly rounded steps: the hardware's own reciprocal root is off by an ulp)
        const float r = 1.f / sqrtf(s * (1.f / D) + p.eps);
#pragma unroll
        for (int u = 0; u < 16; ++u) x[u] = x[u] * r * y[u];
      }
      if (c.turned) apply_turn(x, p.turn.interleaved, cs, sn);
    }
    char* const to = (isv ? p.v : p.k) + page * p.kv_sp + h * p.kv_sh + at * p.kv_ss;  // where a k or v goes
    if (!F8 || isq) {
      if (changed) a[i] = pack8(x), b[i] = pack8(x + 8);
      uint16_t* const o = isq ? p.q_out + n * p.o_st + h * p.o_sh : reinterpret_cast<uint16_t*>(to);
      *reinterpret_cast<uint4*>(o + 8 * c.a) = a[i];
      *reinterpret_cast<uint4*>(o + 8 * c.b) = b[i];
      continue;
    }
    // the maximum by the values' bits, which order NaN above infinity
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < 16; ++u) top = max(top, __float_as_uint(x[u]) & 0x7fffffffu);
    top = max(top, dpp_bits<0xb1>(top));
    top = max(top, dpp_bits<0x4e>(top));
    if (LPH == 8) top = max(top, dpp_bits<0x141>(top));
    // top = f 2^e, 448 = 1.75 2^8: the scale is 2^(e - 8) up to f = 1.75, else 2^(e - 7)
    const int E = max((int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), 10);
    const bool bad = top >= 0x7f800000u;
    const float inv = __uint_as_float((uint32_t)(254 - E) << 23);  // 2^-(E - 127): E is 10 .. 247
    uint2 code[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t c2[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float* const y = x + 8 * q + 4 * u;
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, 0, false);
        word = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, word, true);
        c2[u] = bad ? 0u : (uint32_t)word;
      }
      code[q] = make_uint2(c2[0], c2[1]);
    }
    *reinterpret_cast<uint2*>(to + 8 * c.a) = code[0];
    *reinterpret_cast<uint2*>(to + 8 * c.b) = code[1];
    if (j == 0) (isv ? p.vs : p.ks)[page * p.sc_sp + h * p.sc_sh + at] = (uint8_t)(bad ? 255 : E);
  }
}

struct PagedLoadParams {
  bz::PagedRows rows;
  const char *k, *v;
  int64_t kv_sp, kv_sh, kv_ss;
  const uint8_t *ks, *vs;
  int64_t sc_sp, sc_sh;
  const int32_t* starts;
  int count, heads;
  uint16_t *ok, *ov;
  int64_t o_sb, o_sh, o_st;
};

// Token t of (row, head), 8 dims a lane of K and of V; grid (token chunks, heads, rows), of either of the latter up to kMaxGridYZ, whose
// workgroups go on where there are more.
constexpr int kMaxGridYZ = 65535;  // HIP's
template <int D, bool F8>
__global__ void __launch_bounds__(kPagedThreads) paged_load_kernel(const PagedLoadParams p) {
  constexpr int LPR = D / 8;
  const int64_t t = (int64_t)blockIdx.x * (kPagedThreads / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;
  if (t >= p.count) return;
  for (int b = blockIdx.z; b < p.rows.B; b += gridDim.z) {
    const int64_t pos = p.starts[b] + t;
    const int page = pos > INT32_MAX ? -1 : bz::page_of(p.rows, b, (int)pos);
    for (int h = blockIdx.y; h < p.heads; h += gridDim.y) {
      uint4 x[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
      if (page >= 0) {
        const int at = (int)pos & ((1 << p.rows.pshift) - 1);
        const int64_t off = page * p.kv_sp + h * p.kv_sh + at * p.kv_ss;
        if constexpr (F8) {
          const int64_t so = page * p.sc_sp + h * p.sc_sh + at;
          const uint2 ck = *reinterpret_cast<const uint2*>(p.k + off + 8 * c), cv = *reinterpret_cast<const uint2*>(p.v + off + 8 * c);
          const uint32_t ek = p.ks[so], ev = p.vs[so];
          x[0] = bz::f8_values(ck, ek);
          x[1] = bz::f8_values(cv, ev);
        } else {
          x[0] = *reinterpret_cast<const uint4*>(p.k + off + 16 * c);
          x[1] = *reinterpret_cast<const uint4*>(p.v + off + 16 * c);
        }
      }
      const int64_t o = b * p.o_sb + h * p.o_sh + t * p.o_st + 8 * c;
      *reinterpret_cast<uint4*>(p.ok + o) = x[0];
      *reinterpret_cast<uint4*>(p.ov + o) = x[1];
    }
  }
}

bool aligned(const void* p, int64_t strides) { return !(reinterpret_cast<uintptr_t>(p) & 15) && !(strides & 7); }

int check_rope(const bz_rope& r, int D) {
  if (r.inv_freq == nullptr) return BZ_ERR_NULL;
  if (r.rotary_dim <= 0 || r.rotary_dim > D || r.rotary_dim % 16 != 0) return BZ_ERR_SHAPE;
  return (reinterpret_cast<uintptr_t>(r.inv_freq) & 7) ? BZ_ERR_ALIGNMENT : BZ_OK;
}

TurnParams turn_params(const bz_rope& r, bool inverse) {
  const double turn = 0.15915494309189533577;  // 1 / 2 pi
  return {r.inv_freq, r.rotary_dim, r.interleaved != 0, inverse ? 1.f / r.factor : r.factor, inverse ? -turn : turn};
}

int positions_ok(const void* p, int is64) {
  return !(reinterpret_cast<uintptr_t>(p) & (is64 ? 7 : 3));
}

}  // namespace

#define BZ_EXPORT __attribute__((visibility("default")))

namespace bz {

int check_paged(const bz_paged_cache* c, bool rows) {
  if (c->k == nullptr || c->v == nullptr || c->page_table == nullptr) return BZ_ERR_NULL;
  if (rows && c->seq_lens == nullptr) return BZ_ERR_NULL;
  if (c->pages <= 0 || c->num_kv_heads <= 0 || c->batch <= 0 || c->max_pages <= 0) return BZ_ERR_SHAPE;
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return BZ_ERR_UNSUPPORTED;
  if ((c->head_dim != 64 && c->head_dim != 128) || (c->bits != 8 && c->bits != 16)) return BZ_ERR_UNSUPPORTED;
  if ((int64_t)c->max_pages * c->page_size > kMaxPositions) return BZ_ERR_SHAPE;
  if (rows && (c->tokens <= 0 || c->tokens > kMaxPositions)) return BZ_ERR_SHAPE;
  if (rows && c->q_start == nullptr && c->tokens != c->batch) return BZ_ERR_SHAPE;
  const int64_t row = c->bits == 8 ? c->head_dim : 2 * c->head_dim;
  if (c->stride_s < row || c->stride_s >= (1 << 30) / c->page_size) return BZ_ERR_SHAPE;
  if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) ||
      ((c->stride_page | c->stride_h | c->stride_s) & 15))
    return BZ_ERR_ALIGNMENT;
  if (c->bits == 8) {
    if (c->k_scale == nullptr || c->v_scale == nullptr) return BZ_ERR_NULL;
    if (((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3) ||
        ((c->scale_stride_page | c->scale_stride_h) & 3))
      return BZ_ERR_ALIGNMENT;
  }
  if ((reinterpret_cast<uintptr_t>(c->page_table) | reinterpret_cast<uintptr_t>(c->seq_lens) |
       reinterpret_cast<uintptr_t>(c->q_start)) & 3)
    return BZ_ERR_ALIGNMENT;
  return BZ_OK;
}

PagedRows paged_rows(const bz_paged_cache* c) {
  return {c->page_table, c->table_stride, c->seq_lens,  c->q_start,
          c->batch,      c->tokens,       c->max_pages, c->pages,   __builtin_ctz((unsigned)c->page_size)};
}

}  // namespace bz

extern "C" {

BZ_EXPORT int bz_rope_apply(const bz_rope_args* a, hipStream_t stream) {
  if (a == nullptr || a->x == nullptr || a->out == nullptr || a->positions == nullptr) return BZ_ERR_NULL;
  if (a->tokens <= 0 || a->heads <= 0) return BZ_ERR_SHAPE;
  const int D = a->head_dim;
  if (D != 64 && D != 128) return BZ_ERR_UNSUPPORTED;
  const int rc = check_rope(a->rope, D);
  if (rc != BZ_OK) return rc;
  if (!aligned(a->x, a->x_stride_t | a->x_stride_h) || !aligned(a->out, a->out_stride_t | a->out_stride_h) ||
      !positions_ok(a->positions, a->positions_64))
    return BZ_ERR_ALIGNMENT;
  const RopeParams p{static_cast<const uint16_t*>(a->x), a->x_stride_t, a->x_stride_h, static_cast<uint16_t*>(a->out),
                     a->out_stride_t, a->out_stride_h, a->positions, a->positions_64, a->tokens, a->heads,
                     turn_params(a->rope, a->inverse != 0)};
  const int64_t per = kPagedThreads / (D / 16), grid = ((int64_t)a->tokens * a->heads + per - 1) / per;
  if (grid > kMaxGrid) return BZ_ERR_SHAPE;
  hipLaunchKernelGGL(D == 128 ? rope_kernel<128> : rope_kernel<64>, dim3((unsigned)grid), dim3(kPagedThreads), 0, stream, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

BZ_EXPORT int bz_paged_store(const bz_paged_store_args* a, hipStream_t stream) {
  if (a == nullptr || a->k == nullptr || a->v == nullptr) return BZ_ERR_NULL;
  const bz_paged_cache* c = &a->cache;
  int rc = bz::check_paged(c, true);
  if (rc != BZ_OK) return rc;
  const bool rope = a->rope.inv_freq != nullptr;
  if (!rope && (a->q != nullptr || a->num_q_heads != 0 || a->q_norm_weight != nullptr || a->k_norm_weight != nullptr))
    return BZ_ERR_UNSUPPORTED;
  if (rope && (rc = check_rope(a->rope, c->head_dim)) != BZ_OK) return rc;
  if (a->num_q_heads < 0 || (a->q != nullptr) != (a->num_q_heads > 0)) return BZ_ERR_SHAPE;
  if (a->q != nullptr && a->q_out == nullptr) return BZ_ERR_NULL;
  if (!aligned(a->k, a->k_stride_t | a->k_stride_h) || !aligned(a->v, a->v_stride_t | a->v_stride_h) ||
      !aligned(a->q, a->q_stride_t | a->q_stride_h) || !aligned(a->q_out, a->q_out_stride_t | a->q_out_stride_h) ||
      !aligned(a->q_norm_weight, 0) || !aligned(a->k_norm_weight, 0) || !positions_ok(a->positions, a->positions_64))
    return BZ_ERR_ALIGNMENT;
  const int D = c->head_dim;
  PagedStoreParams p{};
  p.rows = bz::paged_rows(c);
  p.k = static_cast<char*>(c->k), p.v = static_cast<char*>(c->v);
  p.kv_sp = c->stride_page, p.kv_sh = c->stride_h, p.kv_ss = c->stride_s;
  p.ks = static_cast<uint8_t*>(c->k_scale), p.vs = static_cast<uint8_t*>(c->v_scale);
  p.sc_sp = c->scale_stride_page, p.sc_sh = c->scale_stride_h;
  p.xk = static_cast<const uint16_t*>(a->k), p.xv = static_cast<const uint16_t*>(a->v), p.xq = static_cast<const uint16_t*>(a->q);
  p.k_st = a->k_stride_t, p.k_sh = a->k_stride_h, p.v_st = a->v_stride_t, p.v_sh = a->v_stride_h;
  p.q_st = a->q_stride_t, p.q_sh = a->q_stride_h;
  p.q_out = static_cast<uint16_t*>(a->q_out), p.o_st = a->q_out_stride_t, p.o_sh = a->q_out_stride_h;
  p.NH = a->num_q_heads, p.NKV = c->num_kv_heads;
  p.qw = static_cast<const uint16_t*>(a->q_norm_weight), p.kw = static_cast<const uint16_t*>(a->k_norm_weight), p.eps = a->eps;
  p.positions = a->positions, p.positions_64 = a->positions_64;
  if (rope) p.turn = turn_params(a->rope, false);
  const int64_t heads = (int64_t)p.NH + 2 * (int64_t)p.NKV;
  if (heads > INT32_MAX) return BZ_ERR_SHAPE;
  const int HP = rope && c->tokens * heads >= kManyHeads ? 4 : 1;
  const int64_t per = kPagedThreads / (D / 16), grid = (c->tokens * ((heads + HP - 1) / HP) + per - 1) / per;
  if (grid > kMaxGrid) return BZ_ERR_SHAPE;
  using Fn = void (*)(const PagedStoreParams);
  const Fn fns[2][2][3] = {
      {{paged_store_kernel<64, false, false, 1>, paged_store_kernel<64, false, true, 1>, paged_store_kernel<64, false, true, 4>},
       {paged_store_kernel<64, true, false, 1>, paged_store_kernel<64, true, true, 1>, paged_store_kernel<64, true, true, 4>}},
      {{paged_store_kernel<128, false, false, 1>, paged_store_kernel<128, false, true, 1>, paged_store_kernel<128, false, true, 4>},
       {paged_store_kernel<128, true, false, 1>, paged_store_kernel<128, true, true, 1>, paged_store_kernel<128, true, true, 4>}}};
  hipLaunchKernelGGL(fns[D == 128][c->bits == 8][HP == 4 ? 2 : rope], dim3((unsigned)grid), dim3(kPagedThreads), 0, stream, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

BZ_EXPORT int bz_paged_load(const bz_paged_cache* c, const int32_t* starts, int32_t count, void* k, void* v,
                            int64_t x_stride_b, int64_t x_stride_h, int64_t x_stride_t, hipStream_t stream) {
  if (c == nullptr || starts == nullptr || k == nullptr || v == nullptr) return BZ_ERR_NULL;
  const int rc = bz::check_paged(c, false);
  if (rc != BZ_OK) return rc;
  if (count <= 0 || count > kMaxPositions) return BZ_ERR_SHAPE;
  if (!aligned(k, x_stride_b | x_stride_h | x_stride_t) || !aligned(v, 0) || (reinterpret_cast<uintptr_t>(starts) & 3))
    return BZ_ERR_ALIGNMENT;
  PagedLoadParams p{bz::paged_rows(c), static_cast<const char*>(c->k), static_cast<const char*>(c->v), c->stride_page,
                    c->stride_h, c->stride_s, static_cast<const uint8_t*>(c->k_scale), static_cast<const uint8_t*>(c->v_scale),
                    c->scale_stride_page, c->scale_stride_h, starts, count, c->num_kv_heads, static_cast<uint16_t*>(k),
                    static_cast<uint16_t*>(v), x_stride_b, x_stride_h, x_stride_t};
  const int64_t per = kPagedThreads / (c->head_dim / 8), chunks = (count + per - 1) / per;
  if (chunks > kMaxGrid) return BZ_ERR_SHAPE;
  const dim3 grid((unsigned)chunks, std::min(c->num_kv_heads, kMaxGridYZ), std::min(c->batch, kMaxGridYZ));
  using Fn = void (*)(const PagedLoadParams);
  const Fn fns[2][2] = {{paged_load_kernel<64, false>, paged_load_kernel<64, true>},
                        {paged_load_kernel<128, false>, paged_load_kernel<128, true>}};
  hipLaunchKernelGGL(fns[c->head_dim == 128][c->bits == 8], grid, dim3(kPagedThreads), 0, stream, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

}  // extern "C"
