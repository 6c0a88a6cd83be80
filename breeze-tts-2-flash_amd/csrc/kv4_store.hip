// The 4-bit KV cache of include/bz_long_cache.h: rounding new keys and values into it, and reading their values back.
//
// A block of 32 dims is codes c of e2m1 (0 .5 1 1.5 2 3 4 6 and a sign) under one scale 2^(E - 127). The scale is the
// smallest power of two with max |x| <= 7 * scale: up to 7 the largest value's rounding to 6 is within 1, the half step
// of [4, 8), so nothing is clipped by more than it would be rounded. x / scale is exact (a power of two), and the only
// rounding is v_cvt_scalef32_pk_fp4_bf16's to nearest even, saturating at 6.
//
// Both directions are bound by memory (nothing is used twice): 16 bytes of bf16 and 4 of codes a lane, four lanes a
// block, so that a wave reads or writes whole rows. 4 rows x 8 heads x 2047 tokens of 128 dims (33.5 MB of bf16, 8.9 of codes and
// scales): 9.2 us to store, 9.4 to load, 4.5 TB/s, where a large copy moves 5.0. One token a row of 16: 2.0 and 2.2 us, the launch.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "bz_long_cache.h"
#include "device_common.cuh"

namespace {

constexpr int kStoreThreads = 256;
constexpr int kMaxTokens = 1 << 30;  // sums of tokens and workgroup sizes stay in 32 bits

struct StoreParams {
  const uint16_t *k, *v;  // bf16 in (store) or out (load)
  int64_t x_sb, x_sh, x_st;
  uint8_t *ck, *cv, *sk, *sv;
  int64_t c_sb, c_sh, c_ss, s_sb, s_sh;
  const int32_t *slots, *counts;
  int tokens, cap;
};

typedef uint16_t u16x2_s __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_s, a), __builtin_bit_cast(u16x2_s, b)));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}

// The scale byte of a block from the bits of its largest |bf16| (sign cleared). 1.75 = mantissa 0x60: with max = f 2^x the
// scale is 2^(x - 2) where f <= 1.75, else 2^(x - 1); a subnormal max is below 2^-126 and takes the smallest scale.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  if (top >= 0x7f80u) return 255;
  const int e = (int)(top >> 7) - 2 + ((top & 0x7f) > 0x60 ? 1 : 0);
  return (uint32_t)max(e, 1);
}

// Token t of (row, head) and the lane's 8 dims; grid (token chunks, heads, rows * 2): K, then V.
template <int D>
__global__ void __launch_bounds__(kStoreThreads) kv4_store_kernel(const StoreParams p) {
  constexpr int LPR = D / 8;
  const int h = blockIdx.y, b = blockIdx.z >> 1, isv = blockIdx.z & 1;
  const int t = (int)(blockIdx.x * (kStoreThreads / LPR)) + (int)threadIdx.x / LPR, c = threadIdx.x % LPR;
  const int count = p.counts ? min(p.counts[b], p.tokens) : p.tokens;
  const int64_t slot = (int64_t)p.slots[b] + t;
  const bool there = t < count && slot >= 0 && slot < p.cap;
  uint4 x = make_uint4(0, 0, 0, 0);
  if (there) {
    const uint16_t* src = (isv ? p.v : p.k) + (int64_t)b * p.x_sb + (int64_t)h * p.x_sh + (int64_t)t * p.x_st + 8 * c;
    x = *reinterpret_cast<const uint4*>(src);
  }
  constexpr uint32_t kAbs = 0x7fff7fffu;
  uint32_t m = pk_max(pk_max(x.x & kAbs, x.y & kAbs), pk_max(x.z & kAbs, x.w & kAbs));
  m = pk_max(m, dpp_u<0xb1>(m));  // over the four lanes of the block
  m = pk_max(m, dpp_u<0x4e>(m));
  const uint32_t e = scale_byte(max(m & 0xffffu, m >> 16));
  const float scale = __uint_as_float(e << 23);
  uint32_t code = 0;
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, x.x), scale, 0);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, x.y), scale, 1);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, x.z), scale, 2);
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(code, __builtin_bit_cast(bf16x2_t, x.w), scale, 3);
  if (e == 255) code = 0;
  if (!there) return;
  uint8_t* const codes = (isv ? p.cv : p.ck) + (int64_t)b * p.c_sb + (int64_t)h * p.c_sh + slot * p.c_ss;
  *reinterpret_cast<uint32_t*>(codes + 4 * c) = code;
  if (c % 4 == 0) (isv ? p.sv : p.sk)[(int64_t)b * p.s_sb + (int64_t)h * p.s_sh + slot * (D / 32) + c / 4] = (uint8_t)e;
}

template <int D>
__global__ void __launch_bounds__(kStoreThreads) kv4_load_kernel(const StoreParams p) {
  constexpr int LPR = D / 8;
  const int h = blockIdx.y, b = blockIdx.z >> 1, isv = blockIdx.z & 1;
  const int t = (int)(blockIdx.x * (kStoreThreads / LPR)) + (int)threadIdx.x / LPR, c = threadIdx.x % LPR;
  if (t >= p.tokens) return;
  const int64_t slot = (int64_t)p.slots[b] + t;
  uint4 x = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < p.cap) {
    const uint8_t* const codes = (isv ? p.cv : p.ck) + (int64_t)b * p.c_sb + (int64_t)h * p.c_sh + slot * p.c_ss;
    const uint32_t code = *reinterpret_cast<const uint32_t*>(codes + 4 * c);
    const uint32_t e = (isv ? p.sv : p.sk)[(int64_t)b * p.s_sb + (int64_t)h * p.s_sh + slot * (D / 32) + c / 4];
    const float scale = __uint_as_float(e << 23);
    x.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 0));
    x.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 1));
    x.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 2));
    x.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(code, scale, 3));
  }
  uint16_t* const dst =
      const_cast<uint16_t*>(isv ? p.v : p.k) + (int64_t)b * p.x_sb + (int64_t)h * p.x_sh + (int64_t)t * p.x_st + 8 * c;
  *reinterpret_cast<uint4*>(dst) = x;
}

int check_store(const void* k, const void* v, int64_t sb, int64_t sh, int64_t st, int32_t tokens, const int32_t* slots,
                const bz_kv4_cache* c) {
  if (k == nullptr || v == nullptr || slots == nullptr || c == nullptr) return BZ_ERR_NULL;
  if (c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr) return BZ_ERR_NULL;
  if (tokens <= 0 || c->batch <= 0 || c->num_kv_heads <= 0 || c->capacity <= 0) return BZ_ERR_SHAPE;
  if (tokens > kMaxTokens || c->capacity > kMaxTokens) return BZ_ERR_SHAPE;
  if (c->batch > 32767 || c->num_kv_heads > 65535) return BZ_ERR_SHAPE;  // grid limits
  const int D = c->head_dim;
  if (D != 64 && D != 128) return BZ_ERR_UNSUPPORTED;
  if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) || ((sb | sh | st) & 7)) return BZ_ERR_ALIGNMENT;
  const int code_align = D / 8 - 1, scale_align = D / 32 - 1;
  if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & code_align) ||
      ((c->stride_b | c->stride_h | c->stride_s) & code_align))
    return BZ_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) | (uintptr_t)c->scale_stride_b |
       (uintptr_t)c->scale_stride_h) &
      scale_align)
    return BZ_ERR_ALIGNMENT;
  return c->stride_s < D / 2 ? BZ_ERR_SHAPE : BZ_OK;
}

StoreParams store_params(const void* k, const void* v, int64_t sb, int64_t sh, int64_t st, int32_t tokens,
                         const int32_t* slots, const bz_kv4_cache* c) {
  StoreParams p{};
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.x_sb = sb, p.x_sh = sh, p.x_st = st;
  p.ck = static_cast<uint8_t*>(c->k);
  p.cv = static_cast<uint8_t*>(c->v);
  p.sk = static_cast<uint8_t*>(c->k_scale);
  p.sv = static_cast<uint8_t*>(c->v_scale);
  p.c_sb = c->stride_b, p.c_sh = c->stride_h, p.c_ss = c->stride_s;
  p.s_sb = c->scale_stride_b, p.s_sh = c->scale_stride_h;
  p.slots = slots;
  p.tokens = tokens;
  p.cap = c->capacity;
  return p;
}

dim3 store_grid(const bz_kv4_cache* c, int tokens) {
  const int per = kStoreThreads / (c->head_dim / 8);
  return dim3((tokens + per - 1) / per, c->num_kv_heads, 2 * c->batch);
}

}  // namespace

#define BZ_EXPORT __attribute__((visibility("default")))

extern "C" {

BZ_EXPORT int bz_kv4_store(const void* k, const void* v, int64_t x_stride_b, int64_t x_stride_h, int64_t x_stride_t,
                           int32_t tokens, const int32_t* slots, const int32_t* counts, const bz_kv4_cache* cache,
                           hipStream_t stream) {
  const int rc = check_store(k, v, x_stride_b, x_stride_h, x_stride_t, tokens, slots, cache);
  if (rc != BZ_OK) return rc;
  StoreParams p = store_params(k, v, x_stride_b, x_stride_h, x_stride_t, tokens, slots, cache);
  p.counts = counts;
  if (cache->head_dim == 128)
    hipLaunchKernelGGL(kv4_store_kernel<128>, store_grid(cache, tokens), dim3(kStoreThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(kv4_store_kernel<64>, store_grid(cache, tokens), dim3(kStoreThreads), 0, stream, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

BZ_EXPORT int bz_kv4_load(const bz_kv4_cache* cache, const int32_t* slots, int32_t tokens, void* k, void* v,
                          int64_t x_stride_b, int64_t x_stride_h, int64_t x_stride_t, hipStream_t stream) {
  const int rc = check_store(k, v, x_stride_b, x_stride_h, x_stride_t, tokens, slots, cache);
  if (rc != BZ_OK) return rc;
  const StoreParams p = store_params(k, v, x_stride_b, x_stride_h, x_stride_t, tokens, slots, cache);
  if (cache->head_dim == 128)
    hipLaunchKernelGGL(kv4_load_kernel<128>, store_grid(cache, tokens), dim3(kStoreThreads), 0, stream, p);
  else
    hipLaunchKernelGGL(kv4_load_kernel<64>, store_grid(cache, tokens), dim3(kStoreThreads), 0, stream, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

}  // extern "C"
