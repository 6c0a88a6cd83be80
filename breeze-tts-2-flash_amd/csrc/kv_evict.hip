// Eviction from a KV cache by accumulated attention weight (include/bz_long_cache.h): which positions of each (row, kv
// head) stay (bz_kv_select), and the cache's rows moved together (bz_kv_compact).
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "bz_long_cache.h"
#include "device_common.cuh"

namespace {

// ---------------------------------------------------------------------------------------------------- selection
//
// One workgroup per (row, kv head). The threshold is the m-th largest key of the middle positions (m = keep - sinks -
// recent), found by a radix selection from the top digit down (11 + 11 + 10 bits: a histogram in LDS, then the digit
// that holds the m-th key); every key above it stays, and as many equal ones, from the lowest position on, as are still
// missing. Each thread owns one run of consecutive positions, so one scan over the threads gives every kept position its
// place in ascending order.

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kBins = 2048;

struct SelectParams {
  const float* w;
  int64_t w_sb, w_sh;
  const int32_t *seq_lens, *kv_start;
  int32_t *index, *lens;
  float* wo;
  int64_t wo_sb, wo_sh;
  int NKV, cap, keep, sinks, recent;
};

// Order-preserving map of float to uint32; NaN above everything, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float f) {
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if ((u & 0x7fffffffu) == 0) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum of x over the workgroup's threads; total: the sum over all. s: kSelWaves + 1 words of LDS.
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t* s, uint64_t* total) {
  const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
  uint64_t v = x;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const uint64_t y = __shfl_up(v, d);
    if (lane >= d) v += y;
  }
  __syncthreads();  // s may still be read from an earlier scan
  if (lane == kWave - 1) s[w] = v;
  __syncthreads();
  uint64_t before = 0, all = 0;
#pragma unroll
  for (int u = 0; u < kSelWaves; ++u) {
    before += u < w ? s[u] : 0;
    all += s[u];
  }
  *total = all;
  return before + v - x;
}

__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const SelectParams p) {
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint64_t s_scan[kSelWaves];
  __shared__ uint32_t s_found[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int e = min(max(p.seq_lens[b], 0), p.cap);
  const int s = p.kv_start ? min(max(p.kv_start[b], 0), e) : 0;
  const int n = e - s, kept = min(n, p.keep);
  const float* const w = p.w + (int64_t)b * p.w_sb + (int64_t)h * p.w_sh;
  int32_t* const index = p.index + ((int64_t)b * p.NKV + h) * p.keep;

  if (n <= p.keep) {
    for (int d = tid; d < p.keep; d += kSelThreads) index[d] = d < n ? s + d : -1;
  } else {
    const int lo = s + p.sinks, hi = e - p.recent;  // hi - lo > m >= 0
    const uint32_t m = (uint32_t)(p.keep - p.sinks - p.recent);
    uint32_t prefix = 0, left = m;  // the threshold's known top bits; how many of the keys with those bits stay
    int known = 0;                  // bits known
    if (m > 0) {
      for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10, shift = 32 - known - bits;
        for (int i = tid; i < kBins; i += kSelThreads) s_hist[i] = 0;
        __syncthreads();
        for (int i = lo + tid; i < hi; i += kSelThreads) {
          const uint32_t k = weight_key(w[i]);
          if (known == 0 || k >> (32 - known) == prefix) atomicAdd(&s_hist[(k >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // the digit with fewer than `left` keys above it and at least `left` from it on: thread t sums bins from the top
        uint64_t total;
        const int bin = kBins - 2 - 2 * tid;  // this thread's two bins: bin + 1, then bin
        const uint32_t c1 = s_hist[bin + 1], c0 = s_hist[bin];
        const uint32_t above = (uint32_t)block_scan(c0 + c1, s_scan, &total);
        if (above < left && above + c1 >= left) s_found[0] = bin + 1, s_found[1] = left - above;
        else if (above + c1 < left && above + c1 + c0 >= left) s_found[0] = bin, s_found[1] = left - above - c1;
        __syncthreads();
        prefix = (prefix << bits) | s_found[0];
        left = s_found[1];
        known += bits;
      }
    }
    // this thread's run of positions
    const int run = (n + kSelThreads - 1) / kSelThreads, r0 = s + min(n, tid * run), r1 = s + min(n, (tid + 1) * run);
    uint32_t above = 0, equal = 0;
    for (int i = r0; i < r1; ++i) {
      if (i < lo || i >= hi) {
        ++above;
      } else if (m > 0) {
        const uint32_t k = weight_key(w[i]);
        above += k > prefix;
        equal += k == prefix;
      }
    }
    uint64_t total;
    const uint64_t before = block_scan((uint64_t)equal << 32 | above, s_scan, &total);
    uint32_t at_above = (uint32_t)before, at_equal = (uint32_t)(before >> 32);
    for (int i = r0; i < r1; ++i) {
      bool stays = i < lo || i >= hi, same = false;
      if (!stays && m > 0) {
        const uint32_t k = weight_key(w[i]);
        stays = k > prefix;
        same = k == prefix;
      }
      if (stays || (same && at_equal < left)) index[at_above + min(at_equal, left)] = i;
      at_above += stays;
      at_equal += same;
    }
  }
  // Every workgroup of the row has to see seq_lens before one of them may write lens over it: lens of a row is written by
  // kv_lens_kernel, after this launch.
  if (p.wo == nullptr) return;
  float* const wo = p.wo + (int64_t)b * p.wo_sb + (int64_t)h * p.wo_sh;
  // index[d] >= d and ascends, so a chunk that is read whole before it is written never overwrites what a later one reads
  for (int d0 = 0; d0 < kept; d0 += kSelThreads) {
    __syncthreads();  // index is written (first chunk); the chunk before is read
    const int d = d0 + tid;
    const float x = d < kept ? w[index[d]] : 0.f;
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
    if (d < kept) wo[d] = x;
  }
  for (int d = kept + tid; d < e; d += kSelThreads) wo[d] = 0.f;
}

__global__ void __launch_bounds__(kWave) kv_lens_kernel(const SelectParams p, int batch) {
  const int b = blockIdx.x * kWave + threadIdx.x;
  if (b >= batch) return;
  const int e = min(max(p.seq_lens[b], 0), p.cap);
  const int s = p.kv_start ? min(max(p.kv_start[b], 0), e) : 0;
  p.lens[b] = min(e - s, p.keep);
}

// ---------------------------------------------------------------------------------------------------- compaction
//
// Row d of dst is row index[d] of src. In place (index ascends, index[d] >= d) a step of rows is read whole before it is
// written, and no later step reads what it writes; the steps of one (row, head) follow each other, so the parallelism comes
// from the columns: a workgroup takes `lanes` vectors of every row. Otherwise the steps are independent and spread over
// workgroups too.

constexpr int kMoveThreads = 256, kMoveU = 8;

struct MoveParams {
  bz_kv_tensor t[BZ_KV_TENSORS];
  int slices[BZ_KV_TENSORS];   // column slices of each tensor
  int first[BZ_KV_TENSORS];    // its first slice in grid.x
  int lanes[BZ_KV_TENSORS];    // vectors of a slice
  int vec[BZ_KV_TENSORS];      // bytes of a vector
  int in_place[BZ_KV_TENSORS];
  int num, cap, keep, NKV;
  const int32_t *index, *lens;
};

template <class V>
__device__ void move_rows(const MoveParams& p, const bz_kv_tensor& t, const char* src, char* dst, const int32_t* index,
                          int len, int slice, int lanes, bool in_place) {
  const int rows = kMoveThreads / lanes, r = threadIdx.x / lanes, c = slice * lanes + (int)threadIdx.x % lanes;
  const bool mine = r < rows && (int64_t)c * (int)sizeof(V) < t.row_bytes;
  const int step = rows * kMoveU;
  const int d_begin = in_place ? 0 : (int)blockIdx.y * step, d_end = in_place ? len : min(len, d_begin + step);
  for (int d0 = d_begin; d0 < d_end; d0 += step) {
    V x[kMoveU];
    bool put[kMoveU];
#pragma unroll
    for (int u = 0; u < kMoveU; ++u) {
      const int d = d0 + u * rows + r;
      put[u] = false;
      if (mine && d < len) {
        const int i = index[d];
        put[u] = i >= 0 && i < p.cap && !(in_place && i == d);
        if (put[u]) x[u] = *reinterpret_cast<const V*>(src + i * t.src_stride_s + c * (int64_t)sizeof(V));
      }
    }
    if (in_place) {
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kMoveU; ++u)
      if (put[u]) *reinterpret_cast<V*>(dst + (int64_t)(d0 + u * rows + r) * t.dst_stride_s + c * (int64_t)sizeof(V)) = x[u];
  }
}

__global__ void __launch_bounds__(kMoveThreads) kv_compact_kernel(const MoveParams p) {
  int k = 0;
  while (k + 1 < p.num && (int)blockIdx.x >= p.first[k + 1]) ++k;
  const bz_kv_tensor& t = p.t[k];
  const bool in_place = p.in_place[k];
  if (in_place && blockIdx.y > 0) return;
  const int h = blockIdx.z % p.NKV, b = blockIdx.z / p.NKV;
  const int len = min(p.lens[b], p.keep);
  const char* const src = static_cast<const char*>(t.src) + b * t.src_stride_b + h * t.src_stride_h;
  char* const dst = static_cast<char*>(t.dst) + b * t.dst_stride_b + h * t.dst_stride_h;
  const int32_t* const index = p.index + ((int64_t)b * p.NKV + h) * p.keep;
  const int slice = blockIdx.x - p.first[k], lanes = p.lanes[k];
  switch (p.vec[k]) {
    case 16: move_rows<uint4>(p, t, src, dst, index, len, slice, lanes, in_place); break;
    case 8: move_rows<uint2>(p, t, src, dst, index, len, slice, lanes, in_place); break;
    case 4: move_rows<uint32_t>(p, t, src, dst, index, len, slice, lanes, in_place); break;
    case 2: move_rows<uint16_t>(p, t, src, dst, index, len, slice, lanes, in_place); break;
    default: move_rows<uint8_t>(p, t, src, dst, index, len, slice, lanes, in_place); break;
  }
}

}  // namespace

#define BZ_EXPORT __attribute__((visibility("default")))

extern "C" {

BZ_EXPORT int bz_kv_select(const bz_kv_select_args* a, hipStream_t stream) {
  if (a == nullptr || a->weights == nullptr || a->seq_lens == nullptr || a->index == nullptr || a->lens == nullptr)
    return BZ_ERR_NULL;
  if (a->batch <= 0 || a->num_kv_heads <= 0 || a->capacity <= 0 || a->keep <= 0 || a->keep > a->capacity || a->sinks < 0 ||
      a->recent < 0 || (int64_t)a->sinks + a->recent > a->keep || a->batch > 65535)
    return BZ_ERR_SHAPE;
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a->weights) | reinterpret_cast<uintptr_t>(a->weights_out) |
                         reinterpret_cast<uintptr_t>(a->seq_lens) | reinterpret_cast<uintptr_t>(a->kv_start) |
                         reinterpret_cast<uintptr_t>(a->index) | reinterpret_cast<uintptr_t>(a->lens);
  if (ptrs & 3) return BZ_ERR_ALIGNMENT;
  SelectParams p{};
  p.w = a->weights, p.w_sb = a->w_stride_b, p.w_sh = a->w_stride_h;
  p.seq_lens = a->seq_lens, p.kv_start = a->kv_start;
  p.index = a->index, p.lens = a->lens;
  p.wo = a->weights_out, p.wo_sb = a->wo_stride_b, p.wo_sh = a->wo_stride_h;
  p.NKV = a->num_kv_heads, p.cap = a->capacity, p.keep = a->keep, p.sinks = a->sinks, p.recent = a->recent;
  hipLaunchKernelGGL(kv_select_kernel, dim3(a->num_kv_heads, a->batch), dim3(kSelThreads), 0, stream, p);
  if (hipGetLastError() != hipSuccess) return BZ_ERR_LAUNCH;
  hipLaunchKernelGGL(kv_lens_kernel, dim3((a->batch + kWave - 1) / kWave), dim3(kWave), 0, stream, p, a->batch);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

BZ_EXPORT int bz_kv_compact(const bz_kv_tensor* tensors, int32_t num_tensors, const int32_t* index, const int32_t* lens,
                            int32_t batch, int32_t num_kv_heads, int32_t capacity, int32_t keep, hipStream_t stream) {
  if (tensors == nullptr || index == nullptr || lens == nullptr) return BZ_ERR_NULL;
  if (num_tensors <= 0 || num_tensors > BZ_KV_TENSORS || batch <= 0 || num_kv_heads <= 0 || capacity <= 0 || keep <= 0 ||
      keep > capacity || (int64_t)batch * num_kv_heads > 65535)
    return BZ_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(index) | reinterpret_cast<uintptr_t>(lens)) & 3) return BZ_ERR_ALIGNMENT;
  MoveParams p{};
  int grid_x = 0, grid_y = 1;
  for (int k = 0; k < num_tensors; ++k) {
    const bz_kv_tensor& t = tensors[k];
    if (t.src == nullptr || t.dst == nullptr) return BZ_ERR_NULL;
    if (t.row_bytes <= 0 || t.src_stride_s < t.row_bytes || t.dst_stride_s < t.row_bytes) return BZ_ERR_SHAPE;
    p.t[k] = t;
    p.in_place[k] = t.src == t.dst;
    if (p.in_place[k] && (t.src_stride_b != t.dst_stride_b || t.src_stride_h != t.dst_stride_h || t.src_stride_s != t.dst_stride_s))
      return BZ_ERR_SHAPE;
    // the widest vector that divides every row's address and length
    const uint64_t all = reinterpret_cast<uintptr_t>(t.src) | reinterpret_cast<uintptr_t>(t.dst) | (uint64_t)t.src_stride_b |
                         (uint64_t)t.src_stride_h | (uint64_t)t.src_stride_s | (uint64_t)t.dst_stride_b |
                         (uint64_t)t.dst_stride_h | (uint64_t)t.dst_stride_s | (uint64_t)t.row_bytes;
    int vec = 16;
    while (all % vec) vec /= 2;
    const int vectors = t.row_bytes / vec;
    int lanes = 1;
    const int most = p.in_place[k] ? 4 : 16;
    while (lanes < vectors && lanes < most) lanes *= 2;
    p.vec[k] = vec;
    p.lanes[k] = lanes;
    p.slices[k] = (vectors + lanes - 1) / lanes;
    p.first[k] = grid_x;
    grid_x += p.slices[k];
    if (!p.in_place[k]) {
      const int step = kMoveThreads / lanes * kMoveU, chunks = (keep + step - 1) / step;
      if (chunks > grid_y) grid_y = chunks;
    }
  }
  if (grid_y > 65535) return BZ_ERR_SHAPE;
  p.num = num_tensors, p.cap = capacity, p.keep = keep, p.NKV = num_kv_heads, p.index = index, p.lens = lens;
  hipLaunchKernelGGL(kv_compact_kernel, dim3(grid_x, grid_y, batch * num_kv_heads), dim3(kMoveThreads), 0, stream, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

}  // extern "C"
