// Eviction from a KV cache by accumulated attention weight (include/bz_long_cache.h): which positions of each (row, kv
// head) stay (bz_kv_select), and the cache's rows moved together (bz_kv_compact).
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "bz_long_cache.h"
#include "device_common.cuh"

namespace {

constexpr int kMaxCapacity = 1 << 30;  // sums of positions and strip sizes stay in 32 bits

// ---------------------------------------------------------------------------------------------------- selection
//
// One workgroup per (row, kv head). The threshold is the m-th largest key of the middle positions (m = keep - sinks -
// recent), found by a radix selection from the top digit down (11 + 11 + 10 bits: a histogram in LDS, then the digit
// that holds the m-th key); every key above it stays, and as many equal ones, from the lowest position on, as are still
// missing. The kept positions' places in ascending order come from ballots: one count per wave and strip of 1024
// positions, one scan over those.
//
// A row's bytes are few (4 a position) and one workgroup reads them all, so its latencies are the bound: a row of up to
// 1024 IPT positions is loaded once, all loads at a time, and everything after works from registers. A longer one goes
// through in chunks of that many, loaded again for each pass. 32 (row, head) pairs of 7000..8192, keep 4096: 10.0 us (three
// passes of about 2 us between barriers, launch and first loads 3; with keys held beside the weights, not worked out anew in
// each pass, from 10.7).

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
  int NKV, cap, keep, sinks, recent, write_lens;
};

// Order-preserving map of float to uint32; NaN above everything, -0 as 0.
__device__ __forceinline__ uint32_t weight_key(float f) {
  const uint32_t u = __float_as_uint(f);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (u & 0x7fffffffu) > 0x7f800000u ? 0xffffffffu : (u & 0x7fffffffu) == 0 ? 0x80000000u : k;
}

// Exclusive sum of x over the workgroup's threads. s: kSelWaves words of LDS that no earlier read is still at.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* s) {
  static_assert(kSelWaves == 16, "one row of lanes scans the waves' sums");
  const int lane = threadIdx.x % kWave, w = wave_uniform((int)threadIdx.x / kWave);
  const uint32_t v = wave_scan(x);
  if (lane == kWave - 1) s[w] = v;
  __syncthreads();
  const uint32_t sums = row_scan(s[lane % 16]);
  return (w > 0 ? (uint32_t)__builtin_amdgcn_readlane((int)sums, w - 1) : 0u) + v - x;
}

// How many lanes below this one a ballot holds.
__device__ __forceinline__ uint32_t lanes_below(uint64_t m) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}

template <int IPT>
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const SelectParams p) {
  constexpr int kCounts = IPT * kSelWaves, kChunk = IPT * kSelThreads;
  __shared__ uint32_t s_hist[kBins];
  __shared__ uint32_t s_scan[3][kSelWaves];
  __shared__ uint32_t s_found[3][2];
  __shared__ uint32_t s_count[kCounts];  // positions that stay (low half) and that are at the threshold (high half)
  __shared__ uint32_t s_base[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid % kWave, wv = tid / kWave;
  const int e = min(max(p.seq_lens[b], 0), p.cap);
  const int s = p.kv_start ? min(max(p.kv_start[b], 0), e) : 0;
  const int n = e - s, kept = min(n, p.keep);
  const float* const w = p.w + (int64_t)b * p.w_sb + (int64_t)h * p.w_sh;
  float* const wo = p.wo ? p.wo + (int64_t)b * p.wo_sb + (int64_t)h * p.wo_sh : nullptr;
  int32_t* const index = p.index + ((int64_t)b * p.NKV + h) * p.keep;

  // a chunk's weights: strip i holds the positions c0 + 1024 i .. + 1023, one a thread
  const int lo = s + p.sinks, hi = e - p.recent;  // the middle, of which positions stay by weight
  float x[IPT];
  constexpr bool kHold = IPT <= 16;    // the keys as well (with 32 strips there are no registers for both)
  uint32_t key[kHold ? IPT : 1], middle = 0;  // bit i: strip i's position lies in the middle (held as well)
  auto key_of = [&](int i) { return kHold ? key[i] : weight_key(x[i]); };
  auto in_middle = [&](int i, int c0) {
    const int pos = c0 + i * kSelThreads + tid;
    return kHold ? (middle >> i & 1) != 0 : pos >= lo && pos < hi;
  };
  auto load = [&](int c0) {
#pragma unroll
    for (int i = 0; i < IPT; ++i) x[i] = w[max(min(c0 + i * kSelThreads + tid, e - 1), 0)];  // past the row: unused
    if constexpr (kHold) {
      middle = 0;
#pragma unroll
      for (int i = 0; i < IPT; ++i) {
        const int pos = c0 + i * kSelThreads + tid;
        key[i] = weight_key(x[i]);
        middle |= pos >= lo && pos < hi ? 1u << i : 0u;
      }
    }
  };
  load(s);
  const uint32_t m = n > p.keep ? (uint32_t)(p.keep - p.sinks - p.recent) : 0u;
  uint32_t prefix = 0, left = m;  // the threshold's top bits; how many of the keys with those bits stay
  if (m > 0) {                    // then hi - lo > m
    for (int i = tid; i < kBins; i += kSelThreads) s_hist[i] = 0;
    int known = 0;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10, shift = 32 - known - bits;
      __syncthreads();
      for (int c0 = s; c0 < e; c0 += kChunk) {
        if (n > kChunk && (pass > 0 || c0 > s)) load(c0);
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
          if (in_middle(i, c0) && (pass == 0 || key_of(i) >> (32 - known) == prefix)) {
            // lanes that all have one digit count at once (rows of 8192 equal weights: 27.7 us without this)
            const uint32_t digit = (key_of(i) >> shift) & ((1u << bits) - 1), one = __builtin_amdgcn_readfirstlane(digit);
            const uint64_t lanes = __ballot(true);
            if (__ballot(digit != one) != 0) atomicAdd(&s_hist[digit], 1u);
            else if (lanes_below(lanes) == 0) atomicAdd(&s_hist[digit], (uint32_t)__popcll(lanes));
          }
        }
      }
      __syncthreads();
      // the digit with fewer than `left` keys above it and at least `left` from it on: thread t sums two bins from the top
      const int bin = kBins - 2 - 2 * tid;
      const uint32_t c1 = s_hist[bin + 1], c0 = s_hist[bin];
      s_hist[bin + 1] = s_hist[bin] = 0;
      const uint32_t above = block_scan(c0 + c1, s_scan[pass]);
      if (above < left && above + c1 >= left) s_found[pass][0] = bin + 1, s_found[pass][1] = left - above;
      else if (above + c1 < left && above + c1 + c0 >= left) s_found[pass][0] = bin, s_found[pass][1] = left - above - c1;
      __syncthreads();
      prefix = (prefix << bits) | s_found[pass][0];
      left = s_found[pass][1];
      known += bits;
    }
  }
  // Each strip's places. A chunk writes at most up to its own first positions, so wo may be w: what a later chunk reads lies
  // behind, and this one has been read before the barriers.
  uint32_t before = 0, ties_before = 0;  // in the chunks before
  for (int c0 = s; c0 < e; c0 += kChunk) {
    if (n > kChunk && (m > 0 || c0 > s)) load(c0);
    uint32_t above = 0, equal = 0;  // bit i: strip i's position stays, or is at the threshold
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int pos = c0 + i * kSelThreads + tid;
      const uint32_t k = key_of(i);
      const bool ends = n <= p.keep || !in_middle(i, c0);
      const bool stays = pos < e && (ends || (m > 0 && k > prefix)), ties = pos < e && !ends && m > 0 && k == prefix;
      above |= stays ? 1u << i : 0u;
      equal |= ties ? 1u << i : 0u;
      const uint32_t c = (uint32_t)__popcll(__ballot(stays)) | (uint32_t)__popcll(__ballot(ties)) << 16;
      if (lane == 0) s_count[i * kSelWaves + wv] = c;
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);  // the chunk's weights are here before anyone writes wo
    __syncthreads();
    if (wv == 0) {  // exclusive sums over the counts, kCounts / 64 a lane; the halves stay below 2^16 (a chunk has 2^15)
      constexpr int PER = kCounts / kWave;
      uint32_t c[PER], sum = 0;
#pragma unroll
      for (int q = 0; q < PER; ++q) c[q] = s_count[PER * lane + q], sum += c[q];
      uint32_t acc = wave_scan(sum) - sum;
#pragma unroll
      for (int q = 0; q < PER; ++q) s_count[PER * lane + q] = acc, acc += c[q];
      if (lane == kWave - 1) s_base[0] = acc & 0xffffu, s_base[1] = acc >> 16;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const bool stays = (above >> i) & 1, ties = (equal >> i) & 1;
      const uint32_t c = s_count[i * kSelWaves + wv];
      const uint32_t at = before + (c & 0xffffu) + lanes_below(__ballot(stays));
      const uint32_t tie = ties_before + (c >> 16) + lanes_below(__ballot(ties));
      if (stays || (ties && tie < left)) {
        const int d = (int)(at + min(tie, left));
        index[d] = c0 + i * kSelThreads + tid;
        if (wo != nullptr) wo[d] = x[i];
      }
    }
    before += s_base[0], ties_before += s_base[1];
    __syncthreads();
  }
  for (int d = kept + tid; d < p.keep; d += kSelThreads) index[d] = -1;
  if (p.write_lens && h == 0 && tid == 0) p.lens[b] = kept;
  if (wo != nullptr)
    for (int d = kept + tid; d < e; d += kSelThreads) wo[d] = 0.f;
}

// lens of a call that writes it over seq_lens: after every workgroup of the launch before has read those.
__global__ void __launch_bounds__(kWave) kv_lens_kernel(const SelectParams p, int batch) {
  const int b = blockIdx.x * kWave + threadIdx.x;
  if (b >= batch) return;
  const int e = min(max(p.seq_lens[b], 0), p.cap);
  const int s = p.kv_start ? min(max(p.kv_start[b], 0), e) : 0;
  p.lens[b] = min(e - s, p.keep);
}

using SelectFn = void (*)(const SelectParams);
// The fewest registers that hold a row of the capacity (of the first 32768 positions of a longer one).
SelectFn pick_select(int cap) {
  if (cap <= 4 * kSelThreads) return kv_select_kernel<4>;
  if (cap <= 8 * kSelThreads) return kv_select_kernel<8>;
  if (cap <= 16 * kSelThreads) return kv_select_kernel<16>;
  return kv_select_kernel<32>;
}

// ---------------------------------------------------------------------------------------------------- compaction
//
// Row d of dst is row index[d] of src. In place (index ascends, index[d] >= d) a step of rows is read whole before it is
// written, and no later step reads what it writes; the steps of one (row, head) follow each other, so the parallelism comes
// from the columns: a workgroup takes `lanes` vectors of every row, 128 bytes, one line (us, K and V of 4 rows x 8 heads, 4096
// kept of 256 bytes: 64 bytes 43.6, 128 30.3, 256 43.3; 32 bytes 122), with 1024 threads, whose wide steps are few (256
// threads at 64 bytes 39.7; 1 row x 8 heads 28.0, now 21.2). Otherwise the steps are independent and spread over workgroups
// too. Bound by memory: the first of these, 134 MB read and written, to other tensors 23.5 to 25.5 us, 5.2 to 5.7 TB/s (a large
// copy: 5.0); in place by the steps' round trips where rows are few.

constexpr int kMaxRowBytes = 1 << 28, kMaxKeep = 65535 * 128;  // one vector of a byte a slice, 128 rows a workgroup at least
constexpr int kMoveU = 8;  // rows of a thread in flight
constexpr int move_threads(bool in_place) { return in_place ? 1024 : 256; }
typedef uint32_t vec8 __attribute__((ext_vector_type(2)));
typedef uint32_t vec16 __attribute__((ext_vector_type(4)));

struct MoveParams {
  bz_kv_tensor t[BZ_KV_TENSORS];
  int slices[BZ_KV_TENSORS];   // column slices of each tensor
  int first[BZ_KV_TENSORS];    // its first slice in grid.x
  int lanes[BZ_KV_TENSORS];    // vectors of a slice
  int vec[BZ_KV_TENSORS];      // bytes of a vector
  int num, cap, keep, NKV;
  const int32_t *index, *lens;
};

template <class V, bool IN>
__device__ __forceinline__ void move_rows(const bz_kv_tensor& t, const char* src, char* dst, const int32_t* index, int cap,
                                          int len, int slice, int lanes) {
  constexpr int U = kMoveU;
  const int rows = move_threads(IN) / lanes, r = threadIdx.x / lanes, c = slice * lanes + (int)threadIdx.x % lanes;
  const int64_t col = (int64_t)c * (int)sizeof(V);
  const bool mine = col < t.row_bytes;
  const int step = rows * U;
  const int d_begin = IN ? 0 : (int)blockIdx.y * step, d_end = IN ? len : min(len, d_begin + step);
  for (int d0 = d_begin; d0 < d_end; d0 += step) {
    V x[U];
    int from[U];
#pragma unroll
    for (int u = 0; u < U; ++u) from[u] = index[min(d0 + u * rows + r, len - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // every load without a condition; an index that is none reads row 0, unused
      const int64_t i = from[u] >= 0 && from[u] < cap ? from[u] : 0;
      x[u] = __builtin_nontemporal_load(reinterpret_cast<const V*>(src + i * t.src_stride_s + (mine ? col : 0)));
    }
    if constexpr (IN) {
      __builtin_amdgcn_s_waitcnt(0x0f70);
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int d = d0 + u * rows + r;
      if (mine && d < len && from[u] >= 0 && from[u] < cap && !(IN && from[u] == d))
        __builtin_nontemporal_store(x[u], reinterpret_cast<V*>(dst + d * t.dst_stride_s + col));
    }
  }
}

template <bool IN>
__global__ void __launch_bounds__(move_threads(IN)) kv_compact_kernel(const MoveParams p) {
  int k = 0;
  while (k + 1 < p.num && (int)blockIdx.x >= p.first[k + 1]) ++k;
  const bz_kv_tensor& t = p.t[k];
  const int h = blockIdx.z % p.NKV, b = blockIdx.z / p.NKV;
  const int len = min(p.lens[b], p.keep);
  const char* const src = static_cast<const char*>(t.src) + b * t.src_stride_b + h * t.src_stride_h;
  char* const dst = static_cast<char*>(t.dst) + b * t.dst_stride_b + h * t.dst_stride_h;
  const int32_t* const index = p.index + ((int64_t)b * p.NKV + h) * p.keep;
  const int slice = blockIdx.x - p.first[k], lanes = p.lanes[k];
  switch (p.vec[k]) {
    case 16: move_rows<vec16, IN>(t, src, dst, index, p.cap, len, slice, lanes); break;
    case 8: move_rows<vec8, IN>(t, src, dst, index, p.cap, len, slice, lanes); break;
    case 4: move_rows<uint32_t, IN>(t, src, dst, index, p.cap, len, slice, lanes); break;
    case 2: move_rows<uint16_t, IN>(t, src, dst, index, p.cap, len, slice, lanes); break;
    default: move_rows<uint8_t, IN>(t, src, dst, index, p.cap, len, slice, lanes); break;
  }
}

// The tensors that move in place, or the others, in one launch.
template <bool IN>
int launch_moves(const bz_kv_tensor* tensors, int num, MoveParams& p, int batch, hipStream_t stream) {
  int64_t grid_x = 0, grid_y = 1;
  p.num = 0;
  for (int i = 0; i < num; ++i) {
    const bz_kv_tensor& t = tensors[i];
    if ((t.src == t.dst) != IN) continue;
    const int k = p.num++;
    p.t[k] = t;
    // the widest vector that divides every row's address and length
    const uint64_t all = reinterpret_cast<uintptr_t>(t.src) | reinterpret_cast<uintptr_t>(t.dst) | (uint64_t)t.src_stride_b |
                         (uint64_t)t.src_stride_h | (uint64_t)t.src_stride_s | (uint64_t)t.dst_stride_b |
                         (uint64_t)t.dst_stride_h | (uint64_t)t.dst_stride_s | (uint64_t)t.row_bytes;
    int vec = 16;
    while (all % vec) vec /= 2;
    const int vectors = t.row_bytes / vec, most = IN ? 8 : 16;
    int lanes = 1;
    while (lanes < vectors && lanes < most) lanes *= 2;
    p.vec[k] = vec;
    p.lanes[k] = lanes;
    p.slices[k] = (vectors + lanes - 1) / lanes;
    p.first[k] = (int)grid_x;
    grid_x += p.slices[k];
    if (!IN) {
      const int step = move_threads(IN) / lanes * kMoveU;
      grid_y = std::max<int64_t>(grid_y, (p.keep + step - 1) / step);
    }
  }
  if (p.num == 0) return BZ_OK;
  hipLaunchKernelGGL(kv_compact_kernel<IN>, dim3((unsigned)grid_x, (unsigned)grid_y, batch * p.NKV), dim3(move_threads(IN)), 0, stream,
                     p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

}  // namespace

#define BZ_EXPORT __attribute__((visibility("default")))

extern "C" {

BZ_EXPORT int bz_kv_select(const bz_kv_select_args* a, hipStream_t stream) {
  if (a == nullptr || a->weights == nullptr || a->seq_lens == nullptr || a->index == nullptr || a->lens == nullptr)
    return BZ_ERR_NULL;
  if (a->batch <= 0 || a->num_kv_heads <= 0 || a->capacity <= 0 || a->keep <= 0 || a->keep > a->capacity || a->sinks < 0 ||
      a->recent < 0 || (int64_t)a->sinks + a->recent > a->keep || a->batch > 65535 || a->capacity > kMaxCapacity)
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
  // workgroups of a row read seq_lens and kv_start; lens that lies on either is written by a launch of its own
  auto apart = [&](const int32_t* x) { return x == nullptr || a->lens + a->batch <= x || x + a->batch <= a->lens; };
  for (const int32_t* x : {a->seq_lens, a->kv_start})  // shifted over it, one row's lens would be another's end
    if (!apart(x) && a->lens != x) return BZ_ERR_SHAPE;
  p.write_lens = apart(a->seq_lens) && apart(a->kv_start);
  hipLaunchKernelGGL(pick_select(a->capacity), dim3(a->num_kv_heads, a->batch), dim3(kSelThreads), 0, stream, p);
  if (hipGetLastError() != hipSuccess) return BZ_ERR_LAUNCH;
  if (p.write_lens) return BZ_OK;
  hipLaunchKernelGGL(kv_lens_kernel, dim3((a->batch + kWave - 1) / kWave), dim3(kWave), 0, stream, p, a->batch);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

BZ_EXPORT int bz_kv_compact(const bz_kv_tensor* tensors, int32_t num_tensors, const int32_t* index, const int32_t* lens,
                            int32_t batch, int32_t num_kv_heads, int32_t capacity, int32_t keep, hipStream_t stream) {
  if (tensors == nullptr || index == nullptr || lens == nullptr) return BZ_ERR_NULL;
  if (num_tensors <= 0 || num_tensors > BZ_KV_TENSORS || batch <= 0 || num_kv_heads <= 0 || capacity <= 0 || keep <= 0 ||
      keep > capacity || capacity > kMaxCapacity || (int64_t)batch * num_kv_heads > 65535)
    return BZ_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(index) | reinterpret_cast<uintptr_t>(lens)) & 3) return BZ_ERR_ALIGNMENT;
  for (int k = 0; k < num_tensors; ++k) {
    const bz_kv_tensor& t = tensors[k];
    if (t.src == nullptr || t.dst == nullptr) return BZ_ERR_NULL;
    if (t.row_bytes <= 0 || t.src_stride_s < t.row_bytes || t.dst_stride_s < t.row_bytes) return BZ_ERR_SHAPE;
    if (t.row_bytes > kMaxRowBytes) return BZ_ERR_SHAPE;  // grid limits
    if (t.src == t.dst &&
        (t.src_stride_b != t.dst_stride_b || t.src_stride_h != t.dst_stride_h || t.src_stride_s != t.dst_stride_s))
      return BZ_ERR_SHAPE;
  }
  if (keep > kMaxKeep) return BZ_ERR_SHAPE;
  MoveParams p{};
  p.cap = capacity, p.keep = keep, p.NKV = num_kv_heads, p.index = index, p.lens = lens;
  const int rc = launch_moves<false>(tensors, num_tensors, p, batch, stream);
  return rc == BZ_OK ? launch_moves<true>(tensors, num_tensors, p, batch, stream) : rc;
}

}  // extern "C"
