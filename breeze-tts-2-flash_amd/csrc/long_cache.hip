// Host side of include/bz_long_cache.h's attention: argument checks, workspace layout, split counts, launches. The device
// code is in long_cache.cuh.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "bz_long_cache.h"
#include "long_cache.cuh"
#include "window_prefill.cuh"

namespace bz {
int device_cu_count(int* cus);  // gqa_decode.hip
}

namespace {

// Threads of a split workgroup. Eight waves measured 6% faster on long rows of 4 bits (4 rows x 4 kv heads of 20001..32768,
// G 8: 17.9 against 19.0 us) and 2 to 40% slower on everything else.
constexpr int kLongThreads = 256;
// Rows up to which the merging workgroup of a tracked step adds the weights itself (the two turns of its threads whose scores it
// loads with the partials), in place of a second launch (us, second launch / itself, 2 x 8 kv heads, G 2: 500 positions 8.5 /
// 6.5, 1377 10.4 / 8.6, 2048 10.7 / 9.3, 2600 12.2 / 12.0, 4096 13.3 / 14.8; G 8, 1 x 8 x 1024 10.3 / 8.2, 2048 12.4 / 11.0).
constexpr int kFusePositions = 2048;
// Bytes of the longest row a split takes from which on splits are dealt (4 rows of 20001..32768 of 4 bits, 16 splits, 278 KB:
// 18.6 us dealt or not; 16 rows of 128..2048, 2 splits, 139 KB: 10.9 dealt, 10.7 not).
constexpr int64_t kDealBytes = 1 << 18;
constexpr int kCounterLines = BZ_LONG_SHARED_UNITS;
constexpr int kMaxTokens = 1 << 30;  // sums of tokens and tile sizes stay in 32 bits
constexpr int kKv4Tokens = 16;  // most query tokens per row over a 4-bit cache

bool dim_ok(int D) { return D == 64 || D == 128; }
bool group_ok(int G) { return G == 1 || G == 2 || G == 4 || G == 8; }
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// What a call's sizes determine: the column tiles, the splits and where things lie in the workspace (its arrival
// counters first, one 256-byte line per (row, column tile, kv head); they are zero between calls, everything else is
// written before it is read).
struct Plan {
  bool prefill;  // gqa_window: the chunk kernel; unsplit, it needs no workspace
  int cgroups;   // its column groups
  bool balanced; // splits are dealt to the rows by their lengths
  int G, gshift, tpt, tiles, splits, min_tiles, one_split, score_stride;
  int64_t units;
  size_t ml, acc, head_ml, scores, total;
};

int make_plan(int kind, int B, int NH, int NKV, int D, int cap, int T, int window, int sinks, int num_splits, int max_seq_len,
              Plan* pl) {
  if (B <= 0 || NH <= 0 || NKV <= 0 || cap <= 0 || T <= 0 || NH % NKV != 0 || window < 0 || sinks < 0) return BZ_ERR_SHAPE;
  if (T > kMaxTokens || cap > kMaxTokens) return BZ_ERR_SHAPE;
  if (num_splits < 0 || num_splits > kMaxSplits) return BZ_ERR_SHAPE;
  if (!dim_ok(D) || !group_ok(NH / NKV)) return BZ_ERR_UNSUPPORTED;
  if (kind == BZ_LONG_KV4 && T > kKv4Tokens) return BZ_ERR_UNSUPPORTED;
  if (kind == BZ_LONG_TRACKED && T != 1) return BZ_ERR_UNSUPPORTED;
  const bool kv4 = kind == BZ_LONG_KV4;
  pl->G = NH / NKV;
  pl->gshift = __builtin_ctz(pl->G);
  pl->tpt = kLongCols / pl->G < T ? kLongCols / pl->G : T;
  pl->tiles = (T + pl->tpt - 1) / pl->tpt;
  pl->units = (int64_t)B * pl->tiles * NKV;
  int cus = 0;
  if (num_splits == 0 || (kind == BZ_LONG_WINDOW && pl->tiles > 1)) {
    const int rc = bz::device_cu_count(&cus);
    if (rc != BZ_OK) return rc;
  }
  // positions a row holds, and those a column tile attends
  const int64_t longest = max_seq_len > 0 && max_seq_len < cap ? max_seq_len : cap;
  auto attended = [&](int64_t tokens) { return window > 0 ? std::min(longest, (int64_t)window + tokens + sinks) : longest; };

  // the counters' room: a power of two of lines, at least kCounterLines, so that all calls of one room can share a workspace and a
  // server's batches, whatever their sizes, need a few (exact, every batch of more than 64 rows of 8 kv heads had its own)
  int64_t lines = kCounterLines;
  while (lines < pl->units) lines *= 2;
  const size_t counters = (size_t)lines * kCounterStride * sizeof(int);
  pl->prefill = pl->balanced = false;
  if (kind == BZ_LONG_WINDOW && pl->tiles > 1) {
    auto tiles = [&](int cg) { return ((int64_t)T * pl->G + kPreWaveCols * cg - 1) / (kPreWaveCols * cg); };
    const int64_t rows = (int64_t)B * NKV, wide = tiles(4) * rows, steps = attended(4 * kPreWaveCols / pl->G) / 64 + 1;
    // splits of a 128-column tile's positions that give `workgroups`, each of at least `least` steps of 64
    auto shares = [&](int64_t workgroups, int64_t least) { return std::max<int64_t>(std::min(workgroups / wide, steps / least), 1); };
    // a caller's: as many as find kPreMinSteps steps each (the kernel gives none fewer)
    int64_t splits = std::max<int64_t>(std::min<int64_t>(num_splits, (steps + kPreMinSteps - 1) / kPreMinSteps), 1);
    if (pl->units < cus) {
      // Few columns: the split kernel, which reads K and V again for each tile of 16 but spreads a few of them over the whole
      // device, unless the splits of whole 128-column tiles half fill it (us, split kernel / chunk kernel split, 8 kv heads,
      // head_dim 128: 256 columns, 8192 positions 45.3 / 26.5, 2048 positions 16.4 / 20.4; 128, 8192 27.1 / 24.3; 4 q heads, 64
      // tokens, 16384 82.6 / 36.0; 2 kv heads, 512 columns, 4096 16.3 / 20.4).
      const int64_t s = shares(cus, kPreMinSteps);
      pl->prefill = num_splits == 0 && (int64_t)T * pl->G >= 4 * kPreWaveCols && wide * s >= cus / 2;
      if (pl->prefill) splits = s;
    } else {
      // Otherwise the chunk kernel (us, split / chunk kernel, head_dim 128: 8 kv heads, 4096 positions, 512 columns 43.9 / 40.4;
      // 4 rows x 8, window 1024: 256 columns 23.8 / 17.1), by the widest column tiles that still give every CU work, three
      // workgroups each for the widest (us for 1 / 2 / 4 groups, head_dim 128: 2 x 8 kv heads x 2048 tokens 122.8 / 53.1 / 57.5; 8
      // x 8192, window 4096: 509 / 243 / 223; 8 x 1024: 23.1 / 18.0 / 23.6). A chunk behind a long context is split over its
      // positions as well: to two rounds where a split still has 32 steps (8 kv heads, head_dim 128, whole / split: 512
      // tokens over 16384 132 / 80, 1024 over 8192 98 / 81, 2048 over 16384 283 / 253), else to one where the column tiles fill
      // none (512 over 4096 40.6 / 34.2, 256 over 8192 70 / 33, 1024 over 1024 17.9 / 27.2). At head_dim 64, where one column group
      // leaves room for two workgroups a CU, that is only worth it for long splits if those fill it (256 over 8192 43 / 25, 512
      // over 4096 23 / 27, over 16384 78 / 61).
      pl->prefill = true;
      const bool few = D == 128 || tiles(1) * rows < cus;
      if (num_splits == 0) {
        if (wide <= cus && shares(2 * cus, 32) == 2 * cus / wide) splits = 2 * cus / wide;
        else if (tiles(2) * rows < cus) splits = shares(cus, few ? 14 : 64);
      }
    }
    if (pl->prefill) {
      pl->cgroups = splits > 1 || wide >= 3 * cus ? 4 : tiles(2) * rows >= cus ? 2 : 1;
      if (tiles(pl->cgroups) * splits > 65535 || B > 65535 || NKV > 65535) return BZ_ERR_SHAPE;  // grid limits
      pl->tiles = (int)tiles(pl->cgroups);
      pl->splits = (int)splits;
      pl->ml = pl->acc = pl->head_ml = pl->scores = pl->total = 0;
      if (splits > 1) {
        const size_t cols = (size_t)(rows * pl->tiles * splits) * 4 * kPreWaveCols;
        pl->ml = counters;  // room for those of other calls with this workspace
        pl->acc = up256(pl->ml + cols * sizeof(float2));
        pl->total = pl->acc + cols * D * sizeof(float);
      }
      return BZ_OK;
    }
  }
  if ((int64_t)B * pl->tiles > 65535 || NKV > 65535) return BZ_ERR_SHAPE;  // grid limits

  // in wave tiles
  const int64_t len = attended(pl->tpt);
  const bool cut = len < longest;  // the rows reach past the window
  const int P = kv4 ? 32 : 16;
  const int n = (int)((len + P - 1) / P) + 1;
  pl->min_tiles = kLongThreads / kWave;
  pl->one_split = (kOneSplitBytes / (kv4 ? D + D / 16 : 4 * D)) / P;
  // A server's batch: more than three rows, whose lengths differ because no window cuts them. Its splits are dealt to the rows by
  // their lengths where a split streams long enough for that to show (deal_splits costs about 0.5 us before the first load;
  // 64 rows: a lane for each). Two and three rows are taken to be alike, as those of a guidance pair are: dealt they cost a little,
  // and win where they are not (us, not dealt / dealt, 8 kv heads: 2 rows of 8192 14.5 / 14.7, of 16384 tracked 28.2 / 29.5, of
  // 20000..32768 of 4 bits, 4 kv heads of 8 q 12.6 / 15.0, of 500..8192 11.5 / 10.6, of 2000..32768 of 4 bits 16.5 / 12.5; 3 rows
  // of 8192 18.7 / 19.1, of 500..8192 15.3 / 12.9).
  const bool batch = !cut && B > 3;
  const int64_t row_bytes = kv4 ? D + D / 16 : 4 * D;
  auto dealt = [&](int64_t s) { return s > 1 && batch && (int64_t)B * pl->tiles <= kWave && len * row_bytes / s >= kDealBytes; };
  int splits = num_splits;
  if (splits == 0) {
    // One round of workgroups (us: 1 row x 8 kv heads x 8192 positions of 4 bits: 32 splits 7.5, 64 8.6; 2 rows tracked, 1377:
    // 16 splits 10.2, 32 11.1; 4 rows, window 4096: 8 splits 14.8, 16 15.3; 16 rows: 2 splits 42.1, 4 44.5). For a batch two,
    // which even its rows out (16 rows of 128..2048 of 4 bits: 2 splits 11.3, 4 10.8; 32 rows, head_dim 64: 1 split 22.9, 2
    // 18.7; dealt, 8 rows of 100..32768 of 4 bits: 4 splits 39.4, 8 33.1); over bf16 one, if that is at least four dealt splits
    // (us, 8 kv heads, head_dim 128, one round dealt / two, each row as many: 8 rows of 100..8192 27.1 / 31.9; 4 of 9000..16384
    // tracked 46.8 / 48.8; 6 of 500..8192, 4 tokens, 4 kv heads 16.1 / 20.2; fewer are too coarse to deal: 16 of 300..4096
    // tracked, 2 splits dealt 38.6, 4 34.1, 4 each 38.0).
    const int64_t round = cus / pl->units;
    splits = (int)(batch && (kv4 || round < 4 || !dealt(round)) ? 2 * cus / pl->units : round);
    const int most = (n + pl->min_tiles - 1) / pl->min_tiles;
    if (splits > most) splits = most;
    if (splits > 64) splits = 64;
    if (n <= pl->one_split || splits < 1) splits = 1;
  }
  pl->splits = splits;
  pl->balanced = dealt(splits);

  const size_t cols = (size_t)pl->units * splits * pl->tpt * pl->G;
  const bool merged = splits > 1;
  // a tracked call of one split has no use for the counters, but a later call with the same workspace finds them zero
  pl->ml = merged || kind == BZ_LONG_TRACKED ? counters : 0;
  pl->acc = up256(pl->ml + (merged ? cols * sizeof(float2) : 0));
  pl->head_ml = up256(pl->acc + (merged ? cols * D * sizeof(float) : 0));
  pl->total = pl->head_ml;
  pl->scores = 0;
  pl->score_stride = 0;
  if (kind == BZ_LONG_TRACKED) {
    pl->score_stride = (int)(((int64_t)cap + 31) & ~(int64_t)31);  // rows may be longer than max_seq_len, which steers the tiling
    pl->scores = up256(pl->head_ml + (size_t)B * NH * sizeof(float2));
    pl->total = up256(pl->scores + (size_t)B * NH * pl->score_stride * sizeof(float));
  }
  return BZ_OK;
}

int check_base(const bz_gqa_decode_args* a) {
  if (a->q == nullptr || a->k_cache == nullptr || a->v_cache == nullptr || a->out == nullptr || a->seq_lens == nullptr)
    return BZ_ERR_NULL;
  if (a->mask != nullptr || a->mask_dtype != BZ_MASK_NONE) return BZ_ERR_UNSUPPORTED;
  if (a->tokens_per_row < 0) return BZ_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(a->q) & 15) || ((a->q_stride_b | a->q_stride_h) & 7) ||
      (a->tokens_per_row > 1 && (a->q_stride_t & 7)))
    return BZ_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(a->out) & 1) || (reinterpret_cast<uintptr_t>(a->seq_lens) & 3) ||
      (reinterpret_cast<uintptr_t>(a->kv_start) & 3))
    return BZ_ERR_ALIGNMENT;
  return BZ_OK;
}

int check_bf16_cache(const bz_gqa_decode_args* a) {
  if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) return BZ_ERR_ALIGNMENT;
  if ((a->kv_stride_b | a->kv_stride_h | a->kv_stride_s) & 7) return BZ_ERR_ALIGNMENT;
  if (a->kv_stride_s < a->head_dim) return BZ_ERR_SHAPE;
  if (((int64_t)a->capacity + 1024) * a->kv_stride_s * 2 > INT32_MAX) return BZ_ERR_SHAPE;  // 32-bit byte offsets
  return BZ_OK;
}

int check_kv4_cache(const bz_kv4_cache* c) {
  if (c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr) return BZ_ERR_NULL;
  if (c->batch <= 0 || c->num_kv_heads <= 0 || c->capacity <= 0) return BZ_ERR_SHAPE;
  if (!dim_ok(c->head_dim)) return BZ_ERR_UNSUPPORTED;
  const int D = c->head_dim, code_align = D / 8 - 1, scale_align = D / 32 - 1;
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & code_align) return BZ_ERR_ALIGNMENT;
  if ((c->stride_b | c->stride_h | c->stride_s) & code_align) return BZ_ERR_ALIGNMENT;
  if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) | (uintptr_t)c->scale_stride_b |
       (uintptr_t)c->scale_stride_h) &
      scale_align)
    return BZ_ERR_ALIGNMENT;
  if (c->stride_s < D / 2) return BZ_ERR_SHAPE;
  if (((int64_t)c->capacity + 1024) * c->stride_s > INT32_MAX) return BZ_ERR_SHAPE;
  return BZ_OK;
}

int check_workspace(const bz_gqa_decode_args* a, const Plan& pl) {
  if (pl.total == 0) return BZ_OK;
  if (a->workspace == nullptr || a->workspace_bytes < pl.total) return BZ_ERR_WORKSPACE;
  return (reinterpret_cast<uintptr_t>(a->workspace) & 255) ? BZ_ERR_ALIGNMENT : BZ_OK;
}

LongParams long_params(const bz_gqa_decode_args* a, const Plan& pl, int window, int sinks) {
  LongParams p{};
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_sb = a->q_stride_b, p.q_sh = a->q_stride_h, p.q_st = a->q_stride_t;
  p.k = static_cast<const char*>(a->k_cache);
  p.v = static_cast<const char*>(a->v_cache);
  p.kv_sb = 2 * a->kv_stride_b, p.kv_sh = 2 * a->kv_stride_h, p.kv_ss = 2 * a->kv_stride_s;
  p.window = window > 0 ? window : INT32_MAX;
  p.sinks = sinks;
  p.scale_log2 = a->scale * kLog2e;
  p.out = static_cast<uint16_t*>(a->out);
  p.o_sb = a->out_stride_b, p.o_sh = a->out_stride_h, p.o_st = a->out_stride_t;
  p.out_wide = !((reinterpret_cast<uintptr_t>(a->out) & 7) || ((p.o_sb | p.o_sh | p.o_st) & 3));
  p.NKV = a->num_kv_heads, p.G = pl.G, p.gshift = pl.gshift, p.T = a->tokens_per_row > 1 ? a->tokens_per_row : 1;
  p.cap = a->capacity;
  p.tiles = pl.tiles, p.tpt = pl.tpt;
  p.rows = pl.balanced ? a->batch * pl.tiles : 0;
  p.inv_splits = 1.0f / (float)(pl.balanced ? pl.splits * p.rows : pl.splits);
  p.splits = pl.splits, p.min_tiles = pl.min_tiles, p.one_split = pl.one_split;
  char* const ws = static_cast<char*>(a->workspace);
  p.counters = reinterpret_cast<int*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + pl.ml);
  p.part_acc = reinterpret_cast<float*>(ws + pl.acc);
  p.head_ml = reinterpret_cast<float2*>(ws + pl.head_ml);
  p.scores = reinterpret_cast<float*>(ws + pl.scores);
  p.score_stride = pl.score_stride;
  return p;
}

template <int FMT, bool TRACK>
int launch_split(const bz_gqa_decode_args* a, int D, const LongParams& p, const Plan& pl, hipStream_t stream) {
  const dim3 grid = pl.balanced ? dim3(pl.splits * p.rows, p.NKV) : dim3(pl.splits, p.NKV, a->batch * pl.tiles);
  using Fn = void (*)(const int32_t*, const int32_t*, const LongParams);
  const Fn fns[2][2] = {
      {long_split_kernel<64, FMT, TRACK, false, kLongThreads>, long_split_kernel<64, FMT, TRACK, true, kLongThreads>},
      {long_split_kernel<128, FMT, TRACK, false, kLongThreads>, long_split_kernel<128, FMT, TRACK, true, kLongThreads>}};
  hipLaunchKernelGGL(fns[D == 128][pl.balanced], grid, dim3(kLongThreads), 0, stream, a->seq_lens, a->kv_start, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

int tokens_in(const bz_gqa_decode_args* a) { return a->tokens_per_row > 1 ? a->tokens_per_row : 1; }

}  // namespace

#define BZ_EXPORT __attribute__((visibility("default")))

extern "C" {

BZ_EXPORT int bz_long_workspace_size(int32_t kind, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                     int32_t capacity, int32_t tokens_per_row, int32_t window, int32_t sinks,
                                     int32_t num_splits, int32_t max_seq_len, size_t* bytes) {
  if (bytes == nullptr) return BZ_ERR_NULL;
  if (kind < BZ_LONG_WINDOW || kind > BZ_LONG_TRACKED) return BZ_ERR_SHAPE;
  Plan pl;
  const int rc = make_plan(kind, batch, num_q_heads, num_kv_heads, head_dim, capacity, tokens_per_row > 1 ? tokens_per_row : 1,
                           window, sinks, num_splits, max_seq_len, &pl);
  if (rc != BZ_OK) return rc;
  *bytes = pl.total;
  return BZ_OK;
}

BZ_EXPORT int bz_gqa_window(const bz_gqa_window_args* wa, hipStream_t stream) {
  if (wa == nullptr) return BZ_ERR_NULL;
  const bz_gqa_decode_args* a = &wa->base;
  int rc = check_base(a);
  if (rc != BZ_OK) return rc;
  Plan pl;
  rc = make_plan(BZ_LONG_WINDOW, a->batch, a->num_q_heads, a->num_kv_heads, a->head_dim, a->capacity, tokens_in(a), wa->window,
                 wa->sinks, a->num_splits, a->max_seq_len, &pl);
  if (rc == BZ_OK) rc = check_bf16_cache(a);
  if (rc == BZ_OK) rc = check_workspace(a, pl);
  if (rc != BZ_OK) return rc;
  const LongParams p = long_params(a, pl, wa->window, wa->sinks);
  if (!pl.prefill) return launch_split<kBf16, false>(a, a->head_dim, p, pl, stream);
  const dim3 grid(a->num_kv_heads, pl.tiles * pl.splits, a->batch);
  using Fn = void (*)(const int32_t*, const int32_t*, const LongParams);
  const Fn fns[2][4] = {{window_prefill_kernel<64, 1, false>, window_prefill_kernel<64, 2, false>,
                         window_prefill_kernel<64, 4, false>, window_prefill_kernel<64, 4, true>},
                        {window_prefill_kernel<128, 1, false>, window_prefill_kernel<128, 2, false>,
                         window_prefill_kernel<128, 4, false>, window_prefill_kernel<128, 4, true>}};
  const int wide = a->head_dim == 128;
  hipLaunchKernelGGL(fns[wide][pl.splits > 1 ? 3 : pl.cgroups / 2], grid, dim3(kPreThreads), 0, stream, a->seq_lens, a->kv_start, p);
  if (hipGetLastError() != hipSuccess) return BZ_ERR_LAUNCH;
  if (pl.splits == 1) return BZ_OK;
  const dim3 columns((unsigned)(((int64_t)p.T * p.G + 3) / 4), a->num_kv_heads, a->batch);
  const Fn merge = wide ? window_merge_kernel<128> : window_merge_kernel<64>;
  hipLaunchKernelGGL(merge, columns, dim3(kPreThreads), 0, stream, a->seq_lens, a->kv_start, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

BZ_EXPORT int bz_gqa_decode_kv4(const bz_gqa_kv4_args* ka, hipStream_t stream) {
  if (ka == nullptr) return BZ_ERR_NULL;
  bz_gqa_decode_args a = ka->base;
  const bz_kv4_cache* c = &ka->cache;
  int rc = check_kv4_cache(c);
  if (rc != BZ_OK) return rc;
  a.k_cache = c->k, a.v_cache = c->v;
  a.batch = c->batch, a.num_kv_heads = c->num_kv_heads, a.capacity = c->capacity, a.head_dim = c->head_dim;
  rc = check_base(&a);
  if (rc != BZ_OK) return rc;
  Plan pl;
  rc = make_plan(BZ_LONG_KV4, a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim, a.capacity, tokens_in(&a), ka->window,
                 ka->sinks, a.num_splits, a.max_seq_len, &pl);
  if (rc == BZ_OK) rc = check_workspace(&a, pl);
  if (rc != BZ_OK) return rc;
  LongParams p = long_params(&a, pl, ka->window, ka->sinks);
  p.kv_sb = c->stride_b, p.kv_sh = c->stride_h, p.kv_ss = c->stride_s;
  p.k_scale = static_cast<const uint8_t*>(c->k_scale);
  p.v_scale = static_cast<const uint8_t*>(c->v_scale);
  p.sc_sb = c->scale_stride_b, p.sc_sh = c->scale_stride_h;
  if (c->stride_s == a.head_dim / 2) return launch_split<kKv4Packed, false>(&a, a.head_dim, p, pl, stream);
  return launch_split<kKv4, false>(&a, a.head_dim, p, pl, stream);
}

BZ_EXPORT int bz_gqa_decode_tracked(const bz_gqa_tracked_args* ta, hipStream_t stream) {
  if (ta == nullptr) return BZ_ERR_NULL;
  const bz_gqa_decode_args* a = &ta->base;
  int rc = check_base(a);
  if (rc != BZ_OK) return rc;
  if (ta->weights == nullptr || ta->weights_out == nullptr) return BZ_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(ta->weights) | reinterpret_cast<uintptr_t>(ta->weights_out)) & 3) return BZ_ERR_ALIGNMENT;
  Plan pl;
  rc = make_plan(BZ_LONG_TRACKED, a->batch, a->num_q_heads, a->num_kv_heads, a->head_dim, a->capacity, tokens_in(a), 0, 0,
                 a->num_splits, a->max_seq_len, &pl);
  if (rc == BZ_OK) rc = check_bf16_cache(a);
  if (rc == BZ_OK) rc = check_workspace(a, pl);
  if (rc != BZ_OK) return rc;
  LongParams p = long_params(a, pl, 0, 0);
  p.weights = ta->weights, p.w_sb = ta->w_stride_b, p.w_sh = ta->w_stride_h;
  p.weights_out = ta->weights_out, p.wo_sb = ta->wo_stride_b, p.wo_sh = ta->wo_stride_h;
  p.decay = ta->decay;
  const int longest = a->max_seq_len > 0 && a->max_seq_len < a->capacity ? a->max_seq_len : a->capacity;
  p.fuse = longest <= kFusePositions;
  rc = launch_split<kBf16, true>(a, a->head_dim, p, pl, stream);
  if (rc != BZ_OK || p.fuse) return rc;
  const dim3 grid((longest + 4 * kApplyThreads - 1) / (4 * kApplyThreads), a->num_kv_heads, a->batch);
  hipLaunchKernelGGL(track_apply_kernel, grid, dim3(kApplyThreads), 0, stream, a->seq_lens, a->kv_start, p);
  return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
}

}  // extern "C"
