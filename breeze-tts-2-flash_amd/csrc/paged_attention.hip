// Host side of bz_gqa_paged (include/bz_paged_cache.h): argument checks, workspace layout, how the work is dealt, launches. The
// device code is in paged_split.cuh and paged_chunk.cuh.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "bz_paged_cache.h"
#include "paged_chunk.cuh"
#include "paged_split.cuh"

namespace bz {
int device_cu_count(int* cus);  // gqa_decode.hip
}

namespace {

constexpr int kFewThreads = 256;
// Workspace: the arrival counters, then (max, sum) pairs and sums of 2 * kSlotsPerCu slots a CU, at places that depend on nothing else, so
// that calls of all sizes can share one; those of the chunk kernel behind the split kernel's, as one launch may write both. A
// kernel's splits of all kv heads number at most kSlotsPerCu a CU, and those of rows that are split at most twice that (deal_paged).
constexpr int kSlotsPerCu = 2;

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

struct Parts {  // (max, sum) pairs, sums
  size_t ml, acc;
};
struct Layout {
  int64_t slots;
  Parts split, chunk;
  size_t total;
};
Layout layout(int cus, int D, int cols) {
  Layout y;
  y.slots = (int64_t)2 * kSlotsPerCu * cus;
  y.total = (size_t)y.slots * kCounterStride * sizeof(int);
  auto room = [&](int c) {
    const Parts x{y.total, up256(y.total + (size_t)y.slots * c * sizeof(float2))};
    y.total = up256(x.acc + (size_t)y.slots * c * D * sizeof(float));
    return x;
  };
  y.split = room(cols == kChunkCols ? kLongCols : cols);
  y.chunk = cols == kChunkCols ? room(cols) : y.split;
  return y;
}

bool group_ok(int G) { return G == 1 || G == 2 || G == 4 || G == 8; }

// Columns of a workgroup, by the most tokens of a row as far as the host knows: 16 or 32 of the split kernel up to 64 columns a row, else
// 128 of the chunk kernel, with the split kernel's work in it for the batch's rows of few columns (us, 8 rows of 700 .. 8192, 8 kv heads,
// head_dim 128, bf16 / 8 bits: 20 columns 32.9 / 30.6 by two sets of 16, 42.4 / 33.1 by 16 a workgroup, 56.1 / 58.7 by the chunk kernel;
// 64 columns 48.1 / 41.6, 76.0 / 58.5, 57.1 / 61.0).
constexpr int kWideCols = 2 * kLongCols, kSplitCols = 64;
int few_tokens(int G) { return kLongCols / G; }
int columns_of(int G, int64_t max_tokens) {
  return max_tokens <= few_tokens(G) ? kLongCols : max_tokens <= kSplitCols / G ? kWideCols : kChunkCols;
}

}  // namespace

#define BZ_EXPORT __attribute__((visibility("default")))

extern "C" {

BZ_EXPORT int bz_paged_workspace_size(int32_t head_dim, int32_t group, int32_t max_tokens, size_t* bytes) {
  if (bytes == nullptr) return BZ_ERR_NULL;
  if (max_tokens < 0) return BZ_ERR_SHAPE;
  if ((head_dim != 64 && head_dim != 128) || !group_ok(group)) return BZ_ERR_UNSUPPORTED;
  int cus = 0;
  const int rc = bz::device_cu_count(&cus);
  if (rc != BZ_OK) return rc;
  *bytes = layout(cus, head_dim, max_tokens > 0 ? columns_of(group, max_tokens) : kChunkCols).total;
  return BZ_OK;
}

BZ_EXPORT int bz_gqa_paged(const bz_gqa_paged_args* a, hipStream_t stream) {
  if (a == nullptr || a->q == nullptr || a->out == nullptr) return BZ_ERR_NULL;
  const bz_paged_cache* c = &a->cache;
  int rc = bz::check_paged(c, true);
  if (rc != BZ_OK) return rc;
  const int NH = a->num_q_heads, NKV = c->num_kv_heads, D = c->head_dim;
  if (NH <= 0 || NH % NKV != 0 || a->max_tokens < 0 || a->max_seq_len < 0) return BZ_ERR_SHAPE;
  const int G = NH / NKV;
  if (!group_ok(G)) return BZ_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a->q) & 15) || ((a->q_stride_t | a->q_stride_h) & 7)) return BZ_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(a->out) & 1) return BZ_ERR_ALIGNMENT;
  int cus = 0;
  rc = bz::device_cu_count(&cus);
  if (rc != BZ_OK) return rc;

  const int64_t N = c->tokens, B = c->batch;
  // Columns of a workgroup by the most tokens of a row, as far as the host knows; where the caller says that none has many, the split
  // kernel takes whatever comes, several column tiles a row.
  int cols = columns_of(G, c->q_start == nullptr ? 1 : a->max_tokens > 0 ? std::min<int64_t>(a->max_tokens, N) : N);
  const int64_t cap = (int64_t)c->max_pages * c->page_size;
  const int64_t longest = a->max_seq_len > 0 && a->max_seq_len < cap ? a->max_seq_len : cap;
  const int64_t columns = N * NH, length = std::max<int64_t>(longest - std::min(longest, N / B) / 2, 1);  // of all heads; about a token's
  if (cols == kChunkCols) {
    // Short chunks of few heads: the split kernel for all rows. It reads K and V again for each 16 columns, but in one launch (us, split
    // kernel / chunk kernels, 100 tokens alone 6.1 / 8.6, behind 1000 10 .. 14 / 17; 4 kv heads of 2 q, head_dim 128: 300 behind 1000 18.0 /
    // 19.5, 100 behind 6000 22.8 / 26.0, 300 behind 6000 50.9 / 29.8; 2 of 2: 1000 alone 14.9 / 16.0; head_dim 64, 4 of 2: 100 behind 1000
    // 8.8 / 10.6, 300 12.0 / 11.8). Up to more columns where the batch may have rows of few tokens as well: a few column tiles leave CUs
    // idle, which its splits do not (head_dim 128, 300 behind 1000 and six rows of 600 .. 1300 18.5 / 23.4, 60 twice behind 2000, 8 bits,
    // and two of 1000 .. 2000 19.3 / 25.7; head_dim 64, 200 of 8 heads and four rows 6.2 / 6.9, 700 of 2 kv heads and four 11.1 / 8.9).
    const int64_t most = D == 128 ? 512 + (1 << 21) / length : 1280;
    if (columns <= (B > 1 ? most + (D == 128 ? 5 << 19 : 1 << 19) / length : most)) cols = kLongCols;
  } else if (cols == kWideCols && columns * length <= 5 << 19) {
    cols = kLongCols;  // (as few tiles: two sets of columns only make a workgroup slower, 2 rows of 20 tokens behind 500 9.0 / 12.0)
  }
  const bool chunks = cols == kChunkCols;
  const Layout ws = layout(cus, D, cols);
  if (a->workspace == nullptr || a->workspace_bytes < ws.total) return BZ_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(a->workspace) & 255) return BZ_ERR_ALIGNMENT;

  PagedParams p{};
  p.rows = bz::paged_rows(c);
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_st = a->q_stride_t, p.q_sh = a->q_stride_h;
  p.out = static_cast<uint16_t*>(a->out);
  p.o_st = a->out_stride_t, p.o_sh = a->out_stride_h;
  p.out_wide = !((reinterpret_cast<uintptr_t>(a->out) & 7) || ((p.o_st | p.o_sh) & 3));
  p.k = static_cast<const char*>(c->k), p.v = static_cast<const char*>(c->v);
  p.kv_sp = c->stride_page, p.kv_sh = c->stride_h, p.kv_ss = (int)c->stride_s;
  p.page_bytes = (int)(c->stride_s * (c->page_size - 1)) + (c->bits == 8 ? D : 2 * D);
  p.ks = static_cast<const uint8_t*>(c->k_scale), p.vs = static_cast<const uint8_t*>(c->v_scale);
  p.sc_sp = c->scale_stride_page, p.sc_sh = c->scale_stride_h;
  p.NKV = NKV, p.G = G, p.gshift = __builtin_ctz(G);
  p.scale_log2 = a->scale * kLog2e;
  p.part_slots = (int)(ws.slots / NKV);
  char* const base = static_cast<char*>(a->workspace);
  p.counters = reinterpret_cast<int*>(base);
  p.part_ml = reinterpret_cast<float2*>(base + ws.split.ml);
  p.part_acc = reinterpret_cast<float*>(base + ws.split.acc);
  // The chunk kernel's plan. Workgroups with g column groups (of all kv heads; without the tiles that rows' ends leave part empty), and
  // its column tiles at most.
  const bool f8 = c->bits == 8;
  auto tiles = [&](int g) { return (N * G + kPreWaveCols * g - 1) / (kPreWaveCols * g) * NKV; };
  auto units_of = [&](int g) { return N / (kPreWaveCols * g / G) + B; };
  int cg = 0;
  int few_tiles = 1;  // column tiles of 16 of the rows that count as few
  bool split = false, few_first = false;
  if (chunks) {
    const int64_t steps = longest / kChunkStep + 1;
    // Few column tiles of 128 over many positions are split over those as well (us, 8 kv heads of 2 q, head_dim 128, whole / split: 1024
    // tokens over 8192 105 / 82, 2048 over 16384 301 / 263, 256 over 8192 70 / 36); at head_dim 64, where one column group leaves
    // room for two workgroups a CU, only over very many unless even that leaves CUs idle.
    const bool idle = D == 128 || tiles(1) < cus;
    split = (tiles(4) <= cus && steps >= 32 * (2 * cus / tiles(4))) ||
            (tiles(2) < cus && std::min(cus / tiles(4), steps / (idle ? 14 : 64)) > 1);
    // Else four column groups, which read K and V least often, where about a workgroup of the longest row's average length is there for
    // every CU (us, 8 kv heads of 2 q, two groups / four, head_dim 128: 4096 tokens behind 4096 242 / 219, behind 16384 691 / 588, 6000
    // alone 181 / 160, but 2048 alone 38 / 46 and 4096 alone 91 / 95; head_dim 64: 4096 behind 4096 144 / 140, 2500 behind 5000 102 / 118),
    // from half of that on where rows of few tokens fill what is left and one of the two reads more alone (head_dim 128, 16 such rows of
    // 500 .. 3000 and 3000 tokens 83 / 75, 3 times 1024 47 / 42; head_dim 64, 2048 tokens 28.7 / 31.2). Else two where those give every
    // CU work, or one, which at head_dim 128 leaves no room for a second workgroup and so none for other rows' (1500 tokens of 4 kv
    // heads and four rows of 1000 .. 1500: one group 36.2, two 25.4; 1024 tokens alone: 18.7 by one, 26.6 by four, split).
    const int64_t most = std::min<int64_t>(a->max_tokens > 0 ? std::min<int64_t>(a->max_tokens, N) : N, longest);
    const double busy = (double)tiles(4) / cus * (1. - 0.5 * (double)most / (double)longest);
    const bool beside = B > 1 && D == 128;
    cg = split || busy >= (beside ? 0.5 : 1.05) ? 4 : tiles(2) >= cus || beside ? 2 : 1;
    // A row that the chunk kernel takes whole is one workgroup's long way through all its positions, mostly with columns of nobody where it
    // has few tokens. So up to 64 columns count as few, unless the rows are so many, for their lengths, that reading K and V again for
    // each 16 columns costs more (us, up to 16 columns / up to 64, head_dim 128, 8 kv heads of 8 q: 500 tokens and eight rows of five
    // behind 4000 .. 8000 155 / 94, behind 500 .. 1000 31 / 34; 8 bits, head_dim 64, 4 of 8: 700 and four of five behind 500 .. 1000 18 /
    // 13, behind 4500 47 / 17; 8 bits, 8 of 2: 16 rows of 20 behind 500 .. 1000 32 / 41, behind 3000 80 / 62; beside splits, 700 and
    // six of 30 behind 500 .. 3000 33 / 39).
    if (!split && longest >= 20 * B * NKV) few_tiles = kSplitCols / kLongCols;
    // Rows of few tokens come behind the chunks, whose longest have to begin at once, and ahead of them where they are most of the work:
    // an 8-bit batch's positions take about as long as 55 columns of chunks, bf16 ones as 110 (us, 8 kv heads of 2 q, head_dim 128, behind
    // / ahead: 1000 tokens and 32 rows of 500 .. 4000 72.5 / 67.9, two of 512 and 60 of 100 .. 3000, 8 bits, 61 / 53, but 2048 and 16 of
    // 500 .. 2000 50 / 60, and 500 and 16 of 900 .. 5000, which leave CUs without a row, 48.5 / 49.5). Splits are shorter than column
    // tiles, and beside fewer of them those rows go on at the same time (500 behind 4500, 450 behind 2500 and six of 900 .. 5000 68 / 60,
    // 1024 behind 1024 and 32 of 1000 .. 8000 144 / 126; head_dim 64, 4 kv heads of 4 q, 800 behind 4000 and six of 2000 .. 4800 44 / 48).
    const int64_t share = (f8 ? 55 : 110) * B;
    few_first = B > 1 && (split ? N * G <= 4 * share : N * G <= share && B * NKV >= cus);
  }
  // The split kernel's part, for rows of few tokens (all of them, if there are no others; else its work is in the chunk kernel's launch).
  // A batch of one row has that part too, as its tokens may be few and the others padding (us, 8 kv heads of 2 q, head_dim 128: one token
  // behind 4000 in a batch of 300 13.4, by the chunk kernel 21.0; its slots without work cost a chunk at most 0.5 in 277, and 0.1 in 35).
  // One token a row, and no dealing: two or three rows, taken to be alike, and batches of so many that rows may stay whole, whose
  // dealing takes each workgroup a look at all (us, 8 kv heads of 2 q, head_dim 128, dealt / whole: 256 rows of 50 .. 200 36.7 / 26.4, of
  // 500 .. 2000 209 / 207; 128 rows 18.8 / 16.2, 113 / 113). The longest row alone may take no longer than the batch does.
  const int row_bytes = f8 ? 2 * D + 2 : 4 * D;  // of a position
  const bool many = B * NKV >= 4 * cus && longest * row_bytes <= 4 * kOneSplitBytes * (B * NKV / (4 * cus));
  const bool alike = c->q_start == nullptr && (B <= 3 || many);
  int64_t split_slots = 0;
  const int P = f8 ? 32 : 16;
  const int64_t n = (longest + P - 1) / P;
  p.few = chunks ? few_tiles * few_tokens(G) : INT32_MAX;
  p.least = kFewThreads / kWave;
  p.one_split = kOneSplitBytes / row_bytes / P;
  const int64_t round = std::max<int64_t>(cus / NKV, 1);
  if (alike) {
    const int64_t most = (n + p.least - 1) / p.least;
    p.splits = many || n <= p.one_split ? 1 : (int)std::max<int64_t>(std::min({round / B, most, (int64_t)64}), 1);
    split_slots = B * p.splits;
  } else {
    // One round of workgroups, and two for a batch of many rows, whose splits are coarser (us, 8 kv heads of 2 q, head_dim 128, one round /
    // two: 32 rows of 512 .. 8192 of 8 bits 78 / 67, 64 of 128 .. 2048 56 / 52; 8 of 512 .. 8192 30.1 / 29.8; 4 of 1024 .. 16384 of 8 bits 18.7
    // / 21.0; three and four rounds take as long or longer).
    const int64_t units = chunks ? few_tiles * B : N / (cols / G) + B;  // column tiles at most
    const int64_t most = units * 2 > round ? 2 * round : few_first ? (round + 1) / 2 : round;  // (half beside a chunk's splits)
    p.splits = n <= p.one_split ? 0 : (int)std::min<int64_t>(most, p.part_slots / 2);
    p.lanes = units * 2 > round ? (int)round : 0;
    split_slots = units * 2 <= p.splits ? p.splits : p.splits + units;
  }
  auto launch = [&](auto fn, int64_t blocks, const auto&... params) {
    hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(kFewThreads), 0, stream, params...);
    return hipGetLastError() == hipSuccess ? BZ_OK : BZ_ERR_LAUNCH;
  };
  p.slots = (int)split_slots;
  using Fn = void (*)(const PagedParams);
  if (chunks) {
    // The chunk kernel's part: its parameters, grid and merge.
    PagedParams pc = p;
    pc.part_ml = reinterpret_cast<float2*>(base + ws.chunk.ml);
    pc.part_acc = reinterpret_cast<float*>(base + ws.chunk.acc);
    const int64_t all = kSlotsPerCu * cus / NKV;
    pc.splits = split ? (int)(few_first && split_slots < all / 2 ? all - split_slots : all) : 0;
    pc.least = kPreMinSteps, pc.one_split = kPreMinSteps;
    pc.lanes = 0;  // whether chunks are split was decided above, not by how many rows of few tokens stand beside them
    pc.merge_cols = units_of(4) * NKV * (kChunkCols / 16) <= 2 * cus ? 8 : 16;
    const int64_t chunk_slots = units_of(cg) * 2 <= pc.splits ? pc.splits : pc.splits + units_of(cg);
    const int64_t merge_grid = pc.splits > 0 ? units_of(4) * NKV * (kChunkCols / pc.merge_cols) : 0;
    const int64_t grid = (chunk_slots + split_slots) * NKV;
    if (std::max(grid, merge_grid) > kMaxGrid) return BZ_ERR_SHAPE;
    pc.slots = (int)chunk_slots;
    static_assert(kPreThreads == kFewThreads, "all by one launch()");
    using Both = void (*)(const PagedParams, const PagedParams, const int);
    const Both fns[2][2][3] = {{{paged_chunk_kernel<64, false, 1>, paged_chunk_kernel<64, false, 2>, paged_chunk_kernel<64, false, 4>},
                                {paged_chunk_kernel<64, true, 1>, paged_chunk_kernel<64, true, 2>, paged_chunk_kernel<64, true, 4>}},
                               {{paged_chunk_kernel<128, false, 1>, paged_chunk_kernel<128, false, 2>, paged_chunk_kernel<128, false, 4>},
                                {paged_chunk_kernel<128, true, 1>, paged_chunk_kernel<128, true, 2>, paged_chunk_kernel<128, true, 4>}}};
    rc = launch(fns[D == 128][f8][cg / 2], grid, pc, p, (int)few_first);
    if (rc != BZ_OK || merge_grid == 0) return rc;
    const Fn merges[2][2] = {{paged_merge_kernel<64, false>, paged_merge_kernel<64, true>},
                             {paged_merge_kernel<128, false>, paged_merge_kernel<128, true>}};
    return launch(merges[D == 128][f8], merge_grid, pc);
  }
  if (split_slots * NKV > kMaxGrid) return BZ_ERR_SHAPE;
  const Fn fns[2][2][3] = {
      {{paged_split_kernel<64, false, false, 1, kFewThreads>, paged_split_kernel<64, false, true, 1, kFewThreads>,
        paged_split_kernel<64, false, true, 2, kFewThreads>},
       {paged_split_kernel<64, true, false, 1, kFewThreads>, paged_split_kernel<64, true, true, 1, kFewThreads>,
        paged_split_kernel<64, true, true, 2, kFewThreads>}},
      {{paged_split_kernel<128, false, false, 1, kFewThreads>, paged_split_kernel<128, false, true, 1, kFewThreads>,
        paged_split_kernel<128, false, true, 2, kFewThreads>},
       {paged_split_kernel<128, true, false, 1, kFewThreads>, paged_split_kernel<128, true, true, 1, kFewThreads>,
        paged_split_kernel<128, true, true, 2, kFewThreads>}}};
  return launch(fns[D == 128][f8][alike ? 0 : cols == kWideCols ? 2 : 1], split_slots * NKV, p);
}

}  // extern "C"
