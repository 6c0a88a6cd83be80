// Device code of bz_gqa_paged (include/bz_paged_cache.h): how a batch's work is dealt to the workgroups, and the kernel for rows of
// few new tokens. The kernel for chunks is in paged_chunk.cuh.
//
// The (token, q head) pairs that share a kv head are the columns of one product, 16 a workgroup: 16 / G tokens of a row times the
// group's G heads. The row's positions are cut into wave tiles of 16 (bf16) or 32 (8-bit) of them, each in one page (or two, of 16),
// and the tiles dealt to the row's splits and their waves in turn. Masks, the softmax and the products within a wave are
// long_cache.cuh's.
//
// With running maximum m and sum l of a column (in units of log2: s = scale log2(e) q.k), a tile of scores s_p does
//   m' = max(m, max s_p), t_p = 2^(s_p - m'), l' = 2^(m - m') l + sum t_p, O' = 2^(m - m') O + sum t_p v_p
// and two parts of a row join the same way; out = O / l. Each t_p meets V as two bf16 terms, t = hi + lo, off by at most 2^-17 t.
//
// Reading K and V once bounds it (bf16, head_dim 128: 512 bytes a position and kv head for 512 G flops, 768 G as V meets two terms; a
// large product and a large copy meet at 244 flops a byte): 4 rows of up to 32768, 4 kv heads of 8 q, 229 MB in 39.5 us, 5.8 TB/s; 32
// rows of 300 .. 8192 of 8 bits, 8 kv heads of 2 q, 289 MB in 59 us, 4.9 TB/s; 8 rows of 700 .. 8192 with up to five tokens each,
// head_dim 64, 80 MB in 20.5. About 6 us of each are the launch, the lengths', table's and first tiles' round trips and the merge; two
// rows of 1024 take 5.6, as gqa_decode does.
#pragma once

#include "bz_paged_cache.h"
#include "long_cache.cuh"
#include "paged_common.cuh"

namespace bz {

// (Where the fields lie decides how many loads of arguments a kernel begins with: one more int in front of part_acc made every call of the
// split kernel 0.3 us slower.)
struct PagedParams {
  PagedRows rows;
  const uint16_t* q;
  int64_t q_st, q_sh;
  uint16_t* out;
  int64_t o_st, o_sh;
  int out_wide;                 // out and its strides are multiples of 8 bytes
  const char *k, *v;
  int64_t kv_sp, kv_sh;         // bytes
  int kv_ss, page_bytes;
  const uint8_t *ks, *vs;
  int64_t sc_sp, sc_sh;
  int NKV, G, gshift;
  float scale_log2;             // scale * log2(e)
  int few;                      // the split kernel takes the rows of at most `few` new tokens, the chunk kernel the others
  int splits;                   // not dealt: splits of a row; dealt: splits of all rows together (0: rows are not split)
  int lanes;                    // workgroups of a kv head that run at once, where rows may better stay whole (0: they may not)
  int least, one_split;         // tiles of a split at least; up to one_split a row is not split
  int merge_cols;               // columns of a workgroup of the merge kernel
  int part_slots;               // splits of a kv head that the workspace has room for
  int slots;                    // slots of the grid
  float* part_acc;              // [kv head, slot, column, D] unnormalised sums
  float2* part_ml;              // [kv head, slot, column] (max, sum)
  int* counters;                // [kv head, slot] x kCounterStride; the first slot of a column tile counts its splits
};

}  // namespace bz

namespace {

using bz::PagedParams;

// A row's new tokens (T of them from token q0 on) and length.
struct PagedRow {
  int q0, T, len;
};
__device__ __forceinline__ PagedRow paged_row(const bz::PagedRows& r, int b) {
  PagedRow x{b, 1, r.seq_lens[b]};
  if (r.q_start != nullptr) {
    const int q0 = r.q_start[b], q1 = r.q_start[b + 1];
    x.q0 = q0, x.T = q0 >= 0 && q1 > q0 && q1 <= r.tokens ? q1 - q0 : 0;
  }
  return x;
}
// Where a row's token t ends: it attends [0, that), clamped to the table.
__device__ __forceinline__ int paged_end(const bz::PagedRows& r, const PagedRow& x, int t) {
  const int64_t e = (int64_t)x.len - (x.T - 1 - t), cap = (int64_t)r.max_pages << r.pshift;
  return (int)(e < 0 ? 0 : e > cap ? cap : e);
}

// A workgroup's share: column tile `tile` of row b, split `split` of `k`; first: the tile's first slot in the workspace.
struct PagedShare {
  int b, tile, split, k, first;
  PagedRow row;
};

// Every wave works out the same: each row's tiles of columns and positions, how many splits it is cut into so that all are about
// as long and there are about p.splits of them, and which one `at` is (PER_TILE: which column tile). CHUNK: the rows of many tokens,
// else those of few. P positions a tile of positions, cols columns; splits are multiples of STEP tiles.
//
// n tiles in splits of `per`: with U column tiles in all, sum ceil(n / per) <= sum n / per + U. So per = total / splits gives at most
// splits + U (the grid, where U may be more than half of splits), and per = total / (splits - U) at most splits (the grid else).
// Splits of rows that are split (n > per, so ceil(n / per) < 2 n / per) number less than 2 splits: the workspace's slots.
template <bool CHUNK, bool PER_TILE, int P, int STEP>
__device__ __forceinline__ PagedShare deal_paged(const PagedParams& p, int cols, int at) {
  const int lane = threadIdx.x % kWave, B = p.rows.B, tshift = __builtin_ctz(cols) - p.gshift;
  struct Row {
    PagedRow r;
    int nt, n;  // its column tiles, and the position tiles of the longest
  };
  auto row_at = [&](int b) {  // (loads without a branch, so that those of several rows can be on their way)
    Row x{paged_row(p.rows, min(b, B - 1)), 0, 0};
    if (b < B && x.r.T > 0 && (x.r.T > p.few) == CHUNK) {
      x.nt = (x.r.T + (1 << tshift) - 1) >> tshift;
      x.n = (paged_end(p.rows, x.r, x.r.T - 1) + P - 1) / P;
    }
    return x;
  };
  const Row first = row_at(lane);
  float per, inv = 0.f;
  auto splits_of = [&](const Row& x) {
    return inv == 0.f || x.n <= p.one_split ? 1 : max(1, (int)__builtin_ceilf((float)x.n * inv));
  };
  if (p.splits > 0) {
    float total = (float)first.nt * (float)first.n, units = (float)first.nt, most = (float)first.n;
#pragma unroll 4
    for (int b0 = kWave; b0 < B; b0 += kWave) {
      const Row x = row_at(b0 + lane);
      total += (float)x.nt * (float)x.n;
      units += (float)x.nt;
      most = fmaxf(most, (float)x.n);
    }
    total = wave_sum(total), units = wave_sum(units), most = wave_max(most);
    // (a chunk's splits: two rounds of workgroups where each still has 12 steps, else one: their sums' way through memory costs more)
    const float want = CHUNK && total < 12.f * (float)p.splits ? fmaxf(0.5f * (float)p.splits, 1.f) : (float)p.splits, even = 1.00001f * total;
    // Whole column tiles where those keep the device as busy: `lanes` workgroups of a head at a time, each the longest's time.
    const bool whole = p.lanes > 0 && most * (float)p.lanes * __builtin_ceilf(units / (float)p.lanes) <= 1.35f * total;
    // else the shortest of a few `per` that keeps within p.splits, by how many of them are set aside for rounding up: none to U (all
    // tried at once: a turn for each cost 0.2 us)
    constexpr int TRIES = 9;
    constexpr float kAside[TRIES] = {0.f, 0.25f, 0.375f, 0.4375f, 0.5f, 0.5625f, 0.625f, 0.75f, 1.f};
    float pers[TRIES], need[TRIES];
    const float aside = units < want ? units : 0.f;
#pragma unroll
    for (int i = 0; i < TRIES; ++i) {
      pers[i] = fmaxf((float)p.least, even * __builtin_amdgcn_rcpf(want - kAside[i] * aside));
      pers[i] = (float)STEP * __builtin_ceilf(pers[i] * (1.f / STEP));
      need[i] = 0.f;
    }
    for (int b0 = 0; b0 < B && aside > 0.f; b0 += kWave) {
      const Row x = b0 == 0 ? first : row_at(b0 + lane);
#pragma unroll
      for (int i = 0; i < TRIES; ++i) {
        inv = 0.99999f * __builtin_amdgcn_rcpf(pers[i]);  // (never more splits than the exact quotient has)
        need[i] += wave_sum((float)x.nt * (float)splits_of(x));
      }
    }
    per = pers[TRIES - 1];
#pragma unroll
    for (int i = TRIES - 2; i >= 0; --i) per = need[i] <= want ? pers[i] : per;
    inv = whole ? 0.f : 0.99999f * __builtin_amdgcn_rcpf(per);
  }
  int seen = 0, parts = 0;
  Row x = first;
  for (int b0 = 0; b0 < B; b0 += kWave) {
    const Row next = b0 + kWave < B ? row_at(b0 + kWave + lane) : first;
    const int k = splits_of(x), mine = PER_TILE ? x.nt : x.nt * k, part = k > 1 ? x.nt * k : 0;
    const int last = seen + (int)wave_scan((uint32_t)mine), pl = parts + (int)wave_scan((uint32_t)part);
    const uint64_t hit = __ballot(at < last && at >= last - mine);
    if (hit != 0) {
      const int l = __builtin_ctzll(hit);
      const int kk = __builtin_amdgcn_readlane(k, l), u = at - __builtin_amdgcn_readlane(last - mine, l);
      const int tile = PER_TILE ? u : u / kk;
      const PagedRow r{__builtin_amdgcn_readlane(x.r.q0, l), __builtin_amdgcn_readlane(x.r.T, l), __builtin_amdgcn_readlane(x.r.len, l)};
      return {b0 + l, tile, PER_TILE ? 0 : u - tile * kk, kk, __builtin_amdgcn_readlane(pl - part, l) + tile * kk, r};
    }
    seen = __builtin_amdgcn_readlane(last, kWave - 1);
    parts = __builtin_amdgcn_readlane(pl, kWave - 1);
    x = next;
  }
  return {-1, 0, 0, 1, 0, {0, 0, 0}};
}

// The pages of a wave's tiles: lane i holds that of its i-th tile (of the 64 at hand), -1 past the table.
__device__ __forceinline__ int page_ids(const Rsrc& table, int max_pages, int64_t index) {
  const int i = index < max_pages ? (int)index : max_pages;
  const int id = __builtin_amdgcn_raw_buffer_load_b32(table, 4 * i, 0, 0);
  return i < max_pages ? id : -1;
}

// 32 positions of 8-bit codes. K: lane (r, g) holds the D / 4 dims from (D / 4) g on of rows r and 16 + r (the products take dims in
// any order as long as q's operand has the same), V the dims (D / 16) r .. of positions 4 g + i and 16 + 4 g + i, whose scales are
// the bytes of vs.
template <int D>
struct F8Tile {
  uint32_t k[2][D / 16], ks[2], v[8][D / 64], vs[2];
};

template <int D>
__device__ __forceinline__ void load_f8_half(F8Tile<D>& t, int s, const Rsrc& k, const Rsrc& v, const Rsrc& ks, const Rsrc& vs,
                                             uint32_t at, uint32_t row_bytes, int r, int g) {
  const uint32_t ko = (at + r) * row_bytes + (D / 4) * g;
#pragma unroll
  for (int j = 0; j < D / 64; ++j) {
    const uint4 w = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(k, ko + 16 * j, 0, kStream));
    t.k[s][4 * j] = w.x, t.k[s][4 * j + 1] = w.y, t.k[s][4 * j + 2] = w.z, t.k[s][4 * j + 3] = w.w;
  }
  t.ks[s] = __builtin_amdgcn_raw_buffer_load_b8(ks, at + r, 0, 0);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t vo = (at + 4 * g + i) * row_bytes + (D / 16) * r;
    if constexpr (D == 128) {
      const uint2 w = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(v, vo, 0, kStream));
      t.v[4 * s + i][0] = w.x, t.v[4 * s + i][1] = w.y;
    } else {
      t.v[4 * s + i][0] = __builtin_amdgcn_raw_buffer_load_b32(v, vo, 0, kStream);
    }
  }
  t.vs[s] = __builtin_amdgcn_raw_buffer_load_b32(vs, at + 4 * g, 0, 0);
}

// st.acc += what the non-finite values of V add to the columns that attend their positions (accumulate's product of its own for each
// column; ncol columns, one a lane r).
template <int D, int N, class Pos>
__device__ __forceinline__ void odd_columns(LongState<D>& st, const uint32_t (&v)[N][D / 32], const uint32_t (&hi)[N / 2], int r, int ncol,
                                            const Reach& mine, Pos pos) {
  for (int c = 0; c < ncol; ++c) {
    const Reach rc{0, __builtin_amdgcn_readlane(mine.len, c), 0};
    uint32_t keep[N / 2];  // the halves of each operand word whose positions the column attends
#pragma unroll
    for (int a = 0; a < N / 2; ++a)
      keep[a] = (attends(rc, 0, pos(2 * a)) ? 0xffffu : 0u) | (attends(rc, 0, pos(2 * a + 1)) ? 0xffff0000u : 0u);
#pragma unroll
    for (int n = 0; n < D / 16; ++n) {
      uint32_t vt[N / 2];
#pragma unroll
      for (int a = 0; a < N / 2; ++a) {
        vt[a] = n % 2 ? pair_hi(v[2 * a][n / 2], v[2 * a + 1][n / 2]) : pair_lo(v[2 * a][n / 2], v[2 * a + 1][n / 2]);
        vt[a] = odd_pair(vt[a]) & keep[a];
        asm volatile("" : "+v"(vt[a]));  // worked out here, not for all columns before the loop (registers)
      }
      const f32x4_t t = mfma_pv<N>(vt, hi, f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int i = 0; i < 4; ++i) st.acc[n][i] += r == c ? t[i] : 0.f;
    }
  }
}

// The splits of rows of few tokens: slot `at` of kv head h; not dealt (DEAL false, rows taken to be alike): slot = row * splits + split,
// one token a row. C sets of 16 columns a workgroup: two where rows have more than 16, so that K and V are read and converted once for
// both. acc_of(u): LDS of split_floats<D, C>() floats for wave u's sums.
template <int D, int C>
constexpr int split_floats() { return C * kLongCols * (D + 4); }  // (rows of D + 4: 16-byte stores without bank conflicts)

template <int D, bool F8, bool DEAL, int C, int NT, class Acc>
__device__ __forceinline__ void paged_split(const PagedParams& p, int at, int h, Acc acc_of) {
  constexpr int NW = NT / kWave, P = F8 ? 32 : 16, NS = P / 16, N = 4 * NS, NJ = D / 32, COLS = C * kLongCols;
  const int tid = threadIdx.x, lane = tid % kWave, w = wave_uniform(tid / kWave), r = lane % 16, g = lane / 16;
  PagedShare share;
  if constexpr (DEAL) {
    share = deal_paged<false, false, P, NW>(p, COLS, at);
    if (share.b < 0) return;
  } else {
    const int b = at / p.splits;
    share = {b, 0, at - b * p.splits, p.splits, b * p.splits, paged_row(p.rows, b)};
  }
  const PagedRow& row = share.row;
  const int tpt = COLS >> p.gshift, t0 = share.tile * tpt, ntok = min(tpt, row.T - t0), ncol = ntok << p.gshift;
  auto token_end = [&](int t) { return paged_end(p.rows, row, t); };
  const int e1 = wave_uniform(token_end(t0 + ntok - 1)), whole_end = wave_uniform(token_end(t0));  // every column attends [0, whole_end)

  // the B operands of K . q^T: this lane's columns, dims as the tile's K has them
  int col[C];
  Reach mine[C];
  uint4 qr[C][NJ];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    col[c] = (kLongCols * c + r) % ncol;  // columns past the last repeat earlier ones
    const int tok = t0 + (col[c] >> p.gshift), hq = (h << p.gshift) + (col[c] & (p.G - 1));
    const uint16_t* qsrc = p.q + (int64_t)(row.q0 + tok) * p.q_st + (int64_t)hq * p.q_sh;
#pragma unroll
    for (int j = 0; j < NJ; ++j) qr[c][j] = *reinterpret_cast<const uint4*>(qsrc + (F8 ? (D / 4) * g + 8 * j : 32 * j + 8 * g));
    mine[c] = {0, token_end(tok), 0};
  }
  const int n = (e1 + P - 1) / P;
  int k = share.k;
  if constexpr (!DEAL) k = n <= p.one_split ? 1 : min(k, max(1, (n + p.least - 1) / p.least));
  const int nact = max(1, min(k, (n + NW - 1) / NW));  // splits with tiles
  if (share.split >= nact) return;
  const int j0 = share.split * NW + w, stride = nact * NW, count = j0 < n ? (n - j0 + stride - 1) / stride : 0;

  const Rsrc table = span_rsrc(p.rows.table + share.b * p.rows.table_st, p.rows.max_pages * 4);
  int ids[NS];
  auto fetch = [&](int i0) {
    const int64_t pos = (int64_t)P * (j0 + (int64_t)(i0 + lane) * stride);
#pragma unroll
    for (int s = 0; s < NS; ++s) ids[s] = page_ids(table, p.rows.max_pages, (pos + 16 * s) >> p.rows.pshift);
  };
  struct Tile {
    std::conditional_t<F8, F8Tile<D>, WaveTile<D>> t;
    int page[NS];  // -1: none, nothing of it is read
  };
  constexpr bool ONE = F8 && D == 128 && C == 2;  // one tile at a time: two would not fit the registers
  Tile ta, tb;
  const int64_t khead = (int64_t)h * p.kv_sh, shead = (int64_t)h * p.sc_sh;
  const int pmask = (1 << p.rows.pshift) - 1;
  auto load = [&](Tile& x, int i) {
    if ((i & (kWave - 1)) == 0 && i > 0 && i < count) fetch(i);
    const int pos0 = P * (j0 + i * stride);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int id = __builtin_amdgcn_readlane(ids[s], i & (kWave - 1));
      const bool there = i < count && (uint32_t)id < (uint32_t)p.rows.pages;
      x.page[s] = there ? id : -1;
      const int64_t page = there ? id : 0;
      const int bytes = there ? p.page_bytes : 0;
      const int at = (pos0 + 16 * s) & pmask;
      const Rsrc rk = span_rsrc(p.k + page * p.kv_sp + khead, bytes), rv = span_rsrc(p.v + page * p.kv_sp + khead, bytes);
      if constexpr (F8) {
        const int sb = there ? pmask + 1 : 0;
        const Rsrc rks = span_rsrc(p.ks + page * p.sc_sp + shead, sb), rvs = span_rsrc(p.vs + page * p.sc_sp + shead, sb);
        load_f8_half<D>(x.t, s, rk, rv, rks, rvs, at, (uint32_t)p.kv_ss, r, g);
      } else {
        const Spans sp{rk, rv, rk, (uint32_t)p.kv_ss, 0};
        load_wave_tile<D, BZ_MASK_NONE>(x.t, sp, at, r, g);
      }
    }
  };

  LongState<D> st[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    st[c].m = -INFINITY;
    st[c].l = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st[c].acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  fetch(0);
  load(ta, 0);
  if constexpr (!ONE) load(tb, 1);
  __builtin_amdgcn_sched_barrier(0);  // q's conversion waits for q: not before the tiles' loads
  const float scale = positive_scale(p.scale_log2);
  bf16x8_t qf[C][NJ];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < NJ; ++i) qf[c][i] = signed_q(qr[c][i], p.scale_log2);

  auto consume = [&](Tile& y, int i) {
    auto& t = y.t;
    const int pos0 = P * (j0 + i * stride);
    auto pos = [&](int u) { return pos0 + 16 * (u / 4) + 4 * g + u % 4; };
    float x[C][N];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      f32x4_t d[C];
#pragma unroll
      for (int c = 0; c < C; ++c) d[c] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        bf16x8_t kf;
        if constexpr (F8) kf = __builtin_bit_cast(bf16x8_t, bz::f8_values(make_uint2(t.k[u][2 * j], t.k[u][2 * j + 1]), t.ks[u]));
        else kf = k_operand<D>(t, j);
#pragma unroll
        for (int c = 0; c < C; ++c) d[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[c][j], d[c], 0, 0, 0);
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[c][4 * u + i] = d[c][i];
    }
    auto value = [&](int i, int m) __attribute__((always_inline)) {  // dims 2 m and 2 m + 1 of this lane's at its i-th position
      if constexpr (F8) {
        const uint32_t e = (t.vs[i / 4] >> (8 * (i % 4))) & 255u;
        return m % 2 ? bz::f8_pair<true>(t.v[i][m / 2], e) : bz::f8_pair<false>(t.v[i][m / 2], e);
      } else {
        return t.v[i][m];
      }
    };
    // An infinity takes one product alone (odd_columns). Of 8 bits it can only be under the largest scale, and a NaN matters only where
    // not every column attends it.
    bool bad = false;
    if constexpr (F8) {
#pragma unroll
      for (int u = 0; u < NS; ++u)  // a byte of 247 or more
        bad |= (((t.vs[u] & 0x7f7f7f7fu) + 0x09090909u) & t.vs[u] & 0x80808080u) != 0;
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int m = 0; m < NJ; ++m) top = max_u16x2(top, t.v[i][m] & 0x7fff7fffu);
      bad = pair_not_finite(top);
    }
    const bool part = pos0 + P > whole_end || (y.page[0] | y.page[NS - 1]) < 0;  // not every column attends the whole tile
    uint32_t hi[C][N / 2], lo[C][N / 2];
    // st.acc += V^T P, v(m, x): dims 2 m and 2 m + 1 of the lane's positions
    auto products = [&](auto v) __attribute__((always_inline)) {
#pragma unroll
      for (int m = 0; m < NJ; ++m) {
        uint32_t vm[N];
        v(m, vm);
#pragma unroll
        for (int n = 2 * m; n < 2 * m + 2; ++n) {
          uint32_t vt[N / 2];
#pragma unroll
          for (int a = 0; a < N / 2; ++a) vt[a] = n % 2 ? pair_hi(vm[2 * a], vm[2 * a + 1]) : pair_lo(vm[2 * a], vm[2 * a + 1]);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            st[c].acc[n] = mfma_pv<N>(vt, hi[c], st[c].acc[n]);
            st[c].acc[n] = mfma_pv<N>(vt, lo[c], st[c].acc[n]);
          }
        }
      }
    };
    if constexpr (C == 1 && !F8) {  // (one path: with two, 206 registers in place of 151, and 64 rows of 128 .. 2048 take 56.7 us, not 52.3)
      uint32_t v[N][NJ];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int m = 0; m < NJ; ++m) v[i][m] = t.v[i][m];
      if (part) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const bool some = pos(i) < e1 && y.page[i / 4] >= 0;
          x[0][i] = some && pos(i) < mine[0].len ? x[0][i] : -INFINITY;
#pragma unroll
          for (int m = 0; m < NJ; ++m) {
            v[i][m] = some ? v[i][m] : 0u;
            top = max_u16x2(top, v[i][m] & 0x7fff7fffu);
          }
        }
        bad = pair_not_finite(top);
      }
      fold_scores<D, N>(st[0], x[0], scale);
      accumulate<D, N>(st[0], v, x[0], bad, col[0], ncol, mine[0], 0, pos);
      return;
    }
    if (part || __ballot(bad) != 0) {
      // V of positions that none attends (behind the row's end, where a page may hold anything) becomes 0
      uint32_t v[N][NJ], top = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool some = pos(i) < e1 && y.page[i / 4] >= 0;
#pragma unroll
        for (int c = 0; c < C; ++c) x[c][i] = some && pos(i) < mine[c].len ? x[c][i] : -INFINITY;
#pragma unroll
        for (int m = 0; m < NJ; ++m) {
          v[i][m] = some ? value(i, m) : 0u;
          top = max_u16x2(top, v[i][m] & 0x7fff7fffu);
        }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
        fold_scores<D, N>(st[c], x[c], scale);
        split_terms(x[c], hi[c], lo[c]);
      }
      if (__builtin_expect(__ballot(pair_not_finite(top)) != 0, 0)) {
#pragma unroll
        for (int c = 0; c < C; ++c)  // (a set's columns are its lanes r up to their number)
          odd_columns<D, N>(st[c], v, hi[c], r, min(kLongCols, ncol - kLongCols * c), mine[c], pos);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int m = 0; m < NJ; ++m) v[i][m] = finite_pair(v[i][m]);
      }
      products([&](int m, uint32_t (&vm)[N]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; ++i) vm[i] = v[i][m];
      });
      return;
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      fold_scores<D, N>(st[c], x[c], scale);
      split_terms(x[c], hi[c], lo[c]);
    }
    products([&](int m, uint32_t (&vm)[N]) __attribute__((always_inline)) {  // (a few values of 8 bits as bf16 at a time: registers)
#pragma unroll
      for (int i = 0; i < N; ++i) vm[i] = value(i, m);
    });
  };

  if constexpr (ONE) {
    for (int i = 0; i < count; ++i) {
      consume(ta, i);
      load(ta, i + 1);
    }
  } else {
    for (int i = 0; i < count; i += 2) {
      consume(ta, i);
      if (i + 1 >= count) break;
      load(ta, i + 2);
      consume(tb, i + 1);
      load(tb, i + 3);
    }
  }

  constexpr int PD = D + 4;
  float* const my_acc = acc_of(w);
  __shared__ float s_m[NW][COLS], s_l[NW][COLS];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    // the columns are complete over the wave's positions; only the sums are still one per lane group
    float z = st[c].l;
    swap16(st[c].l, z);
    st[c].l += z;
    z = st[c].l;
    swap32(st[c].l, z);
    st[c].l += z;
    const int to = kLongCols * c + r;
    if (to < ncol) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int q = 0; q < D / 16; q += 4)
          *reinterpret_cast<f32x4_t*>(my_acc + to * PD + D / 16 * (4 * g + i) + q) =
              f32x4_t{st[c].acc[q][i], st[c].acc[q + 1][i], st[c].acc[q + 2][i], st[c].acc[q + 3][i]};
      if (g == 0) {
        s_m[w][to] = st[c].m;
        s_l[w][to] = st[c].l;
      }
    }
  }
  __syncthreads();

  auto write = [&](int c, int d, const f32x4_t& a, float, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN sum stays one
    uint16_t* const o = p.out + (int64_t)(row.q0 + t0 + (c >> p.gshift)) * p.o_st +
                        (int64_t)((h << p.gshift) + (c & (p.G - 1))) * p.o_sh + d;
    const uint2 z = make_uint2(pack_bf16x2(a[0] * inv, a[1] * inv), pack_bf16x2(a[2] * inv, a[3] * inv));  // l == 0: a is 0
    if (p.out_wide) {
      *reinterpret_cast<uint2*>(o) = z;
    } else {
      o[0] = (uint16_t)z.x, o[1] = (uint16_t)(z.x >> 16), o[2] = (uint16_t)z.y, o[3] = (uint16_t)(z.y >> 16);
    }
  };
  const int64_t slot = (int64_t)h * p.part_slots + share.first;  // the column tile's first
  for (int o = tid; o < ncol * D / 4; o += NT) {
    const int c = o / (D / 4), d = 4 * (o % (D / 4));
    float M = s_m[0][c];
#pragma unroll
    for (int u = 1; u < NW; ++u) M = fmaxf(M, s_m[u][c]);
    const float mu = (M == -INFINITY) ? 0.f : M;
    float L = 0.f;
    f32x4_t A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NW; ++u) {
      const float f = fast_exp2(s_m[u][c] - mu);
      L = fmaf(f, s_l[u][c], L);
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(acc_of(u) + c * PD + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) A[i] = fmaf(f, a[i], A[i]);
    }
    if (nact == 1) {
      write(c, d, A, M, L);
    } else {
      const int64_t ps = (slot + share.split) * COLS;
      const Rsrc rp = span_rsrc(p.part_acc + ps * D, COLS * D * 4);
      using U4 = decltype(__builtin_amdgcn_raw_buffer_load_b128(rp, 0, 0, 0));
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(U4, A), rp, 16 * o, 0, kSc1);
      if (d == 0) {
        st_agent(reinterpret_cast<float*>(p.part_ml + ps + c), M);
        st_agent(reinterpret_cast<float*>(p.part_ml + ps + c) + 1, L);
      }
    }
  }
  if (nact == 1) return;

  // the last workgroup of this (column tile, kv head) to count in merges, as in gqa_split_kernel
  __shared__ int s_last;
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
  if (tid == 0) {
    int* cnt = p.counters + slot * kCounterStride;
    const int prev = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = (prev == nact - 1);
    if (s_last) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s_last) return;
  merge_columns<D, NT>(p.part_acc + slot * COLS * D, p.part_ml + slot * COLS, COLS, ncol, nact, write);
}

// Grid slots * kv heads, a slot's heads side by side.
template <int D, bool F8, bool DEAL, int C, int NT>
__global__ void __launch_bounds__(NT, 2) paged_split_kernel(const PagedParams p) {
  __shared__ __align__(16) float s_acc[NT / kWave][split_floats<D, C>()];
  const int at = (int)(blockIdx.x / (uint32_t)p.NKV), h = (int)blockIdx.x - at * p.NKV;
  paged_split<D, F8, DEAL, C, NT>(p, at, h, [&](int u) { return &s_acc[u][0]; });
}

}  // namespace
