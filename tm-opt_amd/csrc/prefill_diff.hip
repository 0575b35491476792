// Varlen causal (optionally windowed) differential attention on bf16 MFMA,
// gfx950 (see diff.h for the formula).
//
// Matrix bound: per visible (query, key) pair and map 128 products for the
// score and 256 for the values.
//
//  * A work-group of eight waves owns (run, pair of stored heads, block of 128
//    / REP queries) for REP head pairs: 128 rows of each map, over the same
//    tiles of 32 keys (K, K' and the 256-wide V: 32 KB) in LDS. Wave w has map
//    w >> 2 of row block w & 3 (32 rows), so waves w and w + 4, which share a
//    SIMD, are the two maps of the same rows. O^T of 32 rows x 256 dims takes
//    128 registers, which leaves two waves per SIMD room for 32-key tiles, not
//    for 64-key ones.
//  * S^T = K.Q^T (v_mfma_f32_32x32x16_bf16, keys on M, queries on N) leaves one
//    query per lane; P^T is then the B operand of O^T = V^T.P^T as it is.
//  * Tiles go from global memory straight into LDS (buffer_load ... lds), rows
//    of 256 B, K chunks of 16 B swizzled by row & 15, V blocks of 64 B by row &
//    3: neither the K fragments (16-byte reads) nor the V^T fragments (two
//    transposed reads) conflict. Four stages, tiles issued three ahead.
//  * Ping-pong: the two waves of a SIMD alternate, half a tile apart, between
//    an MFMA phase (P.V of tile t and the scores of tile t + 1: 24 MFMAs) and
//    the softmax of a tile.
//  * The maps meet in LDS at the end: each wave gives its partner half of its
//    normalised O and takes the difference and the norm of the other half.
//  * A launch whose items fit the chip at once, or see few keys each
//    (layout_of), takes work-groups of four waves with 64 rows of each map, two
//    per compute unit: each has two stages, K a tile ahead of V, and no phases
//    to keep; one's start and end run beside the other's products. Graph
//    replays, us, eight / four waves: 30 tokens 64Q/8KV 9.4 / 7.9, 600 32Q/4KV
//    26.6 / 23.7, 777 33.0 / 29.0, 1,200 under a window of 512 32Q/8KV 31.4 /
//    26.4. Full chips are quicker with eight, whose loads reach three tiles
//    ahead and serve twice the rows: 64 x 512 358 / 413, 4 x 8,192 2,750 /
//    2,950. (Four waves with four stages, one work-group per unit, were slower
//    on both.)
//  * Work items are dealt to the XCDs heaviest first (prefill_sched.h).
//
// 4 prompts of 8,192 tokens run at 1,134-1,197 TFLOP/s, 4 of 2K-8K at
// 1,092-1,158 (32Q/4KV, by the session): matrix cycles are 0.67 of all, at the 1.6
// GHz that the power limit leaves a full chip (a plain 8192^3 product 1,263
// TFLOP/s at 1.75 GHz). There
// a tile is 0.97 us of the matrix pipes and takes 1.4; an item's start and end
// cost some 9 us, which no other work-group hides (one per CU by its LDS and
// registers).
#include <algorithm>
#include <type_traits>

#include "diff.h"
#include "prefill_sched.h"

namespace tmopt {
namespace {

constexpr int kBN = 32;                   // keys per tile
constexpr int kRowB = 256;                // one key's slice of a stored head
constexpr int kSliceB = kBN * kRowB;      // 8 KB
constexpr int kStage = 4 * kSliceB;       // K, K', V, V'
// Tiles in LDS of a work-group of W waves, and its bytes with the norm's sums
// and weights.
constexpr int stages_of(int W) { return W == 8 ? 4 : 2; }
constexpr int lds_of(int W) {
  return stages_of(W) * kStage + W * 128 + kDV * 4;
}
constexpr float kLazy = 8.0f;             // lazy-rescale threshold (log2)
constexpr int kRing = 4;                  // fragments read kRing - 1 ahead
// a buffer offset past every resource this kernel builds (their ranges are
// checked below 2^31 - 16 on the host): the load returns zeros
constexpr int kOob = 0x7ffffff0;

struct PrefillDiffArgs {
  const __bf16* q;
  int64_t q_st, q_sh;
  const __bf16* k;         // packed rows, or the pool
  int64_t k_st, k_sh;
  const __bf16* v;
  int64_t v_st, v_sh;
  const int32_t* cu;
  const int32_t* prior;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_width;      // entries a row may be read at: min(bt_stride, 2^31-1)
  int num_pages;
  int HQ;
  int HKV;           // pairs of stored heads as scheduled
  int kv_div;        // scheduled pairs per stored one
  int S;
  int nqb_max;       // query blocks of the longest run
  int window;
  float scale_log2;
  DiffWeights w;
  __bf16* out;
  int64_t o_st, o_sh;
  float* lse;
  int64_t lse_sh;
  const int32_t* reject;
  // split keys (see pieces_of): nsplit > 1 levels of n_base work-groups
  int nsplit, n_base;
  int cus;
  float* part_o;     // [nsplit * n_base][8 waves][32][64 lanes][4] fp32
  float* part_lse;   // [nsplit * n_base][8 waves][32 rows]
  int* part_n;       // [n_base] pieces of each item (0: no such item)
};

// First key a work item reads (a multiple of the tile width at or below the
// first key a query of the block may see) and its tiles from there.
struct Tiles {
  int k_lo, n;
};
__device__ __forceinline__ Tiles item_tiles(const PrefillDiffArgs& a, int BQ,
                                            int prior, int len, int qb) {
  const int q0 = qb * BQ;
  const int lo = a.window > 0 ? max(0, prior + q0 - a.window + 1) : 0;
  const int k_lo = (lo / kBN) * kBN;
  return Tiles{k_lo, (prior + min(len, q0 + BQ) - k_lo + kBN - 1) / kBN};
}

// Work item x of a launch that splits its keys, in the order that schedule()
// takes: its items are numbered without gaps, head pairs first, so that the
// pieces of few items spread over all XCDs (item, then level, is dealt to them
// in turn). Without splits each pair of stored heads keeps to XCDs of its own.
__device__ __forceinline__ int split_item(int pairs, int x) {
  const int kvh = x % pairs, i = x / pairs;
  if (pairs <= 8 && 8 % pairs == 0) {
    const int r = 8 / pairs;
    return 8 * (i / r) + kvh * r + i % r;
  }
  if (pairs % 8 == 0) return 8 * (i * (pairs / 8) + kvh / 8) + kvh % 8;
  return x;
}

// Split keys: a launch of few items, or of few more than there are compute
// units, leaves units idle while its longest items run. It cuts each item's
// tiles into pieces, one work-group each (level s of the grid holds piece s of
// every item); a piece leaves its normalised fp32 results with their LSE (up to
// 257 KB), and prefill_diff_merge joins them in order and takes the difference
// and the norm. The longest item gets the n pieces that the estimate below says
// are quickest, others their share. The estimate, in us: items are taken as
// evenly spread between `low` and `most` tiles, heaviest first, one work-group
// per compute unit; a tile takes 1.05 on up to half the units and 1.4 on all
// (power: 2.1 against 1.6 GHz); pieces cost 5 for their start and the merge,
// 0.1 for each of an item's that it joins, and 0.115 for each of the launch's
// that is written and read, if all its rows are queries. Of four waves, two per
// unit: a tile takes 1.0 alone and 1.5 beside another, a piece is half the
// size.
constexpr int kMinPiece = 4;   // tiles
template <int W>
__device__ __forceinline__ int pieces_of(const PrefillDiffArgs& a, int BQ,
                                         int lane, int tiles) {
  int sum = 0, most = 0, items = 0, rows = 0;
  for (int s = lane; s < a.S; s += 64) {
    const int len = a.cu[s + 1] - a.cu[s];
    const int nb = (len + BQ - 1) / BQ;
    const int prior = a.prior != nullptr ? max(a.prior[s], 0) : 0;
    if (nb > 0) {
      const int t0 = item_tiles(a, BQ, prior, len, 0).n;
      const int t1 = item_tiles(a, BQ, prior, len, nb - 1).n;
      sum += nb * (t0 + t1) / 2;
      most = max(most, max(t0, t1));
      items += nb;
      rows += len;
    }
  }
  for (int x = 1; x < 64; x <<= 1) most = max(most, __shfl_xor(most, x));
  most = __builtin_amdgcn_readfirstlane(most);
  const int count = __builtin_amdgcn_readfirstlane(wave_sum(items));
  if (most <= 0 || count <= 0) return 1;
  const float mean =
      (float)__builtin_amdgcn_readfirstlane(wave_sum(sum)) / count;
  const float low = fmaxf(0.0f, 2.0f * mean - most);
  const float all = (float)count * a.HKV;
  const float full =
      (float)__builtin_amdgcn_readfirstlane(wave_sum(rows)) / (count * BQ);
  float best = 0.0f;
  int n = 1;
  for (int x = 1; x <= a.nsplit; ++x) {
    const float load = all * x / (W == 8 ? a.cus : 2 * a.cus);
    const float len = (low * fmaxf(1.0f, ceilf(load - 0.02f)) +
                       (most - low) * fmaxf(1.0f, 0.5f * load)) / x;
    const float part = fminf(fmaxf(load, 0.5f), 1.0f);
    const float us =
        len * (W == 8 ? 0.7f + 0.7f * part : 0.5f + part) +
        (x > 1 ? 5.0f + 0.1f * x + (0.115f / 8 * W) * full * x * all : 0.0f);
    if (x == 1 || us < best) {
      best = us;
      n = x;
    }
  }
  n = min(min(n, tiles / kMinPiece), (int)((float)n * tiles / most + 0.5f));
  return __builtin_amdgcn_readfirstlane(max(1, n));
}

template <int W, int REP, bool PAGED, bool SPLIT>
__global__ __launch_bounds__(64 * W, 2) void prefill_diff_kernel(
    PrefillDiffArgs a) {
  constexpr int RB = W / 2;            // 32-row blocks of a map
  constexpr int BQ = 32 * RB / REP;    // queries per work-group
  constexpr int QSUB = BQ / 32;        // 32-query sub-blocks per head pair
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int h2 = lane >> 5;       // lane half
  const int level = SPLIT ? (int)blockIdx.x / a.n_base : 0;
  const int item = (int)blockIdx.x - level * a.n_base;
  const Work wk =
      schedule(a, BQ, lane, SPLIT ? split_item(a.HKV, item) : item);
  if (wk.seq < 0) {
    if (SPLIT && level == 0 && tid == 0) a.part_n[item] = 0;
    return;
  }
  const int t0 = wk.t0, len = wk.len, prior = max(wk.prior, 0);
  const int q0 = wk.qb * BQ;
  const int nk = prior + len;                 // keys of this run
  const int pos_lo = prior + q0;              // first query position
  const int pos_hi = pos_lo + min(BQ, len - q0) - 1;   // last valid one
  // first key any query of the block may see
  const int kwin = a.window > 0 ? max(0, pos_lo - a.window + 1) : 0;
  const Tiles tl = item_tiles(a, BQ, prior, len, wk.qb);
  int k_lo = tl.k_lo, ntiles = tl.n;
  int np = 1;
  if constexpr (SPLIT) {
    np = pieces_of<W>(a, BQ, lane, tl.n);
    if (level == 0 && tid == 0) a.part_n[item] = np;
    if (level >= np) return;
    const int b0 = (int)((int64_t)tl.n * level / np);
    k_lo += b0 * kBN;
    ntiles = (int)((int64_t)tl.n * (level + 1) / np) - b0;
  }

  // ---- this wave's row block: map, head pair and 32-query sub-block ------
  const int map = w / RB;
  const int hp = wk.kvh * REP + (w % RB) / QSUB;
  const int row0 = q0 + 32 * ((w % RB) % QSUB);
  const int qi = row0 + l32;                  // this lane's query (column)
  const bool qok = qi < len;
  const int qpos = prior + qi;
  const int kvs = 2 * (wk.kvh / a.kv_div);    // the first stored head
  // (what the end needs is fetched here: its latency would show there)
  const float lam = as_const(a.w.lam)[(int64_t)hp * a.w.lam_stride];
  const uint32_t wlds =
      (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)smem) +
      stages_of(W) * kStage + W * 128;

  // ---- tile loads ----------------------------------------------------------
  // Of eight waves, wave w moves key rows 4w..4w+3 of each of the four slices, one
  // 1 KB instruction each: lane l fills row l >> 4, physical 16-byte slot l & 15,
  // and fetches the logical chunk that belongs there. Of four, rows 8w..8w+7 by
  // two.
  const int grp = lane >> 4, slot = lane & 15;
  const int krow = 32 / W * w + grp;
  const int kchunk = slot ^ (krow & 15);
  const int vchunk = ((((slot >> 2) ^ grp) & 3) << 2) | (slot & 3);
  const uint32_t lds0 =
      (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)smem);
  const int kst_b = (int)(a.k_st * 2), vst_b = (int)(a.v_st * 2);
  // packed: one resource per slice, from the run's first row (rows past the run
  // lie outside it); paged: one per page, lane offsets from the page's rows
  i32x4 rk[2], rv[2];
  int klane, vlane;
  [[maybe_unused]] const int32_t __attribute__((address_space(4)))* trow =
      PAGED ? as_const(a.bt) + (int64_t)wk.seq * a.bt_stride : nullptr;
  if constexpr (PAGED) {
    klane = grp * kst_b + kvs * kRowB + 16 * kchunk;
    vlane = grp * vst_b + kvs * kRowB + 16 * vchunk;
  } else {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      rk[m] = make_rsrc(a.k + (int64_t)t0 * a.k_st + (kvs + m) * a.k_sh,
                        (uint32_t)(((int64_t)(len - 1) * a.k_st + kD) * 2));
      rv[m] = make_rsrc(a.v + (int64_t)t0 * a.v_st + (kvs + m) * a.v_sh,
                        (uint32_t)(((int64_t)(len - 1) * a.v_st + kD) * 2));
    }
    klane = grp * kst_b + 16 * kchunk;
    vlane = grp * vst_b + 16 * vchunk;
  }
  // Eight waves: tile t (index from k_lo) into LDS stage st: 4 instructions.
  // live == false issues the same ones fetching nothing: the loops issue a tile
  // every iteration, past the last one too, so that the count of loads in
  // flight is the same on every path and the waits are exact.
  auto issue_tile = [&](int t, int st, bool live = true)
      __attribute__((always_inline)) {
    const int key0 = k_lo + t * kBN + 4 * w;   // first of the wave's rows
    const uint32_t dst = lds0 + st * kStage + 4 * w * kRowB;
    if constexpr (PAGED) {
      // The resource covers the page's rows in [kwin, nk): others, and pages
      // without an entry, read as zeros and are never fetched.
      const int lp = key0 >> 4;
      const int pg = live && (unsigned)lp < (unsigned)a.bt_width ? trow[lp] : -1;
      const int r_lo = min(kPage, max(0, kwin - kPage * lp));
      const int r_hi = min(kPage, max(0, nk - kPage * lp));
      const bool valid = (unsigned)pg < (unsigned)a.num_pages && r_hi > r_lo;
      const uint32_t nrec = valid ? (uint32_t)((r_hi - r_lo) * kst_b) : 0u;
      const int64_t ofs =
          valid ? ((int64_t)pg * kPage + r_lo) * kst_b : 0;
      const int roff = ((key0 & (kPage - 1)) - r_lo) * kst_b;
      const i32x4 pk =
          make_rsrc(reinterpret_cast<const char*>(a.k) + ofs, nrec);
      const i32x4 pv =
          make_rsrc(reinterpret_cast<const char*>(a.v) + ofs, nrec);
      dma(pk, dst, klane + roff);
      dma(pk, dst + kSliceB, klane + roff + kRowB);
      dma(pv, dst + 2 * kSliceB, vlane + roff);
      dma(pv, dst + 3 * kSliceB, vlane + roff + kRowB);
    } else {
      const int ko = live ? klane + key0 * kst_b : kOob;
      const int vo = live ? vlane + key0 * vst_b : kOob;
      dma(rk[0], dst, ko);
      dma(rk[1], dst + kSliceB, ko);
      dma(rv[0], dst + 2 * kSliceB, vo);
      dma(rv[1], dst + 3 * kSliceB, vo);
    }
  };

  // Four waves: K (v 0) or V (v 1) of tile t into stage t & 1, nothing past the
  // last tile: the waits of these loads are for all of them.
  [[maybe_unused]] const int kstep = 16 * ((kchunk ^ 4) - kchunk);
  auto issue_half = [&](int t, int v) __attribute__((always_inline)) {
    if (t >= ntiles) return;
    const int key0 = k_lo + t * kBN + 8 * w;   // first of the wave's rows
    const uint32_t dst =
        lds0 + (t & 1) * kStage + 2 * v * kSliceB + 8 * w * kRowB;
    const int st_b = v ? vst_b : kst_b;
    i32x4 r0, r1;
    int o;
    if constexpr (PAGED) {   // (as above; the second head is 256 bytes on)
      const int lp = key0 >> 4;
      const int pg = (unsigned)lp < (unsigned)a.bt_width ? trow[lp] : -1;
      const int r_lo = min(kPage, max(0, kwin - kPage * lp));
      const int r_hi = min(kPage, max(0, nk - kPage * lp));
      const bool valid = (unsigned)pg < (unsigned)a.num_pages && r_hi > r_lo;
      r0 = r1 = make_rsrc(
          reinterpret_cast<const char*>(v ? a.v : a.k) +
              (valid ? ((int64_t)pg * kPage + r_lo) * kst_b : 0),
          valid ? (uint32_t)((r_hi - r_lo) * kst_b) : 0u);
      o = ((key0 & (kPage - 1)) - r_lo) * kst_b;
    } else {
      r0 = v ? rv[0] : rk[0];
      r1 = v ? rv[1] : rk[1];
      o = key0 * st_b;
    }
    constexpr int kHead = PAGED ? kRowB : 0;
    const int l0 = (v ? vlane : klane) + o;
    const int l1 = l0 + 4 * st_b + (v ? 0 : kstep);
    dma(r0, dst, l0);
    dma(r0, dst + 4 * kRowB, l1);
    dma(r1, dst + kSliceB, l0 + kHead);
    dma(r1, dst + kSliceB + 4 * kRowB, l1 + kHead);
  };

  // ---- LDS fragment addresses -------------------------------------------
  // K fragment kk of lane (l32, h2): row l32, logical chunk 2 kk + h2 -> slot
  // (2 kk + h2) ^ (l32 & 15).
  const uint32_t ka0 = (uint32_t)(map * kSliceB + l32 * kRowB +
                                  16 * (h2 ^ (l32 & 15)));
  // V^T fragment (db, kk) by two transposed reads: within each 16-lane group,
  // source lane s names key kbase + (s >> 2), dims 4 (s & 3)..+3 of a 16-dim
  // half; lane i of the group then holds dim dbase + i of keys kbase..kbase+3.
  // kbase = 16 kk + 4 h2 (+8 for the second read), dbase = 32 db + 16 (l32 >>
  // 4): the order of this lane's probabilities.
  const int s16 = lane & 15;
  const uint32_t va0 = (uint32_t)(2 * kSliceB + (4 * h2 + (s16 >> 2)) * kRowB +
                                  64 * (s16 >> 2) + 32 * ((lane >> 4) & 1) +
                                  8 * (s16 & 3));
  auto kfrag = [&](uint32_t sb, int kk) -> bf16x8 {
    return lds_ld128((sb + ka0) ^ (32u * kk));
  };
  auto vfrag = [&](uint32_t sb, int db, int kk) -> bf16x8 {
    const uint32_t p = ((sb + va0) ^ (64u * (db & 3))) + (db >> 2) * kSliceB +
                       16 * kk * kRowB;
    const bf16x4 lo = lds_tr16(p);
    const bf16x4 hi = lds_tr16(p + 8 * kRowB);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  bf16x8 qf[8];   // B operand of S^T (column = query, k = dims)
  f32x16 o_acc[8];
#pragma unroll
  for (int db = 0; db < 8; ++db) o_acc[db] = f32x16{};
  float m_run = -INFINITY;
  float l_part = 0.0f;
  f32x16 sc;       // scores of the tile after the one being multiplied
  bf16x8 pf[2];    // probabilities of the tile being multiplied

  // Softmax of the scores of the tile at kt: P^T fragments, running maximum and
  // sum, O^T rescaled when the maximum moved. The maximum only moves when the
  // tile's exceeds it by more than 2^kLazy, so that O^T is rescaled on few
  // tiles; O / l and the LSE are exact for any reference point. Element j of
  // the scores holds key kt + 4 h2 + 8 (j >> 2) + (j & 3). `hook` runs first.
  auto softmax_phase = [&](int kt, bool first, auto&& hook)
      __attribute__((always_inline)) {
    // a tile every valid query of the block sees whole (columns past the run
    // end hold zero queries and are never stored)
    const bool full = (kt + kBN - 1 <= pos_lo) && (kt + kBN <= nk) &&
                      (a.window == 0 || pos_hi - kt < a.window);
    hook();
    if (!full) {
      const int base = kt + 4 * h2;
      const int hi = qok ? min(qpos, nk - 1) - base : -1;
      const int lo = a.window > 0 ? qpos - a.window - base : -1;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int c = 8 * (j >> 2) + (j & 3);
        sc[j] = (c <= hi && c > lo) ? sc[j] : -INFINITY;
      }
    }
    const float sl2 = a.scale_log2;
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; j += 2) mx = fmaxf(fmaxf(mx, sc[j]), sc[j + 1]);
    mx = lane_pair(mx, 32, true);
    const float m_cand = mx * sl2;
    const bool move = m_cand > m_run + kLazy;
    const float m_new = move ? m_cand : m_run;
    const float m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = move ? fast_exp2(m_run - m_use) : 1.0f;
    m_run = m_new;
    float psum = 0.0f;
    uint32_t pw[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float p0 = fast_exp2(__builtin_fmaf(sc[2 * q], sl2, -m_use));
      const float p1 = fast_exp2(__builtin_fmaf(sc[2 * q + 1], sl2, -m_use));
      psum += p0 + p1;
      // (the matrix operand's type: each is off by half a step, 2^-8 of it, at
      // most, the sum above keeps 32 bits; against 64 bits outputs are off by
      // 2.0e-3 to 2.2e-3 where fp32 probabilities give 1.7e-3, which is the
      // outputs' own rounding)
      pw[q] = pack_bf16x2_rn(p0, p1);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
      pf[kk] = __builtin_bit_cast(
          bf16x8, u32x4{pw[4 * kk], pw[4 * kk + 1], pw[4 * kk + 2],
                        pw[4 * kk + 3]});
    l_part = l_part * alpha + psum;
    // (in place, each product tied to its accumulator register: a plain
    // multiply under the branch costs a second copy of O^T)
    if (!first && __builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float x = o_acc[db][j];
          asm volatile("v_mul_f32 %0, %1, %0" : "+v"(x) : "v"(alpha));
          o_acc[db][j] = x;
        }
    }
  };

  // MFMA phase of tile t: O^T += V^T.P^T for tile t, with the scores of tile
  // t + 1 after every second MFMA, fragments read kRing - 1 MFMAs ahead.
  auto mfma_phase = [&](int t, auto with_s_c) __attribute__((always_inline)) {
    constexpr bool with_s = decltype(with_s_c)::value;
    // this wave's MFMAs first; the softmax wave fills the issue slots between
    __builtin_amdgcn_s_setprio(1);
    const uint32_t vb = lds0 + (t & (stages_of(W) - 1)) * kStage;
    const uint32_t kb = lds0 + ((t + 1) & (stages_of(W) - 1)) * kStage;
    constexpr int R = kRing, RK = 3;
    bf16x8 vf[R], kf[RK];
#pragma unroll
    for (int i = 0; i < R - 1; ++i) vf[i] = vfrag(vb, i & 7, i >> 3);
    if (with_s) {
#pragma unroll
      for (int i = 0; i < RK - 1; ++i) kf[i] = kfrag(kb, i);
    }
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      const int x = n + R - 1;
      if (x < 16) vf[x % R] = vfrag(vb, x & 7, x >> 3);
      o_acc[n & 7] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          vf[n % R], pf[n >> 3], o_acc[n & 7], 0, 0, 0);
      if (with_s && (n & 1)) {
        const int kk = n >> 1, y = kk + RK - 1;
        if (y < 8) kf[y % RK] = kfrag(kb, y);
        sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            kf[kk % RK], qf[kk], kk == 0 ? f32x16{} : sc, 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto first_scores = [&] {
    sc = f32x16{};
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
      sc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kfrag(lds0, kk), qf[kk], sc,
                                                   0, 0, 0);
  };

  const bool rejected = a.reject != nullptr && as_const(a.reject)[0] != 0;
  if (!rejected) {
    // Eight waves. Slot 2t: group 0 multiplies tile t, group 1 does the softmax
    // of tile t; slot 2t + 1: group 0 the softmax of tile t + 1, group 1
    // multiplies tile t. Tile t + 3 goes out at the start of slot 2t into the
    // stage of tile t - 1 (last read in slot 2t - 1) and must be in LDS before
    // slot 2t + 4; each wave waits for its own part at the end of every odd
    // slot, before the barrier that publishes it. Four waves. K runs a tile
    // ahead of V: after the products of tile t and the scores of tile t + 1, a
    // barrier frees V(t) and K(t + 1) for V(t + 2) and K(t + 3), which have
    // until the next one to arrive. The queries come first, each wave's own 32
    // rows through its 8 KB of the last stages (rows past the run end arrive as
    // zeros).
    if (w == 0 && a.w.weight)
      dma(make_rsrc(a.w.weight, kDV * 4), wlds, 16 * lane);
    const uint32_t qlds =
        lds0 + stages_of(W) / 2 * kStage + (uint32_t)w * (32 * kRowB);
    {
      const int64_t span = ((int64_t)(len - row0 - 1) * a.q_st + kD) * 2;
      const i32x4 rq = make_rsrc(a.q + (int64_t)(t0 + row0) * a.q_st +
                                     (int64_t)(2 * hp + map) * a.q_sh,
                                 row0 < len ? (uint32_t)span : 0u);
      const int qst_b = (int)(a.q_st * 2);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + grp;
        dma(rq, qlds + i * 1024, r * qst_b + 16 * (slot ^ (r & 15)));
      }
    }
    if constexpr (W == 8) {
      issue_tile(0, 0);
      issue_tile(1, 1, ntiles > 1);
    } else {
      issue_half(0, 0);
      issue_half(0, 1);
    }
    wait_vm<8>();   // the queries
    asm volatile("" ::: "memory");
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      u32x4 x = __builtin_bit_cast(
          u32x4,
          lds_ld128(qlds + l32 * kRowB + 16 * ((2 * kk + h2) ^ (l32 & 15))));
      if (!qok) x = u32x4{0, 0, 0, 0};
      qf[kk] = __builtin_bit_cast(bf16x8, x);
    }
    wait_vm<0>();
    __syncthreads();   // tile 0 (of four stages, 1 too) is there, the others free
    if constexpr (W == 8) {
      if (ntiles > 2) issue_tile(2, 2);
    } else {
      issue_half(1, 0);
      issue_half(1, 1);
    }
    auto odd_end = [&](int n) {
      if (n == 4) wait_vm<4>();
      else wait_vm<0>();
      __syncthreads();
    };
    // (the first and last tiles are peeled off the loops, so that these hold
    // one variant of the MFMA phase and O^T keeps one set of registers)
    constexpr std::true_type kWithS{};
    constexpr std::false_type kNoS{};
    auto none = [] {};
    if constexpr (W == 4) {
      first_scores();
      softmax_phase(k_lo, true, none);
      odd_end(0);   // tile 1 is there, K(0) free
      issue_half(2, 0);
      for (int t = 0; t + 1 < ntiles; ++t) {
        mfma_phase(t, kWithS);
        odd_end(0);
        issue_half(t + 2, 1);
        issue_half(t + 3, 0);
        softmax_phase(k_lo + (t + 1) * kBN, false, none);
      }
      mfma_phase(ntiles - 1, kNoS);
      odd_end(0);
    } else if (map == 0) {
      first_scores();
      softmax_phase(k_lo, true, none);
      for (int t = 0; t + 1 < ntiles; ++t) {
        issue_tile(t + 3, (t + 3) & 3, t + 3 < ntiles);
        mfma_phase(t, kWithS);
        softmax_phase(k_lo + (t + 1) * kBN, false, none);
        odd_end(4);
      }
      mfma_phase(ntiles - 1, kNoS);
      odd_end(0);   // everything, before the outputs go through LDS
    } else {
      issue_tile(3, 3, 3 < ntiles);
      first_scores();
      softmax_phase(k_lo, true, none);
      if (ntiles > 1) mfma_phase(0, kWithS);
      else mfma_phase(0, kNoS);
      odd_end(ntiles > 1 ? 4 : 0);
      for (int t = 1; t + 1 < ntiles; ++t) {
        softmax_phase(k_lo + t * kBN, false, [&] {
          issue_tile(t + 3, (t + 3) & 3, t + 3 < ntiles);
        });
        mfma_phase(t, kWithS);
        odd_end(4);
      }
      if (ntiles > 1) {
        const int t = ntiles - 1;
        softmax_phase(k_lo + t * kBN, false, none);
        mfma_phase(t, kNoS);
        odd_end(0);
      }
    }
  }

  // ---- the maps meet: normalise, difference, norm, store -------------------
  const float l_tot = lane_pair(l_part, 32, false);
  const float inv = rejected ? __builtin_nanf("") :
                    l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
  // (a key that is no number makes the sum none: neither is the LSE)
  const float lse_nat =
      l_tot == 0.0f ? -INFINITY : (m_run + fast_log2(l_tot)) * kLn2;
  if (SPLIT && np > 1) {
    // lane-major partial: every store writes 1 KB (of rows past the run,
    // nothing)
    const int64_t pw = (int64_t)blockIdx.x * W + w;
    float* const po = a.part_o + (pw * 32 * 64 + lane) * 4;
    if (qok)
#pragma unroll
      for (int db = 0; db < 8; ++db)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
          *reinterpret_cast<f32x4*>(po + (4 * db + g4) * 256) =
              f32x4{o_acc[db][4 * g4] * inv, o_acc[db][4 * g4 + 1] * inv,
                    o_acc[db][4 * g4 + 2] * inv, o_acc[db][4 * g4 + 3] * inv};
    if (h2 == 0)
      a.part_lse[pw * 32 + l32] =
          rejected ? __builtin_nanf("") : lse_nat;
    return;
  }
  if (a.lse && h2 == 0 && qok)
    a.lse[(2 * hp + map) * a.lse_sh + t0 + qi] =
        rejected ? __builtin_nanf("") : lse_nat;
  // dims 128 map .. +127 are this wave's; the others go to its partner, lane by
  // lane (16 bytes each: 1 KB per store)
  const uint32_t mine = lds0 + (uint32_t)w * 16384 + 16 * lane;
  const uint32_t theirs = lds0 + (uint32_t)(w ^ RB) * 16384 + 16 * lane;
  f32x4 d[16];   // chunk c: dims 8c + 4 h2 .. +3 of the half
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const int db = c >> 2, j = 4 * (c & 3);
    const f32x4 lo = f32x4{o_acc[db][j], o_acc[db][j + 1], o_acc[db][j + 2],
                           o_acc[db][j + 3]} * inv;
    const f32x4 hi = f32x4{o_acc[4 + db][j], o_acc[4 + db][j + 1],
                           o_acc[4 + db][j + 2], o_acc[4 + db][j + 3]} * inv;
    d[c] = map == 0 ? lo : hi;
    lds_st128(mine + c * 1024,
              __builtin_bit_cast(u32x4, map == 0 ? hi : lo));
  }
  __syncthreads();
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < 16; ++c) {
    const f32x4 y = __builtin_bit_cast(f32x4, lds_ld128(theirs + c * 1024));
    d[c] = map == 0 ? d[c] - y * lam : y - d[c] * lam;
    ss += (d[c][0] * d[c][0] + d[c][1] * d[c][1]) +
          (d[c][2] * d[c][2] + d[c][3] * d[c][3]);
  }
  const uint32_t sums = lds0 + stages_of(W) * kStage;
  if (a.w.weight) {
    ss = lane_pair(ss, 32, false);
    if (h2 == 0)
      *(__attribute__((address_space(3))) float*)(uintptr_t)(sums + 128 * w +
                                                             4 * l32) = ss;
  }
  __syncthreads();   // (and both halves of the exchange have been read)
  if (a.w.weight) {
    f32x4 wt[16];
#pragma unroll
    for (int c = 0; c < 16; ++c)
      wt[c] = __builtin_bit_cast(
          f32x4, lds_ld128(wlds + 4 * (128 * map + 8 * c + 4 * h2)));
    ss += __builtin_bit_cast(float, lds_ld32(sums + 128 * (w ^ RB) + 4 * l32));
    const float f =
        a.w.out_scale * __builtin_amdgcn_rsqf(ss * (1.0f / kDV) + a.w.eps);
#pragma unroll
    for (int c = 0; c < 16; ++c) d[c] = d[c] * f * wt[c];
  } else {
#pragma unroll
    for (int c = 0; c < 16; ++c) d[c] = d[c] * a.w.out_scale;
  }
  // Through LDS, so that the stores are whole rows: 32 queries x 128 dims,
  // query-major (256-byte rows, 16-byte chunks swizzled by row & 15), then 4
  // complete rows per store instruction.
  const uint32_t ob = lds0 + (uint32_t)w * 16384;
#pragma unroll
  for (int c = 0; c < 16; ++c)   // 16-byte chunk: dims 8c .. 8c+7
    lds_st64(ob + l32 * kRowB + 16 * (c ^ (l32 & 15)) + 8 * h2,
             u32x2{pack_bf16x2_rn(d[c][0], d[c][1]),
                   pack_bf16x2_rn(d[c][2], d[c][3])});
  wave_lds_sync();
  u32x4 y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + grp;
    y[i] = __builtin_bit_cast(
        u32x4, lds_ld128(ob + r * kRowB + 16 * (slot ^ (r & 15))));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = 4 * i + grp;
    if (row0 + r < len)
      *reinterpret_cast<u32x4*>(a.out + (int64_t)(t0 + row0 + r) * a.o_st +
                                (int64_t)hp * a.o_sh + 128 * map + 8 * slot) =
          y[i];
  }
}

// Join the pieces of the items that were split, in a fixed order: grid (n_base,
// 16), a work-group per 8 query rows of both maps. Thread t of a group of 256
// has row t & 7 and dims 8 (t >> 3) .. +7 of both, so the difference is its own
// and the norm one sum over threads. Group s of S takes pieces s, s + S, ...,
// four pieces' loads in flight at a time; the groups' results then join through
// LDS in order.
template <int W, int REP, int S>
__global__ __launch_bounds__(256 * S) void prefill_diff_merge(
    PrefillDiffArgs a) {
  constexpr int RB = W / 2, BQ = 32 * RB / REP, QSUB = BQ / 32, kBatch = 4;
  __shared__ float sums[4][8];
  __shared__ float part[S > 1 ? S - 1 : 1][20][S > 1 ? 256 : 1];
  const int np = min(as_const(a.part_n)[blockIdx.x], a.nsplit);
  if (np <= 1) return;                        // no item, or written in place
  const int lane = threadIdx.x & 63;
  const int tid = threadIdx.x & 255, w = tid >> 6;
  const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8);
  const Work wk =
      schedule(a, BQ, lane, split_item(a.HKV, (int)blockIdx.x));
  const int rb = blockIdx.y >> 2;             // 32-row block of the item
  const int l32 = 8 * (blockIdx.y & 3) + (tid & 7);
  const int c = tid >> 3;                     // 8-dim chunk
  const int row0 = wk.qb * BQ + 32 * (rb % QSUB) + 8 * (blockIdx.y & 3);
  if (row0 >= wk.len) return;
  const int qi = row0 + (tid & 7);
  const int hp = wk.kvh * REP + rb / QSUB;
  const float lam = a.w.lam[(int64_t)hp * a.w.lam_stride];
  const bool norm = a.w.weight != nullptr;
  f32x4 wt[2] = {};
  if (norm) {
    wt[0] = *reinterpret_cast<const f32x4*>(a.w.weight + 8 * c);
    wt[1] = *reinterpret_cast<const f32x4*>(a.w.weight + 8 * c + 4);
  }
  float m[2] = {-INFINITY, -INFINITY}, sum[2] = {0, 0};
  f32x4 acc[2][2] = {};
  auto add = [&](int i, float l, float w1, const f32x4 (&o)[2]) {
    const float m_new = fmaxf(m[i], l);
    const float m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float keep = fast_exp2((m[i] - m_use) * kLog2e);
    const float wt = fast_exp2((l - m_use) * kLog2e);
    sum[i] = sum[i] * keep + wt * w1;
#pragma unroll
    for (int x = 0; x < 2; ++x) acc[i][x] = acc[i][x] * keep + o[x] * wt;
    m[i] = m_new;
  };
  for (int s0 = group; qi < wk.len && s0 < np; s0 += kBatch * S) {
    float l[kBatch][2];
    f32x4 o[kBatch][2][2];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int64_t slot =
          (int64_t)min(s0 + j * S, np - 1) * a.n_base + blockIdx.x;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t pw = slot * W + RB * i + rb;
        l[j][i] = a.part_lse[pw * 32 + l32];
#pragma unroll
        for (int x = 0; x < 2; ++x)
          o[j][i][x] = *reinterpret_cast<const f32x4*>(
              a.part_o + ((pw * 32 + c) * 64 + 32 * x + l32) * 4);
      }
    }
    __builtin_amdgcn_sched_barrier(0);   // (all of them, before the first use)
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (s0 + j * S >= np) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) add(i, l[j][i], 1.0f, o[j][i]);
    }
  }
  if constexpr (S > 1) {
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        part[group - 1][10 * i][tid] = m[i];
        part[group - 1][10 * i + 1][tid] = sum[i];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          part[group - 1][10 * i + 2 + e][tid] = acc[i][e >> 2][e & 3];
      }
    }
    __syncthreads();
    if (group == 0)
      for (int g = 0; g + 1 < min(np, S); ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x4 o[2];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            o[e >> 2][e & 3] = part[g][10 * i + 2 + e][tid];
          add(i, part[g][10 * i][tid], part[g][10 * i + 1][tid], o);
        }
  }
  // (a rejected launch's pieces are NaN, and so are their sums)
  const bool rejected = a.reject != nullptr && as_const(a.reject)[0] != 0;
  const bool qok = group == 0 && qi < wk.len;
  if (a.lse && c < 2 && qok)
    a.lse[(2 * hp + c) * a.lse_sh + wk.t0 + qi] =
        rejected ? __builtin_nanf("") :
        sum[c] == 0.0f ? -INFINITY : m[c] + fast_log2(sum[c]) * kLn2;
  const float inv0 = sum[0] > 0.0f ? 1.0f / sum[0] : 0.0f;
  const float inv1 = sum[1] > 0.0f ? 1.0f / sum[1] : 0.0f;
  float ss = 0.0f;
  f32x4 d[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    d[x] = acc[0][x] * inv0 - acc[1][x] * (lam * inv1);
    if (rejected) d[x] = d[x] + __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += d[x][i] * d[x][i];
  }
  float f = a.w.out_scale;
  if (a.w.weight) {
    ss += __shfl_xor(ss, 8);
    ss = lane_pair(lane_pair(ss, 16, false), 32, false);
    if (group == 0 && lane < 8) sums[w][lane] = ss;
    __syncthreads();
    const int q = tid & 7;
    ss = (sums[0][q] + sums[1][q]) + (sums[2][q] + sums[3][q]);
    f *= __builtin_amdgcn_rsqf(ss * (1.0f / kDV) + a.w.eps);
  }
  u32x4 y;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    f32x4 z = d[x] * f;
    if (norm) z *= wt[x];
    y[2 * x] = pack_bf16x2_rn(z[0], z[1]);
    y[2 * x + 1] = pack_bf16x2_rn(z[2], z[3]);
  }
  if (qok)
    *reinterpret_cast<u32x4*>(a.out + (int64_t)(wk.t0 + qi) * a.o_st +
                              (int64_t)hp * a.o_sh + 8 * c) = y;
}

// Work-groups of one level: scheduled pairs * items of each, rounded up to
// whole XCD rounds.
int64_t level_wgs(int pairs, int BQ, int64_t S, int max_seqlen) {
  const int64_t items = S * ((max_seqlen + BQ - 1) / BQ);
  if (pairs <= 8 && 8 % pairs == 0)
    return 8 * ((items + 8 / pairs - 1) / (8 / pairs));
  return pairs * items;
}

// Head pairs per work-group: the largest of 4 (eight waves), 2, 1 dividing HQ /
// HKV; a larger ratio runs as several scheduled pairs per stored one.
int group_of(int ratio, int most) {
  return most >= 4 && ratio % 4 == 0 ? 4 : ratio % 2 == 0 ? 2 : 1;
}

// How a launch is laid out: work-groups of W waves for rep head pairs and BQ
// queries, in levels (1: keys are not split) of n_base.
struct Layout {
  int W, rep, pairs, BQ;
  int levels;
  int64_t n_base;
};
Layout groups_of(int W, int HQ, int HKV) {
  const int rep = group_of(HQ / HKV, W / 2);
  return Layout{W, rep, HQ / 2 / rep, 16 * W / rep, 1, 0};
}

// From what the host knows: the longest run, and the row width of a block
// table, the longest context or the window as bounds of its keys. Up to half the compute units' worth of
// items, as many pieces as there are units; up to one and a half, two or three
// pieces an item even out the rounds where keys are many (below 128 tiles two
// work-groups per unit do it better: a prompt of 1200, 32Q/4KV, 48.8 us a call
// in pieces, 40.5 whole, of 3000, 16Q/2KV, 99.5 / 92.5); larger grids fill the
// chip by themselves. The device decides from the lengths. Four waves where all
// whole items, or the pieces at 20 tiles each or less, are on the chip at once:
// there an item's start and end weigh most. Graph replays of split calls, us,
// eight / four waves: 16 tokens after 1000, 64Q/8KV 21.7 / 19.3, 300 after
// 1000, 32Q/4KV 38.7 / 35.6, 128 after 8000, 16Q/2KV 45 / 41.8; 64 after
// 30,000, 64Q/8KV 114 / 123, one after 20,000 48 / 68 (keys are read for half
// as many rows). And where no query sees more than 8 tiles: 128 prompts of 128,
// 32Q/4KV 124 / 113, of 200 242 / 212, 128 of 500 under a window of 100 555 /
// 513 (64 of 256 142 / 146, 40 of 300, 64Q/8KV 234 / 239).
Layout layout_of(int HQ, int HKV, int64_t S, int max_seqlen,
                 int64_t max_context, int64_t bt_stride, int window,
                 bool split) {
  const int64_t cus = device_cus();
  const Layout w4 = groups_of(4, HQ, HKV), w8 = groups_of(8, HQ, HKV);
  auto count = [&](const Layout& x) {
    return S * ((max_seqlen + x.BQ - 1) / x.BQ) * x.pairs;
  };
  auto tiles_of = [&](const Layout& x) {
    int64_t keys = bt_stride > 0 ? bt_stride * kPage : max_seqlen;
    if (max_context > 0) keys = std::min(keys, max_context);
    if (window > 0 && keys > (int64_t)window + x.BQ + kBN)
      keys = (int64_t)window + x.BQ + kBN;
    return (keys + kBN - 1) / kBN;
  };
  const int64_t few = count(w4);
  // (packed runs see half of their keys)
  const bool four =
      few <= cus && few * tiles_of(w4) <= (bt_stride > 0 ? 20 : 40) * cus;
  Layout r = four ? w4 : w8;
  const int64_t items = count(r), tiles = tiles_of(r);
  int64_t n = (2 * items <= cus ? cus : 3 * cus) * (four ? 2 : 1) / items;
  if (n > 64) n = 64;
  // a piece costs some 5 tiles' time, so it must have more than that
  if (n > tiles / 8) n = tiles / 8;
  if (split && n >= 2 && tiles >= (2 * items <= cus ? 32 : 128)) {
    r.levels = (int)n;
    r.n_base = items;
    return r;
  }
  r = w4;
  r.n_base = level_wgs(r.pairs, r.BQ, S, max_seqlen);
  if (r.n_base <= 2 * cus || tiles_of(w4) <= 8) return r;
  r = w8;
  r.n_base = level_wgs(r.pairs, r.BQ, S, max_seqlen);
  return r;
}

int64_t workspace_bytes_of(const Layout& x) {
  if (x.levels <= 1) return 0;
  return x.levels * x.n_base * x.W * 32 * (kDV + 1) * (int64_t)sizeof(float) +
         ((x.n_base * 4 + 15) & ~(int64_t)15);
}

template <int W, int REP, bool SPLIT>
int launch_whole(const PrefillDiffArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.nsplit * a.n_base));
  if (a.bt)
    hipLaunchKernelGGL((prefill_diff_kernel<W, REP, true, SPLIT>), grid,
                       dim3(64 * W), lds_of(W), st, a);
  else
    hipLaunchKernelGGL((prefill_diff_kernel<W, REP, false, SPLIT>), grid,
                       dim3(64 * W), lds_of(W), st, a);
  return check_launch("prefill_diff");
}

template <int W, int REP>
int launch(const PrefillDiffArgs& a, hipStream_t st) {
  if (a.nsplit <= 1) return launch_whole<W, REP, false>(a, st);
  const int rc = launch_whole<W, REP, true>(a, st);
  if (rc) return rc;
  // many pieces of few items: four groups (3 queries after 22,000, 16Q/2KV, 58
  // us a call with one and the pieces of an item on one XCD, 48 so)
  const dim3 grid(a.n_base, 2 * W);
  if (a.nsplit > 8)
    hipLaunchKernelGGL((prefill_diff_merge<W, REP, 4>), grid, dim3(1024), 0, st,
                       a);
  else
    hipLaunchKernelGGL((prefill_diff_merge<W, REP, 1>), grid, dim3(256), 0, st,
                       a);
  return check_launch("prefill_diff_merge");
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" size_t tmopt_attn_prefill_diff_workspace_size(
    int num_seqs, int max_seqlen_q, int64_t max_context, int HQ, int HKV,
    int64_t bt_stride, int window) {
  if (num_seqs <= 0 || max_seqlen_q <= 0 || HQ <= 0 || HKV <= 0 ||
      HKV % 2 != 0 || HQ % HKV != 0)
    return 0;
  return (size_t)workspace_bytes_of(
      layout_of(HQ, HKV, num_seqs, max_seqlen_q, max_context, bt_stride, window,
                true));
}

extern "C" int tmopt_attn_prefill_diff(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k,
    int64_t k_stride_tok, int64_t k_stride_head, const void* v,
    int64_t v_stride_tok, int64_t v_stride_head, const int32_t* cu_seqlens_q,
    const int32_t* prior_lens, int num_seqs, int max_seqlen_q,
    int64_t max_context, const void* k_pool, const void* v_pool,
    const int32_t* block_table, int64_t bt_stride, int page_size,
    int64_t num_pages, int HQ, int HKV, int D, int window, float scale,
    const float* lam, int lam_stride, const float* norm_weight, float norm_eps,
    float out_scale, void* out, int64_t o_stride_tok, int64_t o_stride_head,
    float* lse, int64_t lse_stride_head, const int32_t* reject, void* workspace,
    size_t workspace_bytes, tmopt_stream_t stream) {
  clear_error();
  if (num_seqs == 0 || max_seqlen_q == 0) return TMOPT_OK;
  TMOPT_REQUIRE(num_seqs > 0 && num_seqs <= 65535 && max_seqlen_q > 0,
                TMOPT_EINVAL, "prefill_diff: num_seqs=%d max_seqlen_q=%d",
                num_seqs, max_seqlen_q);
  TMOPT_REQUIRE(q && out && cu_seqlens_q, TMOPT_EINVAL,
                "prefill_diff: null q/out/cu_seqlens");
  TMOPT_REQUIRE(max_context >= 0, TMOPT_EINVAL,
                "prefill_diff: max_context=%lld", (long long)max_context);
  const int rc = check_diff("prefill_diff", HQ, HKV, D, window, scale, lam,
                            lam_stride, norm_weight, norm_eps);
  if (rc) return rc;
  constexpr int64_t kSpan = 0x7ffffff0;   // bytes a buffer resource reaches
  TMOPT_REQUIRE(q_stride_tok >= 0 && q_stride_head >= 0 &&
                    q_stride_tok % 8 == 0 && q_stride_head % 8 == 0 &&
                    (uintptr_t)q % 16 == 0 && o_stride_tok % 8 == 0 &&
                    o_stride_head % 8 == 0 && (uintptr_t)out % 16 == 0,
                TMOPT_EINVAL, "prefill_diff: q/out rows misaligned");
  TMOPT_REQUIRE(((int64_t)max_seqlen_q * q_stride_tok + kD) * 2 < kSpan,
                TMOPT_EUNSUPPORTED,
                "prefill_diff: a run's q span must stay below 2 GiB");
  const bool paged = block_table != nullptr;
  if (paged) {
    TMOPT_REQUIRE(!k && !v, TMOPT_EINVAL,
                  "prefill_diff: keys come from k/v or from the pools");
    TMOPT_REQUIRE(k_pool && v_pool && bt_stride > 0 && num_pages > 0,
                  TMOPT_EINVAL,
                  "prefill_diff: the paged source needs pools and bt_stride");
    TMOPT_REQUIRE(page_size == kPage, TMOPT_EUNSUPPORTED,
                  "prefill_diff: page_size=%d (only 16)", page_size);
    TMOPT_REQUIRE(((uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0,
                  TMOPT_EINVAL, "prefill_diff: pools must be 16-byte aligned");
  } else {
    TMOPT_REQUIRE(k && v, TMOPT_EINVAL,
                  "prefill_diff: the packed source needs k and v");
    TMOPT_REQUIRE(!prior_lens, TMOPT_EINVAL,
                  "prefill_diff: prior context needs a block table");
    TMOPT_REQUIRE(k_stride_tok >= 0 && k_stride_head >= 0 &&
                      v_stride_tok >= 0 && v_stride_head >= 0 &&
                      (k_stride_tok | k_stride_head | v_stride_tok |
                       v_stride_head) % 8 == 0 &&
                      ((uintptr_t)k | (uintptr_t)v) % 16 == 0,
                  TMOPT_EINVAL, "prefill_diff: k/v rows misaligned");
    const int64_t st =
        k_stride_tok > v_stride_tok ? k_stride_tok : v_stride_tok;
    TMOPT_REQUIRE(((int64_t)max_seqlen_q * st + kD) * 2 < kSpan,
                  TMOPT_EUNSUPPORTED,
                  "prefill_diff: a run's k/v span must stay below 2 GiB");
  }
  const Layout x =
      layout_of(HQ, HKV, num_seqs, max_seqlen_q, max_context,
                paged ? bt_stride : 0, window, workspace != nullptr);
  TMOPT_REQUIRE(x.n_base < 0x7fffffff, TMOPT_EUNSUPPORTED,
                "prefill_diff: %lld work-groups exceed the grid limit",
                (long long)x.n_base);
  const int64_t need = workspace_bytes_of(x);
  TMOPT_REQUIRE(need == 0 || ((int64_t)workspace_bytes >= need &&
                              (uintptr_t)workspace % 16 == 0),
                TMOPT_EWORKSPACE,
                "prefill_diff: workspace %zu bytes < %lld needed (or unaligned)",
                workspace_bytes, (long long)need);
  PrefillDiffArgs a;
  a.q = (const __bf16*)q;
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_head;
  a.k = (const __bf16*)(paged ? k_pool : k);
  a.v = (const __bf16*)(paged ? v_pool : v);
  a.k_st = paged ? (int64_t)HKV * kD : k_stride_tok;
  a.v_st = paged ? (int64_t)HKV * kD : v_stride_tok;
  a.k_sh = paged ? kD : k_stride_head;
  a.v_sh = paged ? kD : v_stride_head;
  a.cu = cu_seqlens_q;
  a.prior = prior_lens;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.bt_width = bt_stride > 0x7fffffff ? 0x7fffffff : (int)bt_stride;
  a.num_pages = num_pages > 0x7fffffff ? 0x7fffffff : (int)num_pages;
  a.HQ = HQ;
  a.HKV = x.pairs;
  a.kv_div = HQ / HKV / x.rep;
  a.S = num_seqs;
  a.nqb_max = (max_seqlen_q + x.BQ - 1) / x.BQ;
  a.window = window;
  a.scale_log2 = scale * kLog2e;
  a.w = DiffWeights{lam, lam_stride, norm_weight, norm_eps, out_scale};
  a.out = (__bf16*)out;
  a.o_st = o_stride_tok;
  a.o_sh = o_stride_head;
  a.lse = lse;
  a.lse_sh = lse_stride_head;
  a.reject = reject;
  a.nsplit = x.levels;
  a.n_base = (int)x.n_base;
  a.cus = device_cus();
  const int64_t rows = x.levels * x.n_base * x.W * 32;
  a.part_o = (float*)workspace;
  a.part_lse = a.part_o + rows * kDV;
  a.part_n = (int*)(a.part_lse + rows);
  const hipStream_t st = (hipStream_t)stream;
  if (x.W == 4) return x.rep == 2 ? launch<4, 2>(a, st) : launch<4, 1>(a, st);
  if (x.rep == 4) return launch<8, 4>(a, st);
  if (x.rep == 2) return launch<8, 2>(a, st);
  return launch<8, 1>(a, st);
}
