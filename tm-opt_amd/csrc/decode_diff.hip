// Differential attention of one new token per request over the paged cache,
// split over the cache's length and joined, for gfx950 (see diff.h for the
// formula).
//
// HBM bound: every visible token's K and V rows are read once (1 KB per pair of
// stored heads), for up to eight head pairs at a time.
//
//  * Both maps of up to eight head pairs are the 16 columns of one MFMA tile:
//    column c is map c >> 3 of pair c & 7. S^T = K.Q^T of a 16-token page is
//    taken with both key heads (v_mfma_f32_16x16x32_bf16), and each lane keeps
//    the product of its column's own one. The values are shared: O^T = V^T.P^T
//    (v_mfma_f32_16x16x16_bf16) multiplies the page's 256-wide values by all
//    columns at once. A plain attention kernel run once per map would read K
//    once and V twice.
//  * Pages of all requests are laid end to end and dealt out in equal
//    contiguous ranges, so that a launch streams the same bytes everywhere
//    whatever the lengths, and its grid does not depend on them (a captured
//    call stays valid). A piece of a request that one range does not hold whole
//    leaves a normalised fp32 result of both maps with their LSE;
//    decode_diff_merge joins the pieces in order, then takes the difference and
//    the norm. No atomics: repeated calls are bitwise equal.
//  * A range belongs to two waves where a work-group has fewer than four pairs
//    of stored heads: the first walks its first half forward, the second its
//    second half backward, so that the request in the middle is the last of
//    both, and they join it in LDS. A 256-wide fp32 row per map and piece is
//    what the split costs, twice that of plain attention.
//  * One page is a wave's step: 16 KB (two K and two V slices of 16 tokens)
//    straight into LDS (buffer_load ... lds), two steps ahead. The resource of
//    a load is the page's rows that hold visible keys; other rows read as zeros
//    and cost no traffic, so every step issues the same loads and the waits
//    count exactly.
//  * Page ids of a range and the norm's weights are fetched into LDS before the
//    walk: a load within it would wait for every page on its way.
//
// Us a call, the merge included (32Q/4KV with the norm unless said): 64
// requests of 1K-8K tokens 103.2, 5.9 TB/s (1.00 of the bytes fetched are the
// formula's); 96 under a window of 512, 64Q/16KV, 66.0, 6.1 TB/s; one of 50,001
// tokens 33.0, 3.1 TB/s: its walk runs at 7.3 TB/s, 5 us go to the start, 8 to
// the merge of its 184 pieces; 4 of 128-1024 tokens 14.0 in a graph, 17.9
// eagerly: two launches and their chains of dependent loads.
#include <algorithm>

#include "diff.h"

namespace tmopt {
namespace {

constexpr int kRowB = 256;                 // one token's slice of a stored head
constexpr int kSliceB = kPage * kRowB;     // a page's slice: 4 KB
constexpr int kStageB = 4 * kSliceB;       // K, K', V, V' of a page
constexpr int kWaveLds = 2 * kStageB + 16 * kRowB;   // two stages, query rows
constexpr int kWaves = 4;
constexpr int kMaxB = 8192;                // prefix table lives in LDS
constexpr int kIds = 3744;                 // page ids kept in LDS, all ranges

struct DecodeDiffArgs {
  const __bf16* q;
  const __bf16* kpool;
  const __bf16* vpool;
  const int32_t* bt;
  int64_t bt_stride;
  int bt_width;      // entries a row may be read at: min(bt_stride, 2^31-1)
  int table_wrap;
  const int32_t* ctx_lens;
  int B, HQ;
  int HKV;           // stored heads of a pool row
  int rep;           // head pairs per scheduled pair of stored heads (1..8)
  int kv_div;        // scheduled pairs per stored one
  int per_wg;        // pairs of stored heads per work-group (1, 2 or 4)
  int num_pages;     // clamped to INT32_MAX: page ids are int32
  int window;
  float scale_log2;
  int min_pages;
  DiffWeights w;
  __bf16* out;
  float* lse;
  int R;             // ranges
  float* part_o;     // [2 R, HQ, 256] fp32 (see part_slot)
  float* part_lse;   // [2 R, HQ]
  int* geo;          // [B + 2]: pages per range, then the page prefix
  int ids_off;       // LDS byte offset of the norm's weights, then the page ids
};

__device__ __forceinline__ int vis_lo(int n, int window) {
  return (window > 0 && n > window) ? n - window : 0;
}
// pages of a request of n tokens that hold a visible key and may have an entry
// in a row of `width` (a ring's pages all have one)
__device__ __forceinline__ int vis_pages(int n, int window, int width) {
  if (n <= 0) return 0;
  const int end = (int)(((uint32_t)n + kPage - 1) / kPage);
  return max(0, min(end, width) - vis_lo(n, window) / kPage);
}

__device__ __forceinline__ int page_id(const DecodeDiffArgs& a, int b, int lp) {
  const int idx = a.table_wrap > 0 ? lp % a.table_wrap : lp;
  // a logical page past the row's width has no entry: its keys are absent
  if ((unsigned)idx >= (unsigned)a.bt_width) return -1;
  const int v = as_const(a.bt)[(int64_t)b * a.bt_stride + idx];
  return (unsigned)v < (unsigned)a.num_pages ? v : -1;
}

// The arguments in the argument segment, read again where they are needed
// rarely (the pointer is opaque to the compiler), so that they hold no
// registers over the walk.
typedef const __attribute__((address_space(4))) DecodeDiffArgs* ArgsPtr;
__device__ __forceinline__ ArgsPtr rare_args() {
  auto p = (ArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// One page of the flattened page stream (wave-uniform).
struct Step {
  int b;       // request (-1: past the end of the range)
  int n;       // its context length
  int pg;      // logical page
  int flags;
};
enum : int {
  kFirst = 1,   // first step of this piece: the query rows come with it
  kLast = 2,    // last step of this piece
  kFull = 4,    // the page is there and all its tokens are visible
  kThere = 8,   // the page is there
  kWhole = 16,  // the piece is the whole request
  kCross = 32,  // the two waves of the range share the piece
  kStarts = 64, // the piece's request starts in this range
};

// Where a piece leaves its result: a range has two at most that are not whole
// requests, of the one that it goes on with and of the one that it begins. (The
// two in halves of their own: a join reads the first kind, 32 KB apart for 32
// heads; side by side, 64 KB apart, one request of 50,001 tokens took 1 us more.)
__device__ __forceinline__ int part_slot(int R, int range, bool starts) {
  return starts ? R + range : range;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Groups of waves per head pair in the merge, from the pieces of an average
// request (at most one more than its share of the R ranges). Graph replays with
// 1 / 2 / 8 groups, us a call, 32Q/4KV: one request of 50,001 tokens 49.4 /
// 38.0 / 32.3, 4 of 4K-8K 25.2 / 22.8 / 20.8, 9 up to 4.7K 24.0 / 21.7 / 20.9,
// 16 up to 2K 21.2 / 20.4 / 21.0, 24 up to 4K 32.1 / 31.5 / 34.5, 64 of 1K-8K
// 112 / 112 / 117.
__host__ __device__ __forceinline__ int merge_groups(int B, int R) {
  return 1 + R / B <= 16 ? 2 : 8;
}

// value of the lane eight columns on (within 16-lane rows): the other map's
__device__ __forceinline__ float other_map(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128,
                                         0xF, 0xF, false));   // row_ror 8
}

// One work-group per CU by its LDS, one wave per SIMD.
__global__ __launch_bounds__(64 * kWaves)
__attribute__((amdgpu_waves_per_eu(2, 2)))
void decode_diff_kernel(DecodeDiffArgs a) {
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15;  // MFMA row / column index
  const int g = lane >> 4;  // MFMA k-group
  // waves of one pair of stored heads, and how many of them share a range
  const int subs = kWaves / a.per_wg;
  const int halves = min(subs, 2);
  const int v = w / a.per_wg;
  const int half = v & (halves - 1);
  const int range = blockIdx.x * (subs / halves) + v / halves;
  const int R = gridDim.x * (subs / halves);
  const int pair = blockIdx.y * a.per_wg + w % a.per_wg;
  int* pref = reinterpret_cast<int*>(smem);  // [B + 1]
  int* wsum = pref + a.B + 1;                // [4] sums, [4] maxima
  int* nlen = wsum + 2 * kWaves;             // [B]
  const int ids_cap = kIds / subs;
  int* ids = reinterpret_cast<int*>(smem + a.ids_off) + kDV + v * (ids_cap + 2);
  const uint32_t lds_wt =
      (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)smem) +
      a.ids_off;

  // ---- 1. prefix sums of visible pages: pref[b] = first page of request b --
  const int width = a.table_wrap > 0 ? 0x7fffffff : a.bt_width;
  int most = 0;   // pages of the longest request
  {
    int carry = 0;
    int next = (int)threadIdx.x < a.B ? a.ctx_lens[threadIdx.x] : 0;
    for (int b0 = 0; b0 < a.B; b0 += 64 * kWaves) {
      const int b = b0 + threadIdx.x;
      const int nb = next;
      next = b + 64 * kWaves < a.B ? a.ctx_lens[b + 64 * kWaves] : 0;
      if (b < a.B) nlen[b] = nb;
      const int np = vis_pages(nb, a.window, width);
      most = max(most, np);
      const int x = wave_scan(np);
      if (lane == 63) wsum[w] = x;
      __syncthreads();
      int before = carry;
      for (int j = 0; j < w; ++j) before += wsum[j];
      if (b < a.B) pref[b + 1] = before + x;
      for (int j = 0; j < kWaves; ++j) carry += wsum[j];
      __syncthreads();
    }
    for (int x = 1; x < 64; x <<= 1) most = max(most, __shfl_xor(most, x));
    if (lane == 0) wsum[kWaves + w] = most;
    if (threadIdx.x == 0) pref[0] = 0;
    __syncthreads();
    for (int j = 0; j < kWaves; ++j) most = max(most, wsum[kWaves + j]);
    most = __builtin_amdgcn_readfirstlane(most);
  }
  // What the end of a piece needs is here before the walk: a load there would
  // wait for every page on its way.
  const int col_h = r & 7;                        // head pair of the column
  const bool col_ok = col_h < a.rep;
  float lam = a.w.lam[(int64_t)(pair * a.rep + min(col_h, a.rep - 1)) *
                      a.w.lam_stride];
  const bool puts_wt = a.w.weight != nullptr && threadIdx.x < kDV / 4;
  u32x4 wt{};
  if (puts_wt)
    wt = *reinterpret_cast<const u32x4*>(a.w.weight + 4 * threadIdx.x);
  const int U = __builtin_amdgcn_readfirstlane(pref[a.B]);
  int C = max((U + R - 1) / R, a.min_pages);
  // The merge takes a request's pieces in rounds of 64 (16 with two groups of
  // waves, merge_groups), about 2.5 us each, a page of both waves 0.45 us: a
  // little longer pieces where they save rounds (one request of 8000 tokens
  // 19.8 -> 17.0 us, of 50,001 as before).
  const int cap = 8 * merge_groups(a.B, R);
  if (most > (int64_t)C * cap) {
    const int r0 = ((most + C - 1) / C + cap - 1) / cap;
    int best = 11 * r0 + 2 * C;
    for (int r = min(r0 - 1, 4); r > 0; --r) {
      const int c = (most + cap * r - 1) / (cap * r);
      if (11 * r + 2 * c < best) {
        best = 11 * r + 2 * c;
        C = c;
      }
    }
  }
  // Whole requests, the same number for every range: nothing is split, nothing
  // joined. Partial results and their merge cost some 1.5 us per 1000 rows (HQ
  // of each request, of no more than there are ranges), a page above the even
  // share 0.3 where two waves walk a range, 0.75 where one does; and up to a
  // sixteenth more is within what an even share spreads. Graph replays, us,
  // evenly / whole: 32Q/4KV 192 requests of 100-300 tokens 34.3 / 24.4, 128 up
  // to 300 26.4 / 21.2, 180 of 500-800 57.8 / 50.0, 600 up to 200 61 / 45;
  // 64Q/16KV 96 of 100-300 43.7 / 37.6, 96 under a window of 512 with contexts
  // of 100-2000 73.8 / 64.3. What stays even would lose: 64 up to 300 19.9 /
  // 21.9, 64 under a window of 512 27 / 32, 64Q/16KV 32 up to 300 21 / 30.
  const int per = (a.B + R - 1) / R;
  if (per > 1) {   // the pages of the heaviest range
    most = 0;
    for (int i = threadIdx.x * per; i < a.B; i += 64 * kWaves * per)
      most = max(most, pref[min(i + per, a.B)] - pref[i]);
    for (int x = 1; x < 64; x <<= 1) most = max(most, __shfl_xor(most, x));
    __syncthreads();
    if (lane == 0) wsum[w] = most;
    __syncthreads();
    for (int j = 0; j < kWaves; ++j) most = max(most, wsum[j]);
    most = __builtin_amdgcn_readfirstlane(most);
  }
  const int slack = min(a.B, R) * a.HQ >> (halves > 1 ? 8 : 9);
  const bool whole = most <= (int64_t)C + C / 16 + 1 + slack;
  // the range [r0, r1), and this wave's pages of it: [u0, u1), backward in the
  // second half
  int r0 = (int)min((int64_t)range * C, (int64_t)U);
  int r1 = (int)min((int64_t)r0 + C, (int64_t)U);
  if (whole) {
    r0 = __builtin_amdgcn_readfirstlane(pref[min(range * per, a.B)]);
    r1 = __builtin_amdgcn_readfirstlane(pref[min((range + 1) * per, a.B)]);
    C = 0x7fffffff;
  }
  // publish the split geometry for the merge (whole requests are one piece)
  if (blockIdx.x == 0 && blockIdx.y == 0) {
    for (int i = threadIdx.x; i <= a.B; i += 64 * kWaves)
      a.geo[1 + i] = pref[i];
    if (threadIdx.x == 0) a.geo[0] = C;
  }
  const int mid = halves > 1 ? r0 + (r1 - r0 + 1) / 2 : r1;
  const int u0 = half == 0 ? r0 : mid, u1 = half == 0 ? mid : r1;
  const bool back = half != 0;
  const int rep = a.rep;
  const int hq = 2 * (pair * rep + col_h) + (r >> 3);   // query head

  // ---- 2. requests with no visible key: output 0, LSE -inf ---------------
  for (int b = range; b < a.B && half == 0; b += R) {
    if (pref[b + 1] != pref[b] || !col_ok) continue;
    __bf16* o = a.out + ((int64_t)b * (a.HQ / 2) + pair * rep + col_h) * kDV +
                (r >> 3) * kD;
#pragma unroll
    for (int blk = 0; blk < 8; ++blk)
      *reinterpret_cast<u32x2*>(o + 16 * blk + 4 * g) = u32x2{0, 0};
    if (a.lse && g == 0) a.lse[(int64_t)b * a.HQ + hq] = -INFINITY;
  }

  // ---- 3. the page stream of [u0, u1) -------------------------------------
  auto seq_of = [&](int u) {   // first request with pref[b + 1] > u
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (pref[mid + 1] > u) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  const int nids = min(u1 - u0, ids_cap);
  for (int i = threadIdx.x - 64 * a.per_wg * v; i < nids; i += 64 * a.per_wg) {
    const int b = seq_of(u0 + i);
    ids[i] = page_id(a, b, vis_lo(nlen[b], a.window) / kPage +
                               (u0 + i - pref[b]));
  }
  int cu = back ? u1 - 1 : u0;   // the next page to hand out
  int left = u1 - u0;
  int cb = __builtin_amdgcn_readfirstlane(seq_of(max(cu, 0)));
  int seq_start = __builtin_amdgcn_readfirstlane(pref[cb]);
  int cur_n = __builtin_amdgcn_readfirstlane(nlen[cb]);
  int seq_end = seq_start + vis_pages(cur_n, a.window, width);
  int pg_of = vis_lo(cur_n, a.window) / kPage - seq_start;   // page of unit u
  int last_b = -1;  // request of the previous step handed out
  if (puts_wt) lds_st128(lds_wt + 16 * threadIdx.x, wt);
  asm volatile("" : "+v"(lam));   // (has arrived: no wait for it in the walk)
  __syncthreads();  // the ids are there; every wave is done with the tables
  const uint32_t ids0 =
      (uint32_t)(uintptr_t)((__attribute__((address_space(3))) int*)ids);
  int id0 = (int)lds_ld32(ids0 + 4 * min(max(cu - u0, 0), ids_cap));
  // The next step, and the page it reads (-1: none).
  auto next_step = [&](Step& st, int& phys) __attribute__((always_inline)) {
    st.b = -1;
    st.n = st.pg = st.flags = 0;
    phys = -1;
    if (left <= 0) return;
    if (cu >= seq_end || cu < seq_start) {   // the next request with a page
      const ArgsPtr ra = rare_args();
      do {
        cb += back ? -1 : 1;
        cur_n = as_const(ra->ctx_lens)[cb];
        const int n = vis_pages(cur_n, a.window, width);
        seq_start = back ? seq_start - n : seq_end;
        seq_end = seq_start + n;
      } while (cu >= seq_end || cu < seq_start);
      pg_of = vis_lo(cur_n, a.window) / kPage - seq_start;
    }
    st.b = cb;
    st.n = cur_n;
    st.pg = cu + pg_of;
    phys = __builtin_amdgcn_readfirstlane(id0);
    if (cu - u0 >= ids_cap) phys = page_id(a, cb, st.pg);
    const bool last = cu == (back ? max(seq_start, u0) : min(seq_end, u1) - 1);
    cu += back ? -1 : 1;
    --left;
    id0 = (int)lds_ld32(ids0 + 4 * min(max(cu - u0, 0), ids_cap));
    // tokens after the page (a ring's positions may come near 2^31)
    const int past = (int)((uint32_t)st.n - (uint32_t)(st.pg + 1) * kPage);
    const bool full = phys >= 0 && past >= 0 &&
                      (a.window <= 0 || past + kPage <= a.window);
    st.flags = (cb != last_b ? kFirst : 0) | (last ? kLast : 0) |
               (full ? kFull : 0) | (phys >= 0 ? kThere : 0) |
               (seq_start >= r0 ? kStarts : 0) |
               (seq_start >= r0 && seq_end <= r1 ? kWhole : 0) |
               (mid < r1 && seq_start < mid && seq_end > mid ? kCross : 0);
    last_b = cb;
  };

  const int row_bytes = a.HKV * kRowB;
  const int kvs = 2 * (pair / a.kv_div);   // the first of the stored heads
  // Tiles in LDS: 16 token rows of 256 B per slice. K row x keeps 16-byte chunk
  // c at slot c ^ x, V row x keeps 32-byte unit u at slot u ^ (x & 7):
  // conflict-free for the K fragment reads (16 rows, one chunk) and for the
  // transposed V reads (8 rows, one unit, per 32 lanes). They arrive by direct
  // loads, 4 rows per instruction: lane l fills row l >> 4, physical slot
  // l & 15, and fetches the chunk that belongs there.
  const int wtok = lane >> 4, wslot = lane & 15;
  int koff[2][4], voff[2][4];   // byte offsets in a page of rows 4i + wtok, less
                                // the 1024 i of the instructions' own offsets
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = 4 * i + wtok;
      const int base = x * row_bytes + (kvs + m) * kRowB - 1024 * i;
      koff[m][i] = base + 16 * (wslot ^ x);
      voff[m][i] = base + 32 * ((wslot >> 1) ^ (x & 7)) + 16 * (wslot & 1);
    }
  const uint32_t lds_w =
      (uint32_t)(uintptr_t)((__attribute__((address_space(3))) char*)smem) +
      w * kWaveLds;
  const uint32_t lds_q = lds_w + 2 * kStageB;
  // K fragment (m, kk) of lane (r, g): row r, chunk 4kk + g (queries alike: row
  // = column)
  const uint32_t kr0 = lds_w + r * kRowB + 16 * (g ^ r);
  // transposed V reads: rows 4g + (s >> 2), unit blk, dims 4 (s & 3)
  const int x0 = 4 * g + (wslot >> 2);
  const uint32_t vr0 = lds_w + 2 * kSliceB + x0 * kRowB + 32 * (x0 & 7) +
                       8 * (wslot & 3);

  // ---- direct loads of one step: 8 for K, then 8 for V --------------------
  auto page_dma = [&](const __bf16* pool, const Step& st, int phys,
                      uint32_t dst, const int (&off)[2][4])
      __attribute__((always_inline)) {
    const int past = st.n - st.pg * kPage;   // tokens from the page's first on
    const int r_lo = a.window > 0 ? max(0, past - a.window) : 0;
    const int r_hi = min(kPage, past);
    const uint64_t base = (uint64_t)(uint32_t)max(phys, 0) *
                              (uint32_t)(kPage * row_bytes) +
                          (uint32_t)(r_lo * row_bytes);
    const i32x4 rs =
        make_rsrc(reinterpret_cast<const char*>(pool) + base,
                  phys >= 0 ? (uint32_t)((r_hi - r_lo) * row_bytes) : 0u);
    if (r_lo > 0) {   // the window's first page
      const int d = r_lo * row_bytes;
#pragma unroll
      for (int m = 0; m < 2; ++m)
        dma4_nt<false>(rs, dst + m * kSliceB, off[m][0] - d,
                       off[m][1] + 1024 - d, off[m][2] + 2048 - d,
                       off[m][3] + 3 * 1024 - d);
    } else {
#pragma unroll
      for (int m = 0; m < 2; ++m)
        dma4_nt<true>(rs, dst + m * kSliceB, off[m][0], off[m][1], off[m][2],
                      off[m][3]);
    }
  };
  auto issue_k = [&](const Step& st, int phys, int stage)
      __attribute__((always_inline)) {
    page_dma(a.kpool, st, phys, lds_w + stage * kStageB, koff);
  };
  auto issue_v = [&](const Step& st, int phys, int stage)
      __attribute__((always_inline)) {
    page_dma(a.vpool, st, phys, lds_w + stage * kStageB + 2 * kSliceB, voff);
  };
  // the 16 query rows of a piece, row c = column c's (columns without a head:
  // past the resource, zeros)
  auto issue_q = [&](int b) __attribute__((always_inline)) {
    const i32x4 rs =
        make_rsrc(a.q + ((int64_t)b * a.HQ + (int64_t)2 * pair * rep) * kD,
                  (uint32_t)(2 * rep * kRowB));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = 4 * i + wtok;
      dma(rs, lds_q + 1024 * i,
          (2 * (x & 7) + (x >> 3)) * kRowB + 16 * (wslot ^ x));
    }
  };
  // this wave's LDS reads are complete: what they read may be overwritten
  auto lds_done = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));   // lgkmcnt 0
    asm volatile("" ::: "memory");
  };

  // ---- per-piece state ----------------------------------------------------
  f32x4 o_acc[16];
#pragma unroll
  for (int blk = 0; blk < 16; ++blk) o_acc[blk] = f32x4{0, 0, 0, 0};
  float m_run = -INFINITY;
  float l_part = 0.0f;
  bf16x8 qf[4];   // query fragments

  // End of a piece: the result of a whole request (difference and norm
  // included), or both maps' normalised partials for the merge.
  auto finish_piece = [&](int b, int flags) {
    const float l_tot = lane_pair(lane_pair(l_part, 16, false), 32, false);
    const float inv = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
    // (a key that is no number makes the sum none: neither is the LSE)
    const float lse_nat =
        l_tot == 0.0f ? -INFINITY : (m_run + fast_log2(l_tot)) * kLn2;
    const ArgsPtr ra = rare_args();
    const int HQ = ra->HQ;
    if (flags & kWhole) {
      float ss = 0.0f;
#pragma unroll
      for (int blk = 0; blk < 16; ++blk)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = o_acc[blk][i] * inv;
          const float d = x - lam * other_map(x);   // (columns of map 0)
          o_acc[blk][i] = d;
          ss += d * d;
        }
      float f = ra->w.out_scale;
      const bool norm = ra->w.weight != nullptr;
      if (norm) {
        ss = lane_pair(lane_pair(ss, 16, false), 32, false);
        f *= __builtin_amdgcn_rsqf(ss * (1.0f / kDV) + ra->w.eps);
      }
#pragma unroll
      for (int blk = 0; blk < 16; ++blk) o_acc[blk] = o_acc[blk] * f;
      if (norm) {
#pragma unroll
        for (int blk = 0; blk < 16; ++blk)
          o_acc[blk] *= __builtin_bit_cast(f32x4,
                                           lds_ld128(lds_wt + 64 * blk + 16 * g));
      }
      if (col_ok && r < 8) {
        __bf16* const o = ra->out +
                          ((int64_t)b * (HQ / 2) + pair * rep + col_h) * kDV +
                          4 * g;
#pragma unroll
        for (int blk = 0; blk < 16; ++blk)
          *reinterpret_cast<u32x2*>(o + 16 * blk) =
              u32x2{pack_bf16x2_rn(o_acc[blk][0], o_acc[blk][1]),
                    pack_bf16x2_rn(o_acc[blk][2], o_acc[blk][3])};
      }
      float* const lse = ra->lse;
      if (lse != nullptr && col_ok && g == 0)
        lse[(int64_t)b * HQ + hq] = lse_nat;
    } else if (col_ok) {
      const int64_t slot =
          (int64_t)part_slot(ra->R, range, flags & kStarts) * HQ + hq;
      float* const o = ra->part_o + slot * kDV + 4 * g;
#pragma unroll
      for (int blk = 0; blk < 16; ++blk)
        *reinterpret_cast<f32x4*>(o + 16 * blk) = o_acc[blk] * inv;
      if (g == 0) ra->part_lse[slot] = lse_nat;
    }
#pragma unroll
    for (int blk = 0; blk < 16; ++blk) o_acc[blk] = f32x4{0, 0, 0, 0};
    m_run = -INFINITY;
    l_part = 0.0f;
  };

  // ---- 4. software-pipelined walk ------------------------------------------
  // Step s sits in stage s & 1. Its fragments are read into registers first,
  // each half of the stage then makes room for step s + 2 at once: two steps
  // (32 KB per wave) are in flight while one is computed. Queries: those of the
  // next step, if it starts a piece, go out at the top of this one.
  constexpr int kNK = 8, kNS = 16;   // loads of a step's K, and of a step
  Step cur, nx, nn;
  int phys;
  int end_b = -1, end_flags = 0;   // the piece that both waves share
  next_step(cur, phys);
  issue_q(max(cur.b, 0));
  issue_k(cur, phys, 0);
  issue_v(cur, phys, 0);
  next_step(nx, phys);
  issue_k(nx, phys, 1);
  issue_v(nx, phys, 1);
  auto read_q = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      qf[kk] = lds_ld128((kr0 ^ (64u * kk)) + 2 * kStageB);
    lds_done();
  };
  wait_vm<2 * kNS>();
  read_q();
  cur.flags &= ~kFirst;
  while (cur.b >= 0) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (k == 1 && cur.b < 0) break;
      const uint32_t so = k * kStageB;
      if (cur.flags & kFirst) {
        wait_vm<kNS>();
        read_q();
      }
      if (nx.flags & kFirst) issue_q(nx.b);
      // ---- K fragments -----------------------------------------------------
      wait_vm<kNK + kNS>();   // after K(s), in flight: V(s) and step s + 1
      asm volatile("" ::: "memory");
      bf16x8 kf[2][4];
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int m = 0; m < 2; ++m)
          kf[m][kk] = lds_ld128((kr0 ^ (64u * kk)) + so + m * kSliceB);
      next_step(nn, phys);
      lds_done();
      // ---- S^T = K.Q^T with both key heads -----------------------------------
      f32x4 sc[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int m = 0; m < 2; ++m)
          sc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[m][kk], qf[kk],
                                                          sc[m], 0, 0, 0);
      issue_k(nn, phys, k);
      // ---- V^T fragments -------------------------------------------------------
      // A operand (dims 16 blk + r, tokens 4g..4g+3) by one transposed read:
      // source lane s of each 16-lane group names token 4g + (s >> 2) and dims
      // 16 blk + 4 (s & 3)..+3
      wait_vm<kNS + kNK>();   // after V(s): step s + 1 and K(s + 2)
      asm volatile("" ::: "memory");
      bf16x4 vf[16];
#pragma unroll
      for (int blk = 0; blk < 16; ++blk)
        vf[blk] = lds_tr16((vr0 ^ (32u * (blk & 7))) + so +
                           (blk >> 3) * kSliceB);
      __builtin_amdgcn_sched_barrier(0);   // (or the reads sink to their uses)
      // ---- mask, running max -----------------------------------------------
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] = (r < 8 ? sc[0][i] : sc[1][i]) * a.scale_log2;
      if (!(cur.flags & kFull)) {
        const int lo = vis_lo(cur.n, a.window);
        const bool there = cur.flags & kThere;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kpos = cur.pg * kPage + 4 * g + i;
          x[i] = there && kpos >= lo && kpos < cur.n ? x[i] : -INFINITY;
        }
      }
      float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
      mx = lane_pair(lane_pair(mx, 16, true), 32, true);
      const bool move = mx > m_run;
      if (__builtin_amdgcn_ballot_w64(move)) {
        const float m_new = move ? mx : m_run;
        const float alpha = move ? fast_exp2(m_run - m_new) : 1.0f;
        m_run = m_new;
        l_part *= alpha;
#pragma unroll
        for (int blk = 0; blk < 16; ++blk) o_acc[blk] = o_acc[blk] * alpha;
      }
      const float m_use = m_run == -INFINITY ? 0.0f : m_run;
      // ---- probabilities: fp32 sum, bf16 operand -----------------------------
      // (B-operand element i is token 4g + i; rounded to what the matrix
      // instruction takes, each by half a step at most, while the sum that
      // divides them keeps 32 bits: against 64 bits outputs are off by 1.7e-3
      // to 1.9e-3 where fp32 probabilities give 1.7e-3)
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = fast_exp2(x[i] - m_use);
      l_part += (p[0] + p[1]) + (p[2] + p[3]);
      const s16x4 pf = __builtin_bit_cast(
          s16x4, u32x2{pack_bf16x2_rn(p[0], p[1]), pack_bf16x2_rn(p[2], p[3])});
      // ---- O^T += V^T.P^T ------------------------------------------------------
      lds_done();
#pragma unroll
      for (int blk = 0; blk < 16; ++blk)
        o_acc[blk] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
            __builtin_bit_cast(s16x4, vf[blk]), pf, o_acc[blk], 0, 0, 0);
      issue_v(nn, phys, k);
      if (cur.flags & kLast) {
        if (cur.flags & kCross) {   // (no step comes after it)
          end_b = cur.b;
          end_flags = cur.flags;
        } else {
          finish_piece(cur.b, cur.flags);
          asm volatile("" ::: "memory");   // (its stores come before any wait)
        }
      }
      cur = nx;
      nx = nn;
    }
  }
  wait_vm<0>();   // no direct load outlives the wave, or lands on what follows
  asm volatile("" ::: "memory");

  // ---- 5. the request in the middle of the range ---------------------------
  // (it has a page in both halves or in neither: all waves know; the second
  // wave's results go through its own stages)
  if (halves == 1) return;
  const uint32_t at = lds_w + (half == 0 ? a.per_wg * kWaveLds : 0) + 16 * lane;
  if (half != 0 && end_b >= 0) {
#pragma unroll
    for (int blk = 0; blk < 16; ++blk)
      lds_st128(at + 1024 * blk, __builtin_bit_cast(u32x4, o_acc[blk]));
    lds_st64(at + 16384, u32x2{__builtin_bit_cast(uint32_t, m_run),
                               __builtin_bit_cast(uint32_t, l_part)});
  }
  __syncthreads();
  if (half != 0 || end_b < 0) return;
  const float m1 = __builtin_bit_cast(float, lds_ld32(at + 16384));
  const float l1 = __builtin_bit_cast(float, lds_ld32(at + 16388));
  const float m_new = fmaxf(m_run, m1);
  const float m_use = m_new == -INFINITY ? 0.0f : m_new;
  const float f0 = fast_exp2(m_run - m_use), f1 = fast_exp2(m1 - m_use);
  l_part = l_part * f0 + l1 * f1;
  m_run = m_new;
#pragma unroll
  for (int blk = 0; blk < 16; ++blk)
    o_acc[blk] = o_acc[blk] * f0 +
                 __builtin_bit_cast(f32x4, lds_ld128(at + 1024 * blk)) * f1;
  finish_piece(end_b, end_flags);
}

// Join the pieces of every request that several ranges shared, in a fixed
// order: grid (B, HQ / 2 / H), H head pairs per work-group, for each S groups
// of two waves, one per map (4 dims per lane). Group s takes pieces s, s + S,
// ..., eight loads in flight at a time; the groups' results then merge through
// LDS in order, and the first group takes the difference and the norm.
template <int H, int S>
__global__ __launch_bounds__(128 * H * S) void decode_diff_merge(
    DecodeDiffArgs a) {
  const int b = blockIdx.x;
  const int C = as_const(a.geo)[0];
  const int s0 = as_const(a.geo)[1 + b];
  const int s1 = as_const(a.geo)[2 + b];
  if (s1 <= s0) return;                  // no visible key: written already
  const int first = s0 / C;
  const int np = (s1 - 1) / C - first + 1;
  if (np <= 1) return;                   // one piece: written in place
  __shared__ float part[H * S][2][6][64];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = w & 1, grp = w >> 1, sub = grp % S;
  const int h = blockIdx.y * H + grp / S;
  const bool hok = h < a.HQ / 2;
  const int d0 = 4 * lane;
  const int head = 2 * (hok ? h : 0) + m;
  float mx = -INFINITY, sum = 0.0f;
  f32x4 acc = f32x4{0, 0, 0, 0};
  auto add = [&](float l, float w1, f32x4 o) {   // a piece (LSE l, weight w1)
    const float m_new = fmaxf(mx, l);
    const float m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float keep = fast_exp2((mx - m_use) * kLog2e);
    const float wt = fast_exp2((l - m_use) * kLog2e);
    sum = sum * keep + wt * w1;
    acc = acc * keep + o * wt;
    mx = m_new;
  };
  constexpr int kBatch = 8;
  for (int k = sub; k < np; k += kBatch * S) {
    float l[kBatch];
    f32x4 o[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const bool in = k + j * S < np;
      const int x = in ? k + j * S : 0;
      const int64_t slot =
          (int64_t)part_slot(a.R, first + x, x == 0) * a.HQ + head;
      l[j] = in ? a.part_lse[slot] : -INFINITY;
      o[j] = *reinterpret_cast<const f32x4*>(a.part_o + slot * kDV + d0);
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j)     // (0 x infinity: weight 0 won't do)
      add(l[j], 1.0f, k + j * S < np ? o[j] : f32x4{0, 0, 0, 0});
  }
  auto put = [&]() {
    part[grp][m][0][lane] = mx;
    part[grp][m][1][lane] = sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) part[grp][m][2 + i][lane] = acc[i];
  };
  if (sub > 0) put();
  __syncthreads();
  if (sub == 0)
    for (int j = 1; j < min(np, S); ++j) {
      f32x4 o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = part[grp + j][m][2 + i][lane];
      add(part[grp + j][m][0][lane], part[grp + j][m][1][lane], o);
    }
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  acc = acc * inv;
  if (sub == 0 && hok && a.lse && lane == 0)
    a.lse[(int64_t)b * a.HQ + 2 * h + m] =
        sum == 0.0f ? -INFINITY : mx + fast_log2(sum) * kLn2;
  // the second map goes to the first one's wave
  if (sub == 0 && m == 1) put();
  __syncthreads();
  if (sub > 0 || m > 0 || !hok) return;
  const float lam = a.w.lam[(int64_t)h * a.w.lam_stride];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc[i] -= lam * part[grp][1][2 + i][lane];
    ss += acc[i] * acc[i];
  }
  acc = acc * a.w.out_scale;
  if (a.w.weight) {
    for (int x = 1; x < 64; x <<= 1) ss += __shfl_xor(ss, x);
    acc = acc * __builtin_amdgcn_rsqf(ss * (1.0f / kDV) + a.w.eps) *
          *reinterpret_cast<const f32x4*>(a.w.weight + d0);
  }
  *reinterpret_cast<u32x2*>(a.out + ((int64_t)b * (a.HQ / 2) + h) * kDV + d0) =
      u32x2{pack_bf16x2_rn(acc[0], acc[1]), pack_bf16x2_rn(acc[2], acc[3])};
}

void launch_merge(const DecodeDiffArgs& a, int R, hipStream_t st) {
  const int H = a.HQ / 2;
  if (merge_groups(a.B, R) == 2 || H > 65535)
    hipLaunchKernelGGL((decode_diff_merge<2, 2>), dim3(a.B, (H + 1) / 2),
                       dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((decode_diff_merge<1, 8>), dim3(a.B, H), dim3(1024), 0,
                       st, a);
}

// Head pairs per scheduled pair of stored heads: the whole ratio up to 8 (two
// maps each fill the 16 MFMA columns), else its largest divisor up to 8, the
// stored pair then scheduled several times (each reading its pages once).
int group_of(int ratio) {
  int rep = ratio;
  while (rep > 8 || ratio % rep != 0) --rep;
  return rep;
}

struct Shape {
  int rep, pairs, per_wg, G, R;   // R: ranges of the launch
};
// Three work-groups per four CUs, as the plain decode; four waves each, which
// take 4, 2 or 1 pairs of stored heads of 1, 1 or 2 ranges. Four pairs where
// there are requests for two thirds of their ranges, which then are likely
// whole; else two, whose ranges two waves share (graph replays, us, by two /
// four: 64Q/8KV 8 requests of 1K-8K 37.9 / 41.2, one of 50,000 46.0 / 49.8, 64
// of 100-1000 39.9 / 41.5; 64Q/16KV 32 up to 300 20.9 / 22.1, 96 up to 300 38.8
// / 37.6, 96 under a window of 512 68.5 / 64.1).
Shape shape_of(int B, int HQ, int HKV, int num_workgroups) {
  Shape s;
  s.rep = group_of(HQ / HKV);
  s.pairs = HQ / 2 / s.rep;
  auto groups = [&](int per_wg) {
    const int ny = s.pairs / per_wg;
    return std::max(1, num_workgroups > 0 ? num_workgroups
                                          : 3 * device_cus() / (4 * ny));
  };
  s.per_wg = s.pairs % 2 == 0 ? 2 : 1;
  if (s.pairs % 4 == 0 && B >= 2 * groups(4) / 3) s.per_wg = 4;
  s.G = groups(s.per_wg);
  const int subs = kWaves / s.per_wg;
  s.R = s.G * (subs > 1 ? subs / 2 : 1);
  return s;
}

size_t ws_layout(int B, int HQ, int R, size_t* off_lse, size_t* off_geo) {
  const size_t slots = 2 * (size_t)R;
  const size_t o_bytes = slots * HQ * kDV * sizeof(float);
  const size_t l_bytes = (slots * HQ * sizeof(float) + 255) & ~(size_t)255;
  const size_t g_bytes = (((size_t)B + 2) * sizeof(int) + 255) & ~(size_t)255;
  if (off_lse) *off_lse = o_bytes;
  if (off_geo) *off_geo = o_bytes + l_bytes;
  return o_bytes + l_bytes + g_bytes;
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" size_t tmopt_attn_decode_diff_workspace_size(int B, int HQ, int HKV,
                                                        int D,
                                                        int num_workgroups) {
  (void)D;
  if (B <= 0 || HQ <= 0 || HKV <= 0 || HKV % 2 != 0 || HQ % HKV != 0) return 0;
  return ws_layout(B, HQ, shape_of(B, HQ, HKV, num_workgroups).R, nullptr,
                   nullptr);
}

extern "C" int tmopt_attn_decode_diff(
    const void* q, const void* k_pool, const void* v_pool,
    const int32_t* block_table, int64_t bt_stride, int table_wrap,
    const int32_t* ctx_lens, int B, int HQ, int HKV, int D, int page_size,
    int64_t num_pages, int window, float scale, const float* lam,
    int lam_stride, const float* norm_weight, float norm_eps, float out_scale,
    int min_pages, int num_workgroups, void* out, float* lse, void* workspace,
    size_t workspace_bytes, tmopt_stream_t stream) {
  clear_error();
  if (B == 0) return TMOPT_OK;
  TMOPT_REQUIRE(B > 0, TMOPT_EINVAL, "decode_diff: B=%d", B);
  TMOPT_REQUIRE(B <= kMaxB, TMOPT_EUNSUPPORTED, "decode_diff: B=%d above %d",
                B, kMaxB);
  TMOPT_REQUIRE(q && k_pool && v_pool && out && block_table && ctx_lens,
                TMOPT_EINVAL, "decode_diff: null tensor pointer");
  const int rc = check_diff("decode_diff", HQ, HKV, D, window, scale, lam,
                            lam_stride, norm_weight, norm_eps);
  if (rc) return rc;
  TMOPT_REQUIRE(page_size == kPage, TMOPT_EUNSUPPORTED,
                "decode_diff: page_size=%d (only 16)", page_size);
  TMOPT_REQUIRE(num_pages > 0 && bt_stride > 0 && table_wrap >= 0 &&
                    (table_wrap == 0 || table_wrap <= bt_stride),
                TMOPT_EINVAL,
                "decode_diff: num_pages=%lld bt_stride=%lld table_wrap=%d",
                (long long)num_pages, (long long)bt_stride, table_wrap);
  TMOPT_REQUIRE(table_wrap == 0 ||
                    (window > 0 &&
                     (int64_t)window <= (int64_t)table_wrap * kPage),
                TMOPT_EINVAL,
                "decode_diff: window=%d outside a ring of %d pages", window,
                table_wrap);
  TMOPT_REQUIRE(min_pages > 0 && num_workgroups >= 0 &&
                    num_workgroups <= 65535,
                TMOPT_EINVAL, "decode_diff: min_pages=%d num_workgroups=%d",
                min_pages, num_workgroups);
  TMOPT_REQUIRE(((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool |
                 (uintptr_t)out) % 16 == 0,
                TMOPT_EINVAL, "decode_diff: tensors must be 16-byte aligned");
  const Shape s = shape_of(B, HQ, HKV, num_workgroups);
  const int ny = s.pairs / s.per_wg;
  TMOPT_REQUIRE(ny <= 65535, TMOPT_EUNSUPPORTED,
                "decode_diff: %d pairs of stored heads exceed the grid",
                s.pairs);
  size_t off_lse = 0, off_geo = 0;
  const size_t need = ws_layout(B, HQ, s.R, &off_lse, &off_geo);
  TMOPT_REQUIRE(workspace && workspace_bytes >= need &&
                    (uintptr_t)workspace % 16 == 0,
                TMOPT_EWORKSPACE,
                "decode_diff: workspace %zu bytes < %zu needed (or unaligned)",
                workspace_bytes, need);
  DecodeDiffArgs a;
  a.q = (const __bf16*)q;
  a.kpool = (const __bf16*)k_pool;
  a.vpool = (const __bf16*)v_pool;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.bt_width = bt_stride > 0x7fffffff ? 0x7fffffff : (int)bt_stride;
  a.table_wrap = table_wrap;
  a.ctx_lens = ctx_lens;
  a.B = B;
  a.HQ = HQ;
  a.HKV = HKV;
  a.rep = s.rep;
  a.kv_div = HQ / HKV / s.rep;
  a.per_wg = s.per_wg;
  a.num_pages = num_pages > 0x7fffffff ? 0x7fffffff : (int)num_pages;
  a.window = window;
  a.scale_log2 = scale * kLog2e;
  a.min_pages = min_pages;
  a.w = DiffWeights{lam, lam_stride, norm_weight, norm_eps, out_scale};
  a.out = (__bf16*)out;
  a.lse = lse;
  a.R = s.R;
  a.part_o = (float*)workspace;
  a.part_lse = (float*)((char*)workspace + off_lse);
  a.geo = (int*)((char*)workspace + off_geo);
  const size_t tab =
      ((2 * (size_t)B + 1 + 2 * kWaves) * sizeof(int) + 15) & ~(size_t)15;
  const size_t tiles = (size_t)kWaves * kWaveLds;
  a.ids_off = (int)(tab > tiles ? tab : tiles);
  const size_t lds = a.ids_off + (kDV + kIds + 2 * kWaves) * sizeof(int);
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(decode_diff_kernel, dim3(s.G, ny), dim3(64 * kWaves), lds,
                     st, a);
  const int rc2 = check_launch("decode_diff");
  if (rc2) return rc2;
  launch_merge(a, s.R, st);
  return check_launch("decode_diff_merge");
}
