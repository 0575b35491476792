// The page plan of a serving step, made on the GPU from the requests' lengths,
// and the release of finished requests' pages.
//
// Request i holds ceil(ctx_i / 16) pages in its row of the page table and needs
// ceil((ctx_i + new_i) / 16). With first_i the exclusive sum of the pages the
// requests before it take, its page old_i + j comes from the stack of free
// pages as free[count - 1 - first_i - j]. Token t of the step belongs to the
// request i with cu[i] <= t < cu[i + 1] (cu the exclusive sum of new), sits at
// position p = ctx_i + t - cu[i] and goes to pool row table[p / 16] * 16 +
// p % 16. A release pushes the pages back in order; entries of its rows that
// name no page (a window's that went back before) are left out.
//
// The checks decide about the whole step, so whoever writes an output needs the
// sums over all requests. Up to 1024 requests every work-group makes them for
// itself (the lengths are a few KB in the L2), holds them in LDS and writes its
// 1024 elements at a time of the block table, the slot map and the positions:
// one launch. A new page is read off the stack by whoever needs it, and its
// entry of the page table written by the work-group that fills that part of the
// block table, so no work-group waits for another. Where an output is one of
// the inputs (a graph that steps on in place), or above 1024 requests, one
// work-group makes the sums and the new pages, and a second launch the rest; a
// small step in place is one work-group's. A release needs the number of pages
// that each row names before it can place any, so it is two launches, the first
// of which counts, above 1024 table entries. Bound by latency: launches and
// dependent loads. Graph replays, us a step, where an empty kernel takes 2.1: 4
// decode rows 3.4, 64 rows 3.8, 96 rows and 2 chunks of 2048 tokens under
// tables of 4,224 pages 6.3; a release of one row of 500 pages 3.9, of 64 rows
// of up to 4,096 6.6.
#include "common.h"

namespace tmopt {
namespace {

constexpr int kPage = 16;
constexpr int kMaxRequests = 8192;      // the sums live in LDS
constexpr int kMaxRows = 1 << 18;       // one bit per table row in LDS
constexpr int kMaxTokens = 1 << 24;     // sums of a wave stay below 2^31
constexpr int kOwnSums = 1024;          // requests a fill may sum for itself
constexpr int kOwnEntries = 1024;       // entries a release may count for itself
constexpr int kPlanThreads = 1024;
constexpr int kFillThreads = 256;
constexpr int kChunk = 1024;            // elements per work-group of a fill

struct PlanArgs {
  int32_t* table;          // [S, W]
  int64_t S;
  int W;
  const int64_t* slots;    // [B], negative: padding
  const int32_t* ctx;
  const int32_t* add;      // plan: new tokens; release: NULL
  int B;
  int32_t* free;           // [F]
  int F;
  const int32_t* count_in;
  int max_tokens;
  int width;
  int32_t* block;          // [B, width]
  int32_t* seq;
  int32_t* cu;             // [B + 1]
  int64_t* slot_map;       // [max_tokens]
  int64_t* pos;
  int32_t* count_out;
  int32_t* reject;
  int32_t* gaps;           // release: [B + 1], see release_gaps_kernel
};

__device__ __forceinline__ int pages_of(int n) {
  return (int)(((uint32_t)n + kPage - 1) / kPage);
}

// last index i in [0, n) with s[i] <= x (s ascending, s[0] = 0 <= x)
template <class P>
__device__ __forceinline__ int run_of(P s, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Checks and sums of a step, by one work-group of T threads: tok / page [B + 1]
// (LDS) get the exclusive sums of the new tokens and of the pages taken (plan),
// or of a release's entries (modulo 2^32) and of the pages handed back (gaps[b]
// of row b's entries name none). Returns whether the step is accepted (the same in
// every thread); leaves its totals in tot and the stack's height in n.
template <int T>
__device__ bool step_sums(const PlanArgs& a, const int* gaps, int* tok,
                          int* page, uint32_t* seen, int64_t (&tot)[2],
                          int& n) {
  const bool release = gaps != nullptr;
  __shared__ int64_t wsum[2][T / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  n = a.count_in[0];      // (read before count_out, which may be it, is written)
  const int nwords = (int)((a.S + 31) / 32);
  for (int i = threadIdx.x; i < nwords; i += T) seen[i] = 0;
  __syncthreads();
  int bad = 0;
  tot[0] = tot[1] = 0;
  for (int b0 = 0; b0 < a.B; b0 += T) {
    const int b = b0 + threadIdx.x;
    int nt = 0, np = 0;
    if (b < a.B) {
      const int64_t slot = a.slots[b];
      const int ctx = a.ctx[b], add = release ? 0 : a.add[b];
      if (slot >= 0) {
        const int64_t end = (int64_t)ctx + add;
        const int most = release ? a.W : min(a.W, a.width);
        bool ok = slot < a.S && ctx >= 0 && add >= 0 &&
                  add <= (release ? 0 : a.max_tokens) &&
                  end <= (int64_t)most * kPage;
        if (ok) {
          const uint32_t bit = 1u << (slot & 31);
          ok = !(atomicOr(&seen[slot >> 5], bit) & bit);   // once per step
        }
        if (ok) {
          nt = release ? pages_of(ctx) : add;
          np = release ? pages_of(ctx) - gaps[b]
                       : pages_of((int)end) - pages_of(ctx);
        }
        bad |= !ok;
      }
    }
    const int st = wave_scan(nt), sp = wave_scan(np);
    if (lane == 63) {
      wsum[0][w] = st;
      wsum[1][w] = sp;
    }
    __syncthreads();
    int64_t bt = tot[0], bp = tot[1];
    for (int j = 0; j < T / 64; ++j) {
      if (j < w) {
        bt += wsum[0][j];
        bp += wsum[1][j];
      }
      tot[0] += wsum[0][j];
      tot[1] += wsum[1][j];
    }
    if (b < a.B) {      // (truncated only in a step that is refused)
      tok[b + 1] = (int)(bt + st);
      page[b + 1] = (int)(bp + sp);
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) tok[0] = page[0] = 0;
  bad |= n < 0 || n > a.F ||
         (release ? n + tot[1] > a.F
                  : tot[0] > a.max_tokens || tot[1] > n);
  return !__syncthreads_or(bad);
}

// The sums of a refused step: no tokens, no pages.
template <int T>
__device__ void no_step(const PlanArgs& a, int* tok, int* page,
                        int64_t (&tot)[2]) {
  for (int i = threadIdx.x; i <= a.B; i += T) tok[i] = page[i] = 0;
  tot[0] = tot[1] = 0;
  __syncthreads();
}

// How rows of `width` entries are cut into parts of about 1024: `per` parts per
// row, or `rows` whole rows per part.
struct Cut {
  int per, rows, parts;
};
Cut cut_rows(int B, int64_t width) {
  Cut c;
  c.per = (int)((width + kChunk - 1) / kChunk);
  c.rows = width < kChunk ? (int)(kChunk / width) : 1;
  c.parts = c.per > 1 ? B * c.per : (B + c.rows - 1) / c.rows;
  return c;
}

// A whole step of up to kOwnSums requests: c.parts parts of the block table,
// then 1024 tokens each.
template <int T>
__global__ __launch_bounds__(T) void plan_kernel(PlanArgs a, Cut c,
                                                 int parts) {
  extern __shared__ int lds[];
  int* const tok = lds;
  int* const page = tok + a.B + 1;
  int* const ctx = page + a.B + 1;    // [B] tokens held
  int* const row = ctx + a.B;         // [B] table row, -1: padding
  uint32_t* const seen = (uint32_t*)(row + a.B);
  for (int i = threadIdx.x; i < a.B; i += T) {
    const int64_t slot = a.slots[i];
    const bool real = slot >= 0 && slot < a.S;
    row[i] = real ? (int)slot : -1;
    ctx[i] = slot >= 0 ? a.ctx[i] : 0;
  }
  int64_t tot[2];
  int n;
  const bool ok = step_sums<T>(a, nullptr, tok, page, seen, tot, n);
  if (!ok) no_step<T>(a, tok, page, tot);
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < a.B; i += T) {
      a.cu[i + 1] = tok[i + 1];
      a.seq[i] = ctx[i] + (tok[i + 1] - tok[i]);
    }
    if (threadIdx.x == 0) {
      a.cu[0] = 0;
      a.count_out[0] = n - (int)tot[1];
      a.reject[0] = !ok;
    }
  }
  // page j of request i, which holds `old` already
  auto page_at = [&](int i, int j, int old) {
    return j < old ? a.table[(int64_t)row[i] * a.W + j]
                   : a.free[n - 1 - (page[i] + j - old)];
  };
  for (int part = blockIdx.x; part < parts; part += gridDim.x) {
    if (part < c.parts) {
      const int i0 = c.per > 1 ? part / c.per : part * c.rows;
      const int j0 = c.per > 1 ? (part - i0 * c.per) * kChunk : 0;
      const int rows = min(c.rows, a.B - i0);
      const int width = min(kChunk, a.width - j0);
      const bool wide = ((a.width | a.W) & 3) == 0 &&
                        (((uintptr_t)a.block | (uintptr_t)a.table) & 15) == 0;
      const int step = wide ? 4 : 1, units = width / step;   // per row
      for (int u = threadIdx.x; u < rows * units; u += T) {
        const int r = u / units, i = i0 + r, j = j0 + step * (u - r * units);
        const int old = pages_of(ctx[i]);
        const int have = ok && row[i] >= 0 ? old + page[i + 1] - page[i] : 0;
        int32_t* const src = a.table + (int64_t)max(row[i], 0) * a.W + j;
        int32_t* const out = a.block + (int64_t)i * a.width + j;
        if (wide) {     // 16 bytes at a time, except across the new pages
          i32x4 x{-1, -1, -1, -1};
          if (j + 4 <= min(old, have)) {
            x = *reinterpret_cast<const i32x4*>(src);
          } else if (j < have) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (j + e < have) {
                x[e] = page_at(i, j + e, old);
                if (j + e >= old) src[e] = x[e];
              }
          }
          *reinterpret_cast<i32x4*>(out) = x;
        } else {
          const int x = j < have ? page_at(i, j, old) : -1;
          out[0] = x;
          if (j >= old && j < have) src[0] = x;
        }
      }
    } else {
      const int t0 = (part - c.parts) * kChunk;
      for (int t = t0 + threadIdx.x; t < min(t0 + kChunk, a.max_tokens);
           t += T) {
        int64_t slot = -1, pos = 0;
        if (t < (int)tot[0]) {
          const int i = run_of(tok, a.B, t);
          const int p = ctx[i] + t - tok[i];
          const int pg = page_at(i, p / kPage, pages_of(ctx[i]));
          pos = p;
          slot = pg < 0 ? -1 : (int64_t)pg * kPage + p % kPage;
        }
        a.slot_map[t] = slot;
        a.pos[t] = pos;
      }
    }
  }
}

// ---- two launches: the sums and the new pages, then the rest ---------------

// 4 entries j .. j+3 of block-table row i holding `have` pages of table row
// `row`
__device__ __forceinline__ void fill_table(const PlanArgs& a, int i, int j,
                                           const int32_t* row, int have) {
  int32_t* const dst = a.block + (int64_t)i * a.width + j;
  const bool wide = ((a.width | a.W) & 3) == 0 &&
                    (((uintptr_t)a.block | (uintptr_t)a.table) & 15) == 0;
  if (wide) {
    i32x4 x{-1, -1, -1, -1};
    if (j < have) {
      x = *reinterpret_cast<const i32x4*>(row + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = j + e < have ? x[e] : -1;
    }
    *reinterpret_cast<i32x4*>(dst) = x;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < a.width) dst[e] = j + e < have ? row[j + e] : -1;
  }
}

// token t of a step of `total` tokens, cu their exclusive sums
template <class P>
__device__ __forceinline__ void fill_token(const PlanArgs& a, P cu, int total,
                                           int t) {
  int64_t slot = -1, pos = 0;
  if (t < total) {
    const int i = run_of(cu, a.B, t);
    const int p = a.seq[i] - cu[i + 1] + t;
    const int pg = a.table[a.slots[i] * a.W + p / kPage];
    pos = p;
    slot = pg < 0 ? -1 : (int64_t)pg * kPage + p % kPage;
  }
  a.slot_map[t] = slot;
  a.pos[t] = pos;
}

__global__ __launch_bounds__(kPlanThreads) void plan_sums_kernel(PlanArgs a) {
  extern __shared__ int lds[];
  int* const tok = lds;
  int* const page = tok + a.B + 1;
  uint32_t* const seen = (uint32_t*)(page + a.B + 1);
  int64_t tot[2];
  int n;
  const bool ok = step_sums<kPlanThreads>(a, nullptr, tok, page, seen, tot, n);
  if (!ok) no_step<kPlanThreads>(a, tok, page, tot);
  for (int i = threadIdx.x; i < a.B; i += kPlanThreads) {
    const int ctx = a.slots[i] < 0 ? 0 : a.ctx[i];
    a.cu[i + 1] = tok[i + 1];
    a.seq[i] = ctx + (tok[i + 1] - tok[i]);    // (seq may be ctx)
  }
  if (threadIdx.x == 0) {
    a.cu[0] = 0;
    a.count_out[0] = n - (int)tot[1];
    a.reject[0] = !ok;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < (int)tot[1]; p += kPlanThreads) {
    const int i = run_of(page, a.B, p);
    const int have = pages_of(a.seq[i]);
    a.table[a.slots[i] * a.W + have - (page[i + 1] - p)] = a.free[n - 1 - p];
  }
}

// the rest: work-groups [0, B * per) the block table, 1024 entries of a row
// each, the others 1024 tokens each
__global__ __launch_bounds__(kFillThreads) void plan_fill_kernel(PlanArgs a,
                                                                 int per) {
  extern __shared__ int cu[];
  const int ntab = a.B * per;
  if ((int)blockIdx.x < ntab) {
    const int i = blockIdx.x / per;
    const int64_t slot = a.slots[i];
    const int have =
        slot >= 0 && a.reject[0] == 0 ? pages_of(a.seq[i]) : 0;
    const int j = (blockIdx.x - i * per) * kChunk + 4 * threadIdx.x;
    if (j < a.width)
      fill_table(a, i, j, a.table + (slot < 0 ? 0 : slot) * a.W, have);
    return;
  }
  for (int i = threadIdx.x; i <= a.B; i += kFillThreads) cu[i] = a.cu[i];
  __syncthreads();
  const int t0 = (blockIdx.x - ntab) * kChunk + threadIdx.x;
#pragma unroll
  for (int k = 0; k < kChunk / kFillThreads; ++k) {
    const int t = t0 + k * kFillThreads;
    if (t < a.max_tokens) fill_token(a, (const int*)cu, cu[a.B], t);
  }
}

// ---- release ----------------------------------------------------------------

// entries of the page table that request b of a release names (0: none, or one
// that refuses the step)
__device__ __forceinline__ int named(const PlanArgs& a, int b) {
  const int64_t slot = a.slots[b];
  const int n = a.ctx[b];
  return slot >= 0 && slot < a.S && n >= 0 && n <= (int64_t)a.W * kPage
             ? pages_of(n)
             : 0;
}

// sum over a work-group, in every thread
__device__ __forceinline__ int group_sum(int x, int* wsum) {
  x = wave_scan(x);
  __syncthreads();      // (the last sum has been read)
  if ((threadIdx.x & 63) == 63) wsum[threadIdx.x >> 6] = x;
  __syncthreads();
  int sum = 0;
  for (int j = 0; j < (int)blockDim.x / 64; ++j) sum += wsum[j];
  return sum;
}

// The first of two launches: gaps[b] = how many entries of request b's name no
// page, by a work-group each (of 64 to 1024 threads, by the rows' width);
// gaps[B] = the stack's height, which the second launch may write over.
__global__ __launch_bounds__(kPlanThreads) void release_gaps_kernel(
    PlanArgs a) {
  __shared__ int wsum[kPlanThreads / 64];
  const int b = blockIdx.x;
  const int n = named(a, b);
  const int32_t* const row = a.table + (n > 0 ? a.slots[b] : 0) * a.W;
  int gaps = 0;
#pragma unroll 4
  for (int j = threadIdx.x; j < n; j += blockDim.x) gaps += row[j] < 0;
  gaps = group_sum(gaps, wsum);
  if (threadIdx.x == 0) {
    a.gaps[b] = gaps;
    if (b == 0) a.gaps[a.B] = a.count_in[0];
  }
}

// Pushes part [j0, end) of a row with gaps: the pages before the part are
// counted, then 'T' entries at a time go behind each other.
template <int T>
__device__ void push_with_gaps(const int32_t* row, int j0, int end,
                               int32_t* dst, int* wsum) {
  const int w = threadIdx.x >> 6;
  int before = 0;
  for (int j = threadIdx.x; j < j0; j += T) before += row[j] >= 0;
  dst += group_sum(before, wsum);
  for (int b = j0; b < end; b += T) {
    const int j = b + threadIdx.x;
    const int page = j < end ? row[j] : -1;
    const int x = wave_scan(page >= 0);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) wsum[w] = x;
    __syncthreads();
    int at = x - 1;
    for (int k = 0; k < T / 64; ++k) {
      if (k < w) at += wsum[k];
    }
    if (page >= 0) dst[at] = page;
    for (int k = 0; k < T / 64; ++k) dst += wsum[k];
  }
}

// A release in parts of 1024 entries of a row. OWN: a whole one of up to
// kOwnSums requests and kOwnEntries entries, whose work-groups each count the
// gaps; otherwise the second of two launches.
template <int T, bool OWN>
__global__ __launch_bounds__(T) void release_kernel(PlanArgs a, int per) {
  extern __shared__ int lds[];
  __shared__ int wsum[T / 64];
  int* const tok = lds;
  int* const page = tok + a.B + 1;
  uint32_t* const seen = (uint32_t*)(page + a.B + 1);
  const int* gaps = a.gaps;
  if constexpr (OWN) {
    int* const own = (int*)(seen + (a.S + 31) / 32);   // [B]
    for (int i = threadIdx.x; i < a.B; i += T) {
      own[i] = 0;
      tok[i] = named(a, i);
    }
    __syncthreads();
#pragma unroll 4
    for (int x = threadIdx.x; x < a.B * a.W; x += T) {
      const int b = x / a.W, j = x - b * a.W;
      if (j < tok[b] && a.table[a.slots[b] * a.W + j] < 0)
        atomicAdd(own + b, 1);
    }
    __syncthreads();
    gaps = own;
  }
  int64_t tot[2];
  int n;
  const bool ok = step_sums<T>(a, gaps, tok, page, seen, tot, n);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    a.count_out[0] = n + (ok ? (int)tot[1] : 0);
    a.reject[0] = !ok;
  }
  if (!ok) return;
  for (int part = blockIdx.x; part < a.B * per; part += gridDim.x) {
    const int i = part / per, j0 = (part - i * per) * kChunk;
    const int have = page[i + 1] - page[i];
    const int all = (int)((uint32_t)tok[i + 1] - (uint32_t)tok[i]);
    const int end = min(j0 + kChunk, all);
    if (have == 0 || j0 >= end) continue;
    const int32_t* const row = a.table + a.slots[i] * a.W;
    int32_t* const dst = a.free + n + page[i];
    if (have == all)
      for (int j = j0 + threadIdx.x; j < end; j += T) dst[j] = row[j];
    else
      push_with_gaps<T>(row, j0, end, dst, wsum);
  }
}

size_t plan_lds(int B, int64_t S) {
  return (size_t)(2 * (B + 1) + (S + 31) / 32) * sizeof(int);
}

int check_plan(const char* what, const void* table, int64_t S, int64_t W,
               const void* slots, const void* ctx, int B, const void* free,
               int64_t F, const void* count_in, const void* count_out,
               const void* reject) {
  TMOPT_REQUIRE(table && free && count_in && count_out && reject &&
                    (B == 0 || (slots && ctx)),
                TMOPT_EINVAL, "%s: null pointer", what);
  TMOPT_REQUIRE(B >= 0 && B <= kMaxRequests, TMOPT_EUNSUPPORTED,
                "%s: %d requests (at most %d)", what, B, kMaxRequests);
  TMOPT_REQUIRE(S > 0 && S <= kMaxRows, TMOPT_EUNSUPPORTED,
                "%s: %lld table rows (1 to %d)", what, (long long)S, kMaxRows);
  TMOPT_REQUIRE(W > 0 && W <= kMaxTokens && F > 0 && F <= 0x7fffffff,
                TMOPT_EUNSUPPORTED, "%s: rows of %lld pages, %lld free pages",
                what, (long long)W, (long long)F);
  return TMOPT_OK;
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" int tmopt_plan_pages(
    int32_t* page_table, int64_t table_rows, int64_t table_width,
    const int64_t* slots, const int32_t* ctx_lens, const int32_t* new_lens,
    int B, const int32_t* free_pages, int64_t free_capacity,
    const int32_t* free_count, int64_t max_tokens, int64_t width,
    int32_t* block_table, int32_t* seq_lens, int32_t* cu_seqlens,
    int64_t* slot_mapping, int64_t* positions, int32_t* free_count_out,
    int32_t* reject, tmopt_stream_t stream) {
  clear_error();
  const int rc = check_plan("plan_pages", page_table, table_rows, table_width,
                            slots, ctx_lens, B, free_pages, free_capacity,
                            free_count, free_count_out, reject);
  if (rc) return rc;
  TMOPT_REQUIRE(max_tokens >= 0 && max_tokens <= kMaxTokens && width > 0 &&
                    width <= kMaxTokens,
                TMOPT_EUNSUPPORTED, "plan_pages: max_tokens=%lld width=%lld",
                (long long)max_tokens, (long long)width);
  TMOPT_REQUIRE(cu_seqlens && (B == 0 || (new_lens && block_table && seq_lens)) &&
                    (max_tokens == 0 || (slot_mapping && positions)),
                TMOPT_EINVAL, "plan_pages: null pointer");
  const int64_t per = (width + kChunk - 1) / kChunk;
  const int64_t tokens = (max_tokens + kChunk - 1) / kChunk;
  TMOPT_REQUIRE(B * per + tokens < 0x7fffffff, TMOPT_EUNSUPPORTED,
                "plan_pages: %lld work-groups exceed the grid limit",
                (long long)(B * per + tokens));
  PlanArgs a{};
  a.table = page_table;
  a.S = table_rows;
  a.W = (int)table_width;
  a.slots = slots;
  a.ctx = ctx_lens;
  a.add = new_lens;
  a.B = B;
  a.free = const_cast<int32_t*>(free_pages);
  a.F = (int)free_capacity;
  a.count_in = free_count;
  a.max_tokens = (int)max_tokens;
  a.width = (int)width;
  a.block = block_table;
  a.seq = seq_lens;
  a.cu = cu_seqlens;
  a.slot_map = slot_mapping;
  a.pos = positions;
  a.count_out = free_count_out;
  a.reject = reject;
  const hipStream_t st = (hipStream_t)stream;
  const bool in_place = seq_lens == ctx_lens || free_count_out == free_count;
  // Small enough for one work-group (graph replays, us a step, by one / by two
  // launches: 4 requests of 64 pages 4.4 / 5.6, 32 of 512 6.5 / 5.9, 2 of 2048
  // new tokens 6.2 / 7.3, of 4096 8.2 / 7.3).
  const bool small = B * width <= 16384 && max_tokens <= 4096;
  if (B <= kOwnSums && (small || !in_place)) {
    const size_t lds = plan_lds(B, table_rows) + 2 * (size_t)B * sizeof(int);
    const Cut c = cut_rows(B, width);
    const int parts = c.parts + (int)tokens;
    if (in_place)
      hipLaunchKernelGGL((plan_kernel<kPlanThreads>), dim3(1),
                         dim3(kPlanThreads), lds, st, a, c, parts);
    else
      hipLaunchKernelGGL((plan_kernel<kFillThreads>),
                         dim3((unsigned)(parts > 0 ? parts : 1)),
                         dim3(kFillThreads), lds, st, a, c, parts);
    return check_launch("plan_pages");
  }
  const int64_t groups = B * per + tokens;
  hipLaunchKernelGGL(plan_sums_kernel, dim3(1), dim3(kPlanThreads),
                     plan_lds(B, table_rows), st, a);
  const int rc2 = check_launch("plan_pages");
  if (rc2 || groups == 0) return rc2;
  hipLaunchKernelGGL(plan_fill_kernel, dim3((unsigned)groups),
                     dim3(kFillThreads), (B + 1) * sizeof(int), st, a,
                     (int)per);
  return check_launch("plan_pages");
}

extern "C" size_t tmopt_release_pages_workspace_size(int B) {
  return B > 0 ? (((size_t)B + 1) * sizeof(int32_t) + 15) & ~(size_t)15 : 0;
}

extern "C" int tmopt_release_pages(
    const int32_t* page_table, int64_t table_rows, int64_t table_width,
    const int64_t* slots, const int32_t* lens, int B, int32_t* free_pages,
    int64_t free_capacity, const int32_t* free_count, int32_t* free_count_out,
    int32_t* reject, void* workspace, size_t workspace_bytes,
    tmopt_stream_t stream) {
  clear_error();
  const int rc = check_plan("release_pages", page_table, table_rows,
                            table_width, slots, lens, B, free_pages,
                            free_capacity, free_count, free_count_out, reject);
  if (rc) return rc;
  const size_t need = tmopt_release_pages_workspace_size(B);
  TMOPT_REQUIRE(B == 0 || (workspace && workspace_bytes >= need &&
                           (uintptr_t)workspace % 16 == 0),
                TMOPT_EWORKSPACE,
                "release_pages: workspace %zu bytes < %zu needed (or unaligned)",
                workspace_bytes, need);
  const int64_t per = (table_width + kChunk - 1) / kChunk;
  TMOPT_REQUIRE(B * per < 0x7fffffff, TMOPT_EUNSUPPORTED,
                "release_pages: %lld work-groups exceed the grid limit",
                (long long)(B * per));
  PlanArgs a{};
  a.table = const_cast<int32_t*>(page_table);
  a.S = table_rows;
  a.W = (int)table_width;
  a.slots = slots;
  a.ctx = lens;
  a.B = B;
  a.free = free_pages;
  a.F = (int)free_capacity;
  a.count_in = free_count;
  a.count_out = free_count_out;
  a.reject = reject;
  a.gaps = (int32_t*)workspace;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t parts = B * per > 0 ? B * per : 1;
  if (B <= kOwnSums && B * table_width <= kOwnEntries) {
    // (one work-group where the height is written over; one launch of 8 rows of
    // 1024 pages takes 15.7 us where two take 6.6, one row of 4096 10.2 / 6.5)
    const size_t lds = plan_lds(B, table_rows) + (size_t)B * sizeof(int);
    if (free_count_out == free_count)
      hipLaunchKernelGGL((release_kernel<kPlanThreads, true>), dim3(1),
                         dim3(kPlanThreads), lds, st, a, (int)per);
    else
      hipLaunchKernelGGL((release_kernel<kFillThreads, true>),
                         dim3((unsigned)parts), dim3(kFillThreads), lds, st, a,
                         (int)per);
    return check_launch("release_pages");
  }
  const int threads = table_width <= 256    ? 64
                      : table_width <= 2048 ? kFillThreads
                                            : kPlanThreads;
  hipLaunchKernelGGL(release_gaps_kernel, dim3(B), dim3(threads), 0, st, a);
  const int rc2 = check_launch("release_pages");
  if (rc2) return rc2;
  a.count_in = a.gaps + B;
  // above kOwnSums the sums weigh most: no more work-groups than there are
  // compute units (4096 rows of up to 64 pages: 256 work-groups 19.5 us in a
  // graph, 128 24.7, 512 26.8)
  const int64_t most = B <= kOwnSums ? 1024 : 256;
  const unsigned groups = (unsigned)(parts < most ? parts : most);
  const size_t lds = plan_lds(B, table_rows);
  if (B <= kOwnSums)
    hipLaunchKernelGGL((release_kernel<kFillThreads, false>), dim3(groups),
                       dim3(kFillThreads), lds, st, a, (int)per);
  else
    hipLaunchKernelGGL((release_kernel<kPlanThreads, false>), dim3(groups),
                       dim3(kPlanThreads), lds, st, a, (int)per);
  return check_launch("release_pages");
}
