// The page plan of a serving step, made on the GPU from the requests' lengths,
// and the release of finished requests' pages.
//
// Request i holds ceil(ctx_i / 16) pages in its row of the page table and needs
// ceil((ctx_i + new_i) / 16). With first_i the exclusive sum of the pages the
// requests before it take, its page old_i + j comes from the stack of free
// pages as free[count - 1 - first_i - j]. Token t of the step belongs to the
// request i with cu[i] <= t < cu[i + 1] (cu the exclusive sum of new), sits at
// position p = ctx_i + t - cu[i] and goes to pool row table[p / 16] * 16 +
// p % 16. A release pushes the pages back in order.
//
// One work-group checks the step and makes the sums and the new pages (the
// checks decide about the whole step, and a few thousand lengths are a few
// microseconds' work of one compute unit); then every element of the block
// table, the slot map and the positions is independent, and as many work-groups
// as there are of 1024 elements write them. Small steps stay in the first
// work-group, one launch. Bound by latency: launches and dependent loads.
#include "common.h"

namespace tmopt {
namespace {

constexpr int kPage = 16;
constexpr int kMaxRequests = 8192;      // the sums live in LDS
constexpr int kMaxRows = 1 << 18;       // one bit per table row in LDS
constexpr int kMaxTokens = 1 << 24;     // sums of a wave stay below 2^31
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
  int32_t* first;          // release: [B] stack index of each row's first page
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

// Checks and sums of a step, by one work-group: tok / page [B + 1] (LDS) get
// the exclusive sums of the new tokens and of the pages taken (plan) or handed
// back (release). Returns whether the step is accepted (the same in every
// thread); leaves its totals in tot and the stack's height in n.
__device__ bool step_sums(const PlanArgs& a, bool release, int* tok, int* page,
                          uint32_t* seen, int64_t (&tot)[2], int& n) {
  __shared__ int64_t wsum[2][kPlanThreads / 64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nwords = (int)((a.S + 31) / 32);
  for (int i = threadIdx.x; i < nwords; i += kPlanThreads) seen[i] = 0;
  __syncthreads();
  int bad = 0;
  tot[0] = tot[1] = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    int nt = 0, np = 0;
    if (b < a.B) {
      const int64_t slot = a.slots[b];
      if (slot >= 0) {
        const int ctx = a.ctx[b], add = release ? 0 : a.add[b];
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
          nt = add;
          np = release ? pages_of(ctx) : pages_of((int)end) - pages_of(ctx);
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
    for (int j = 0; j < kPlanThreads / 64; ++j) {
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
  n = a.count_in[0];      // (read before count_out, which may be it, is written)
  bad |= n < 0 || n > a.F || tot[0] > (release ? 0 : a.max_tokens) ||
         (release ? n + tot[1] > a.F : tot[1] > n);
  return !__syncthreads_or(bad);
}

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

// one work-group: the checks, the sums, the new pages; `whole`: and the rest
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanArgs a,
                                                            int whole) {
  extern __shared__ int lds[];
  int* const tok = lds;
  int* const page = tok + a.B + 1;
  uint32_t* const seen = (uint32_t*)(page + a.B + 1);
  int64_t tot[2];
  int n;
  const bool ok = step_sums(a, false, tok, page, seen, tot, n);
  if (!ok) {
    for (int i = threadIdx.x; i <= a.B; i += kPlanThreads) tok[i] = 0;
    tot[0] = tot[1] = 0;
    __syncthreads();
  }
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
  if (!whole) return;
  __syncthreads();
  const int per = (a.width + 3) / 4;
  for (int x = threadIdx.x; x < a.B * per; x += kPlanThreads) {
    const int i = x / per;
    const int64_t slot = a.slots[i];
    fill_table(a, i, 4 * (x - i * per), a.table + (slot < 0 ? 0 : slot) * a.W,
               ok && slot >= 0 ? pages_of(a.seq[i]) : 0);
  }
  for (int t = threadIdx.x; t < a.max_tokens; t += kPlanThreads)
    fill_token(a, (const int*)tok, (int)tot[0], t);
}

// the rest of a large step: work-groups [0, B * per) the block table, 1024
// entries of a row each, the others 1024 tokens each
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

__global__ __launch_bounds__(kPlanThreads) void release_kernel(PlanArgs a,
                                                               int whole) {
  extern __shared__ int lds[];
  int* const tok = lds;
  int* const page = tok + a.B + 1;
  uint32_t* const seen = (uint32_t*)(page + a.B + 1);
  int64_t tot[2];
  int n;
  const bool ok = step_sums(a, true, tok, page, seen, tot, n);
  if (threadIdx.x == 0) {
    a.count_out[0] = n + (ok ? (int)tot[1] : 0);
    a.reject[0] = !ok;
  }
  if (whole) {
    for (int p = threadIdx.x; ok && p < (int)tot[1]; p += kPlanThreads) {
      const int i = run_of(page, a.B, p);
      a.free[n + p] = a.table[a.slots[i] * a.W + p - page[i]];
    }
  } else {
    for (int i = threadIdx.x; i < a.B; i += kPlanThreads)
      a.first[i] = n + page[i];
  }
}

// rows' pages of a large release: 1024 entries of a row per work-group
__global__ __launch_bounds__(kFillThreads) void release_fill_kernel(PlanArgs a,
                                                                    int per) {
  const int i = blockIdx.x / per;
  const int j0 = (blockIdx.x - i * per) * kChunk + threadIdx.x;
  const int64_t slot = a.slots[i];
  if (slot < 0 || a.reject[0] != 0) return;
  const int have = pages_of(a.ctx[i]);
  const int32_t* const row = a.table + slot * a.W;
  int32_t* const dst = a.free + a.first[i];
#pragma unroll
  for (int k = 0; k < kChunk / kFillThreads; ++k) {
    const int j = j0 + k * kFillThreads;
    if (j < have) dst[j] = row[j];
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
  const int64_t groups = B * per + (max_tokens + kChunk - 1) / kChunk;
  TMOPT_REQUIRE(groups < 0x7fffffff, TMOPT_EUNSUPPORTED,
                "plan_pages: %lld work-groups exceed the grid limit",
                (long long)groups);
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
  const bool whole = B * width <= 16384 && max_tokens <= 4096;
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kPlanThreads),
                     plan_lds(B, table_rows), st, a, (int)whole);
  const int rc2 = check_launch("plan_pages");
  if (rc2 || whole) return rc2;
  hipLaunchKernelGGL(plan_fill_kernel, dim3((unsigned)groups),
                     dim3(kFillThreads), (B + 1) * sizeof(int), st, a,
                     (int)per);
  return check_launch("plan_pages");
}

extern "C" size_t tmopt_release_pages_workspace_size(int B) {
  return B > 0 ? ((size_t)B * sizeof(int32_t) + 15) & ~(size_t)15 : 0;
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
  a.first = (int32_t*)workspace;
  const hipStream_t st = (hipStream_t)stream;
  const bool whole = B * table_width <= 16384;
  hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kPlanThreads),
                     plan_lds(B, table_rows), st, a, (int)whole);
  const int rc2 = check_launch("release_pages");
  if (rc2 || whole) return rc2;
  hipLaunchKernelGGL(release_fill_kernel, dim3((unsigned)(B * per)),
                     dim3(kFillThreads), 0, st, a, (int)per);
  return check_launch("release_pages");
}
