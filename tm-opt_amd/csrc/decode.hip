// C entry points of the paged decode (kernels: decode_kernel.h).
#include <mutex>

#include "decode_kernel.h"

namespace tmopt {
namespace {

template <int REP, int KIND>
void launch_kind(const DecodeArgs& a, dim3 grid, int nw, size_t lds,
                 hipStream_t st) {
  if (a.rel)
    hipLaunchKernelGGL((decode_kernel<REP, true, KIND>), grid,
                       dim3(64 * nw), lds, st, a);
  else
    hipLaunchKernelGGL((decode_kernel<REP, false, KIND>), grid,
                       dim3(64 * nw), lds, st, a);
}

template <int REP>
void launch(const DecodeArgs& a, int G, int nw, size_t lds, hipStream_t st) {
  const dim3 grid(G, a.HKV / nw);
  if (a.bt_kind == 2) launch_kind<REP, 2>(a, grid, nw, lds, st);
  else if (a.bt_kind == 1) launch_kind<REP, 1>(a, grid, nw, lds, st);
  else launch_kind<REP, 0>(a, grid, nw, lds, st);
}

// ---- static scratch of the allocation-free entry point -------------------
// Device memory for tmopt_attn_decode_paged_noalloc's workspace: a fixed
// array in the library's code object, so the call needs no allocation.
// Every GPU the library runs on holds its own copy until the process ends.
constexpr size_t kScratchBytes = size_t(16) << 20;   // 16 MiB per GPU
static __device__ __align__(256) char scratch[kScratchBytes];

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch_addr[kMaxDevices] = {};

// Device address of the current device's copy of `scratch`. The array's
// name is a host-side stand-in in host code, never a device address: it is
// resolved here, once per device with that device current, and only the
// resolved address is passed to kernels.
int scratch_address(void** addr) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  TMOPT_REQUIRE(e == hipSuccess && dev >= 0 && dev < kMaxDevices,
                TMOPT_ELAUNCH, "decode_noalloc: no current device (%s)",
                hipGetErrorString(e));
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (g_scratch_addr[dev] == nullptr) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    TMOPT_REQUIRE(e == hipSuccess && p != nullptr, TMOPT_ELAUNCH,
                  "decode_noalloc: hipGetSymbolAddress failed on device %d: "
                  "%s", dev, hipGetErrorString(e));
    g_scratch_addr[dev] = p;
  }
  *addr = g_scratch_addr[dev];
  return TMOPT_OK;
}

// The block table of attn_global's per-token rows (model.py:938-945: flat
// [b, j] = table[b][j / 16] * 16 + j % 16 for live j, 0 past the length):
// table[b][i] = flat[b][16 i] / 16, and ctx_lens[b] = pos[b] + 1. One thread
// per table entry (entries of pages past a row's length are 0, never read).
__global__ __launch_bounds__(256) void table_from_flat_kernel(
    const int64_t* __restrict__ flat, int64_t Lg, const int64_t* __restrict__ pos,
    int npages, int32_t* __restrict__ table, int64_t table_stride,
    int32_t* __restrict__ ctx_lens) {
  const int b = blockIdx.y;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < npages)
    table[(int64_t)b * table_stride + i] =
        (int32_t)(flat[(int64_t)b * Lg + (int64_t)kPS * i] / kPS);
  if (i == 0) ctx_lens[b] = (int32_t)(pos[b] + 1);
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" int tmopt_attn_decode_default_workgroups(int HKV) {
  if (HKV <= 0) return 0;
  return default_wgs(HKV);
}

extern "C" size_t tmopt_attn_decode_workspace_size(int B, int HQ, int HKV,
                                                   int D, int num_workgroups) {
  (void)D;
  if (B <= 0 || HQ <= 0 || HKV <= 0) return 0;
  const int G = num_workgroups > 0 ? num_workgroups : default_wgs(HKV);
  return ws_layout(B, HQ, G, nullptr, nullptr);
}

// The decode launch behind the entry points: `kind` 0 = int32 block table
// + int32 lengths (block_table, ctx_lens), 1 = per-token flat rows + int64
// positions (rows64, pos64), 2 = ring slots + int64 positions. (Flat rows,
// one page id per 128 bytes, cost nothing over a table since a range's ids
// are fetched at once: looked up step by step they measured 17% slower, and a
// launch that makes a table of them first takes 4.8 us: 60.1 against 58.1 us
// per call at 16 sequences of 1K-8K, 64Q/8KV.)
static int decode_impl(
    int kind, const void* q, const void* k_pool, const void* v_pool,
    const int32_t* block_table, const int64_t* rows64, int64_t bt_stride,
    int table_wrap, const int32_t* ctx_lens, const int64_t* pos64, int B,
    int HQ, int HKV, int D, int page_size, int64_t num_pages, int window,
    float scale, const void* rel, int rel_extent, int min_pages,
    int num_workgroups, int seqs_per_wg, void* out, float* lse,
    void* workspace, size_t workspace_bytes, tmopt_stream_t stream) {
  if (B == 0) return TMOPT_OK;
  TMOPT_REQUIRE(B > 0, TMOPT_EINVAL, "decode: B=%d", B);
  TMOPT_REQUIRE(B <= kMaxB, TMOPT_EUNSUPPORTED, "decode: B=%d above %d", B,
                kMaxB);
  TMOPT_REQUIRE(q && k_pool && v_pool && out &&
                    (kind == 0 ? block_table && ctx_lens : rows64 && pos64),
                TMOPT_EINVAL, "decode: null tensor pointer");
  TMOPT_REQUIRE(D == kD, TMOPT_EUNSUPPORTED, "decode: D=%d (only 128)", D);
  TMOPT_REQUIRE(page_size == kPS, TMOPT_EUNSUPPORTED,
                "decode: page_size=%d (only 16)", page_size);
  TMOPT_REQUIRE(HKV > 0 && HQ > 0 && HQ % HKV == 0, TMOPT_EINVAL,
                "decode: HQ=%d HKV=%d", HQ, HKV);
  // Query heads per scheduled KV head: the whole ratio up to 16 (the MFMA
  // columns), else its largest divisor up to 16, the stored head then
  // scheduled kv_div times (each reading its pages once per group).
  const int ratio = HQ / HKV;
  int rep = ratio;
  while (rep > 16 || ratio % rep != 0) --rep;
  const int kv_div = ratio / rep;
  TMOPT_REQUIRE((int64_t)HKV * kv_div <= 65535, TMOPT_EUNSUPPORTED,
                "decode: HKV=%d x %d query-head groups exceeds 65535", HKV,
                kv_div);
  TMOPT_REQUIRE((int64_t)kPS * HKV * kD * 2 < (1ll << 31), TMOPT_EUNSUPPORTED,
                "decode: page too large");
  TMOPT_REQUIRE(num_pages > 0 && bt_stride > 0 && table_wrap >= 0 &&
                    (table_wrap == 0 || table_wrap <= bt_stride),
                TMOPT_EINVAL,
                "decode: num_pages=%lld bt_stride=%lld table_wrap=%d",
                (long long)num_pages, (long long)bt_stride, table_wrap);
  TMOPT_REQUIRE(window >= 0, TMOPT_EINVAL, "decode: window=%d", window);
  // a ring table holds the last table_wrap * 16 positions: a wider (or no)
  // window would read rows the ring has already overwritten
  TMOPT_REQUIRE(table_wrap == 0 ||
                    (window > 0 && (int64_t)window <= (int64_t)table_wrap * kPS),
                TMOPT_EINVAL, "decode: window=%d outside a ring of %d pages",
                window, table_wrap);
  TMOPT_REQUIRE(min_pages > 0 && num_workgroups >= 0, TMOPT_EINVAL,
                "decode: min_pages=%d num_workgroups=%d", min_pages,
                num_workgroups);
  TMOPT_REQUIRE(rel == nullptr || rel_extent > 0, TMOPT_EINVAL,
                "decode: rel_extent=%d", rel_extent);
  TMOPT_REQUIRE(((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool |
                 (uintptr_t)out) % 16 == 0,
                TMOPT_EINVAL, "decode: tensors must be 16-byte aligned");
  const int G = num_workgroups > 0 ? num_workgroups : default_wgs(HKV);
  TMOPT_REQUIRE(G <= 65535, TMOPT_EINVAL, "decode: num_workgroups=%d", G);
  TMOPT_REQUIRE(seqs_per_wg >= 0 &&
                    (seqs_per_wg == 0 || (int64_t)seqs_per_wg * G >= B),
                TMOPT_EINVAL,
                "decode: %d work-groups of %d whole sequences do not cover "
                "B=%d",
                G, seqs_per_wg, B);
  size_t off_lse = 0, off_geo = 0;
  const size_t need = ws_layout(B, HQ, G, &off_lse, &off_geo);
  TMOPT_REQUIRE(workspace && workspace_bytes >= need &&
                    (uintptr_t)workspace % 16 == 0,
                TMOPT_EWORKSPACE,
                "decode: workspace %zu bytes < %zu needed (or unaligned)",
                workspace_bytes, need);

  DecodeArgs a;
  a.q = (const __bf16*)q;
  a.kpool = (const __bf16*)k_pool;
  a.vpool = (const __bf16*)v_pool;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  const int64_t width = kind == 1 ? (bt_stride + kPS - 1) / kPS : bt_stride;
  a.bt_width = width > 0x7fffffff ? 0x7fffffff : (int)width;
  a.table_wrap = table_wrap;
  a.ctx_lens = ctx_lens;
  a.bt_kind = kind;
  a.rows64 = rows64;
  a.pos64 = pos64;
  a.B = B;
  a.HQ = HQ;
  a.HKV = HKV * kv_div;
  a.rep = rep;
  a.kv_div = kv_div;
  a.HKV_stored = HKV;
  a.num_pages = num_pages > 0x7fffffff ? 0x7fffffff : (int)num_pages;
  a.window = window;
  a.scale_log2 = scale * kLog2e;
  a.rel = (const __bf16*)rel;
  a.rel_extent = rel ? rel_extent : 0;
  // (a work-group's first page, its index times this, stays within int32)
  a.min_pages = min_pages < 32768 ? min_pages : 32768;
  a.seqs_per_wg = seqs_per_wg;
  a.out = (__bf16*)out;
  a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_lse = (float*)((char*)workspace + off_lse);
  a.geo = (int*)((char*)workspace + off_geo);

  const int nw = waves_per_wg(a.HKV);
  const size_t tab = ((2 * (size_t)B + 1 + 4) * sizeof(int) + 15) & ~(size_t)15;
  const size_t tiles = (size_t)nw * wave_lds(rel != nullptr);
  a.ids_off = (int)(tab > tiles ? tab : tiles);
  const size_t lds = a.ids_off + (ids_kept(rel != nullptr) + 2) * sizeof(int);
  hipStream_t st = (hipStream_t)stream;
  switch (kv_div == 1 ? rep : 0) {
    case 1: launch<1>(a, G, nw, lds, st); break;
    case 2: launch<2>(a, G, nw, lds, st); break;
    case 4: launch<4>(a, G, nw, lds, st); break;
    case 8: launch<8>(a, G, nw, lds, st); break;
    case 16: launch<16>(a, G, nw, lds, st); break;
    default: launch<0>(a, G, nw, lds, st); break;
  }
  int rc = check_launch("decode");
  if (rc || seqs_per_wg > 0) return rc;   // whole sequences: nothing to merge
  launch_combine(a, G, st);
  return check_launch("decode_combine");
}

extern "C" int tmopt_attn_decode_paged(
    const void* q, const void* k_pool, const void* v_pool,
    const int32_t* block_table, int64_t bt_stride, int table_wrap,
    const int32_t* ctx_lens, int B, int HQ, int HKV, int D, int page_size,
    int64_t num_pages, int window, float scale, const void* rel,
    int rel_extent, int min_pages, int num_workgroups, void* out, float* lse,
    void* workspace, size_t workspace_bytes, tmopt_stream_t stream) {
  clear_error();
  return decode_impl(0, q, k_pool, v_pool, block_table, nullptr, bt_stride,
                     table_wrap, ctx_lens, nullptr, B, HQ, HKV, D, page_size,
                     num_pages, window, scale, rel, rel_extent, min_pages,
                     num_workgroups, 0, out, lse, workspace, workspace_bytes,
                     stream);
}

extern "C" int tmopt_attn_decode_ring(
    const void* q, const void* k_pool, const void* v_pool,
    const int64_t* slots, int ring_pages, const int64_t* pos, int B, int HQ,
    int HKV, int D, int64_t num_pages, int window, float scale,
    const void* rel, int rel_extent, int min_pages, int num_workgroups,
    int seqs_per_workgroup, void* out, float* lse, void* workspace,
    size_t workspace_bytes, tmopt_stream_t stream) {
  clear_error();
  TMOPT_REQUIRE(ring_pages > 0, TMOPT_EINVAL, "decode_ring: ring_pages=%d",
                ring_pages);
  return decode_impl(2, q, k_pool, v_pool, nullptr, slots, ring_pages,
                     ring_pages, nullptr, pos, B, HQ, HKV, D, kPS, num_pages,
                     window, scale, rel, rel_extent, min_pages,
                     num_workgroups, seqs_per_workgroup, out, lse, workspace,
                     workspace_bytes, stream);
}

extern "C" int tmopt_attn_decode_flat(
    const void* q, const void* k_pool, const void* v_pool,
    const int64_t* flat, int64_t Lg, const int64_t* pos, int B, int HQ,
    int HKV, int D, int page_size, int64_t num_pages, float scale,
    const void* rel, int rel_extent, int min_pages, int num_workgroups,
    void* out, float* lse, void* workspace, size_t workspace_bytes,
    tmopt_stream_t stream) {
  clear_error();
  return decode_impl(1, q, k_pool, v_pool, nullptr, flat, Lg, 0, nullptr, pos,
                     B, HQ, HKV, D, page_size, num_pages, 0, scale, rel,
                     rel_extent, min_pages, num_workgroups, 0, out, lse,
                     workspace, workspace_bytes, stream);
}

extern "C" int tmopt_attn_decode_paged_noalloc(
    const void* q, const void* k_pool, const void* v_pool,
    const int32_t* block_table, int64_t bt_stride, int table_wrap,
    const int32_t* ctx_lens, int B, int HQ, int HKV, int D, int page_size,
    int64_t num_pages, int window, float scale, const void* rel,
    int rel_extent, int min_pages, int num_workgroups, void* out, float* lse,
    tmopt_stream_t stream) {
  clear_error();
  if (B == 0) return TMOPT_OK;
  // the workspace this launch shape needs (0 for arguments the full entry
  // point rejects: it reports them)
  const size_t need =
      tmopt_attn_decode_workspace_size(B, HQ, HKV, D, num_workgroups);
  TMOPT_REQUIRE(need <= kScratchBytes, TMOPT_EWORKSPACE,
                "decode_noalloc: the launch needs %zu bytes of scratch, above "
                "the %zu-byte static buffer (use tmopt_attn_decode_paged with "
                "a workspace)",
                need, kScratchBytes);
  void* ws = nullptr;
  const int rc = scratch_address(&ws);
  if (rc != TMOPT_OK) return rc;
  return tmopt_attn_decode_paged(q, k_pool, v_pool, block_table, bt_stride,
                                 table_wrap, ctx_lens, B, HQ, HKV, D,
                                 page_size, num_pages, window, scale, rel,
                                 rel_extent, min_pages, num_workgroups, out,
                                 lse, ws, kScratchBytes, stream);
}

extern "C" int tmopt_decode_table_from_flat(const int64_t* flat, int64_t Lg,
                                            const int64_t* pos, int B,
                                            int32_t* block_table,
                                            int64_t bt_stride,
                                            int32_t* ctx_lens,
                                            tmopt_stream_t stream) {
  clear_error();
  if (B == 0) return TMOPT_OK;
  TMOPT_REQUIRE(B > 0 && B <= 65535 && Lg > 0, TMOPT_EINVAL,
                "table_from_flat: B=%d Lg=%lld", B, (long long)Lg);
  TMOPT_REQUIRE(flat && pos && block_table && ctx_lens, TMOPT_EINVAL,
                "table_from_flat: null pointer");
  const int64_t npages = (Lg + kPS - 1) / kPS;
  TMOPT_REQUIRE(npages <= 0x7fffffff && bt_stride >= npages, TMOPT_EINVAL,
                "table_from_flat: bt_stride=%lld < %lld pages",
                (long long)bt_stride, (long long)npages);
  hipLaunchKernelGGL(table_from_flat_kernel,
                     dim3((unsigned)((npages + 255) / 256), B), dim3(256), 0,
                     (hipStream_t)stream, flat, Lg, pos, (int)npages,
                     block_table, bt_stride, ctx_lens);
  return check_launch("table_from_flat");
}
