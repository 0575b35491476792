// C entry point of the scored paged decode: score functions and first keys over
// the bf16 cache (kernels: decode_kernel.h).
#define TMOPT_DECODE_SCORED
#include "decode_kernel.h"

namespace tmopt {
namespace {

template <int REP>
void launch(const DecodeArgs& a, int G, int nw, size_t lds, hipStream_t st) {
  hipLaunchKernelGGL((decode_kernel<REP, false, 0>), dim3(G, a.HKV / nw),
                     dim3(64 * nw), lds, st, a);
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" int tmopt_attn_decode_scored(
    const void* q, const void* k_pool, const void* v_pool,
    const int32_t* block_table, int64_t bt_stride, int table_wrap,
    const int32_t* ctx_lens, int B, int HQ, int HKV, int D, int page_size,
    int64_t num_pages, int window, float scale, float softcap,
    const float* slopes, const int32_t* first_keys, int min_pages,
    int num_workgroups, void* out, float* lse, void* workspace,
    size_t workspace_bytes, tmopt_stream_t stream) {
  clear_error();
  if (B == 0) return TMOPT_OK;
  TMOPT_REQUIRE(B > 0, TMOPT_EINVAL, "decode_scored: B=%d", B);
  TMOPT_REQUIRE(B <= kMaxB, TMOPT_EUNSUPPORTED, "decode_scored: B=%d above %d",
                B, kMaxB);
  TMOPT_REQUIRE(q && k_pool && v_pool && out && block_table && ctx_lens,
                TMOPT_EINVAL, "decode_scored: null tensor pointer");
  TMOPT_REQUIRE(D == kD && page_size == kPS, TMOPT_EUNSUPPORTED,
                "decode_scored: D=%d page_size=%d (only 128, 16)", D,
                page_size);
  TMOPT_REQUIRE(HKV > 0 && HQ > 0 && HQ % HKV == 0, TMOPT_EINVAL,
                "decode_scored: HQ=%d HKV=%d", HQ, HKV);
  // query heads per scheduled KV head, as in decode_paged
  const int ratio = HQ / HKV;
  int rep = ratio;
  while (rep > 16 || ratio % rep != 0) --rep;
  const int kv_div = ratio / rep;
  TMOPT_REQUIRE(HQ <= 131072 && (int64_t)HKV * kv_div <= 65535,
                TMOPT_EUNSUPPORTED,
                "decode_scored: HQ=%d, HKV=%d x %d query-head groups", HQ, HKV,
                kv_div);
  TMOPT_REQUIRE((int64_t)kPS * HKV * kD * 2 < (1ll << 31), TMOPT_EUNSUPPORTED,
                "decode_scored: page too large");
  TMOPT_REQUIRE(num_pages > 0 && bt_stride > 0 && table_wrap >= 0 &&
                    table_wrap <= bt_stride && window >= 0,
                TMOPT_EINVAL,
                "decode_scored: num_pages=%lld bt_stride=%lld table_wrap=%d "
                "window=%d",
                (long long)num_pages, (long long)bt_stride, table_wrap, window);
  TMOPT_REQUIRE(table_wrap == 0 ||
                    (window > 0 && (int64_t)window <= (int64_t)table_wrap * kPS),
                TMOPT_EINVAL,
                "decode_scored: window=%d outside a ring of %d pages", window,
                table_wrap);
  TMOPT_REQUIRE(scale > 0.0f && scale < INFINITY && good_cap(softcap, scale),
                TMOPT_EINVAL, "decode_scored: scale=%g softcap=%g", scale,
                softcap);
  TMOPT_REQUIRE(min_pages > 0 && num_workgroups >= 0 && num_workgroups <= 65535,
                TMOPT_EINVAL, "decode_scored: min_pages=%d num_workgroups=%d",
                min_pages, num_workgroups);
  TMOPT_REQUIRE(((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool |
                 (uintptr_t)out) % 16 == 0,
                TMOPT_EINVAL, "decode_scored: tensors must be 16-byte aligned");
  const int G = num_workgroups > 0 ? num_workgroups : default_wgs(HKV);
  size_t off_lse = 0, off_geo = 0;
  const size_t need = ws_layout(B, HQ, G, &off_lse, &off_geo);
  TMOPT_REQUIRE(workspace && workspace_bytes >= need &&
                    (uintptr_t)workspace % 16 == 0,
                TMOPT_EWORKSPACE,
                "decode_scored: workspace %zu bytes < %zu needed (or "
                "unaligned)",
                workspace_bytes, need);
  DecodeArgs a{};
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
  a.HKV = HKV * kv_div;
  a.rep = rep;
  a.kv_div = kv_div;
  a.HKV_stored = HKV;
  a.num_pages = num_pages > 0x7fffffff ? 0x7fffffff : (int)num_pages;
  a.window = window;
  a.scale_log2 = scale * kLog2e;
  // (a work-group's first page, its index times this, stays within int32)
  a.min_pages = min_pages < 32768 ? min_pages : 32768;
  a.out = (__bf16*)out;
  a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_lse = (float*)((char*)workspace + off_lse);
  a.geo = (int*)((char*)workspace + off_geo);
  a.cap = make_cap(softcap, scale);
  a.slopes = slopes;
  a.first = first_keys;
  const int nw = waves_per_wg(a.HKV);
  const size_t tab = ((2 * (size_t)B + 1 + 4) * sizeof(int) + 15) & ~(size_t)15;
  const size_t tiles = (size_t)nw * wave_lds(false);
  a.ids_off = (int)(tab > tiles ? tab : tiles);
  const size_t lds = a.ids_off + (ids_kept(false) + 2) * sizeof(int);
  hipStream_t st = (hipStream_t)stream;
  switch (kv_div == 1 ? rep : 0) {
    case 4: launch<4>(a, G, nw, lds, st); break;
    case 8: launch<8>(a, G, nw, lds, st); break;
    default: launch<0>(a, G, nw, lds, st); break;
  }
  const int rc = check_launch("decode_scored");
  if (rc) return rc;
  launch_combine<true>(a, G, st);
  return check_launch("decode_scored merge");
}
