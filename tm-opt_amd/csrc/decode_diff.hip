// Differential attention of one new token per request over the paged cache.
// One work-group per (request, head pair).
#include "diff_row.h"

namespace tmopt {
namespace {

struct DecodeDiffArgs {
  const __bf16* q;
  const __bf16* kpool;
  const __bf16* vpool;
  const int32_t* bt;
  int64_t bt_stride;
  int table_wrap;
  const int32_t* ctx_lens;
  int HQ, HKV;
  int64_t num_pages;
  int window;
  float scale;
  DiffWeights w;
  __bf16* out;
  float* lse;
};

__global__ __launch_bounds__(256) void decode_diff_kernel(DecodeDiffArgs a) {
  const int h = blockIdx.x, b = blockIdx.y;
  const int n = max(0, a.ctx_lens[b]);
  const int lo = a.window > 0 && n > a.window ? n - a.window : 0;
  const int64_t row_e = (int64_t)a.HKV * kD;
  const int32_t* const row = a.bt + b * a.bt_stride;
  auto rows = [&](int pos, int64_t& kr, int64_t& vr) {
    int lp = pos / kPage;
    if (a.table_wrap > 0) lp %= a.table_wrap;
    if (lp >= a.bt_stride) return;
    const int pg = row[lp];
    if (pg < 0 || pg >= a.num_pages) return;
    kr = vr = ((int64_t)pg * kPage + pos % kPage) * row_e;
  };
  const __bf16* const q = a.q + ((int64_t)b * a.HQ + 2 * h) * kD;
  float* const lse = a.lse ? a.lse + (int64_t)b * a.HQ + 2 * h : nullptr;
  diff_row<true>(q, q + kD, a.kpool, kD, a.vpool, kD, rows, h / (a.HQ / a.HKV), lo,
           n, a.scale, a.w, h, false,
           a.out + ((int64_t)b * (a.HQ / 2) + h) * kDV, lse, lse + 1);
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" size_t tmopt_attn_decode_diff_workspace_size(int B, int HQ, int HKV,
                                                        int D,
                                                        int num_workgroups) {
  (void)D;
  (void)num_workgroups;
  return B > 0 && HQ > 0 && HKV > 0 ? 16 : 0;
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
  TMOPT_REQUIRE(B <= 8192, TMOPT_EUNSUPPORTED, "decode_diff: B=%d above 8192",
                B);
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
  const size_t need = tmopt_attn_decode_diff_workspace_size(B, HQ, HKV, D,
                                                            num_workgroups);
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
  a.table_wrap = table_wrap;
  a.ctx_lens = ctx_lens;
  a.HQ = HQ;
  a.HKV = HKV;
  a.num_pages = num_pages;
  a.window = window;
  a.scale = scale;
  a.w = DiffWeights{lam, lam_stride, norm_weight, norm_eps, out_scale};
  a.out = (__bf16*)out;
  a.lse = lse;
  hipLaunchKernelGGL(decode_diff_kernel, dim3(HQ / 2, B), dim3(256), 0,
                     (hipStream_t)stream, a);
  return check_launch("decode_diff");
}
