// Varlen causal differential attention. One work-group per (query, head pair).
#include "diff_row.h"

namespace tmopt {
namespace {

struct PrefillDiffArgs {
  const __bf16* q;
  int64_t q_st, q_sh;
  const __bf16* k;
  int64_t k_st, k_sh;
  const __bf16* v;
  int64_t v_st, v_sh;
  const int32_t* cu;
  const int32_t* prior;
  const int32_t* bt;     // NULL: packed k / v
  int64_t bt_stride;
  int64_t num_pages;
  int HQ, HKV, S;
  int window;
  float scale;
  DiffWeights w;
  __bf16* out;
  int64_t o_st, o_sh;
  float* lse;
  int64_t lse_sh;
  const int32_t* reject;
};

__global__ __launch_bounds__(256) void prefill_diff_kernel(PrefillDiffArgs a) {
  const int h = blockIdx.x, j = blockIdx.y, s = blockIdx.z;
  const int t0 = a.cu[s], len = a.cu[s + 1] - t0;
  if (j >= len) return;
  const int pos = (a.prior ? a.prior[s] : 0) + j;
  const int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  const int32_t* const row = a.bt ? a.bt + s * a.bt_stride : nullptr;
  auto rows = [&](int p, int64_t& kr, int64_t& vr) {
    if (!row) {
      kr = (int64_t)(t0 + p) * a.k_st;
      vr = (int64_t)(t0 + p) * a.v_st;
      return;
    }
    if (p / kPage >= a.bt_stride) return;
    const int pg = row[p / kPage];
    if (pg < 0 || pg >= a.num_pages) return;
    kr = vr = ((int64_t)pg * kPage + p % kPage) * a.k_st;
  };
  const __bf16* const q = a.q + (int64_t)(t0 + j) * a.q_st + 2 * h * a.q_sh;
  const bool rejected = a.reject && *a.reject != 0;
  float* const lse = a.lse ? a.lse + 2 * h * a.lse_sh + t0 + j : nullptr;
  diff_row<false>(q, q + a.q_sh, a.k, a.k_sh, a.v, a.v_sh, rows, h / (a.HQ / a.HKV),
           lo, rejected ? lo : pos + 1, a.scale, a.w, h, rejected,
           a.out + (int64_t)(t0 + j) * a.o_st + h * a.o_sh, lse, lse + a.lse_sh);
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" size_t tmopt_attn_prefill_diff_workspace_size(
    int num_seqs, int max_seqlen_q, int HQ, int HKV, int64_t bt_stride,
    int window) {
  (void)num_seqs;
  (void)max_seqlen_q;
  (void)HQ;
  (void)HKV;
  (void)bt_stride;
  (void)window;
  return 0;
}

extern "C" int tmopt_attn_prefill_diff(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k,
    int64_t k_stride_tok, int64_t k_stride_head, const void* v,
    int64_t v_stride_tok, int64_t v_stride_head, const int32_t* cu_seqlens_q,
    const int32_t* prior_lens, int num_seqs, int max_seqlen_q,
    const void* k_pool, const void* v_pool, const int32_t* block_table,
    int64_t bt_stride, int page_size, int64_t num_pages, int HQ, int HKV,
    int D, int window, float scale, const float* lam, int lam_stride,
    const float* norm_weight, float norm_eps, float out_scale, void* out,
    int64_t o_stride_tok, int64_t o_stride_head, float* lse,
    int64_t lse_stride_head, const int32_t* reject, void* workspace, size_t workspace_bytes,
    tmopt_stream_t stream) {
  clear_error();
  if (num_seqs == 0 || max_seqlen_q == 0) return TMOPT_OK;
  TMOPT_REQUIRE(num_seqs > 0 && num_seqs <= 65535 && max_seqlen_q > 0,
                TMOPT_EINVAL, "prefill_diff: num_seqs=%d max_seqlen_q=%d",
                num_seqs, max_seqlen_q);
  TMOPT_REQUIRE(q && out && cu_seqlens_q, TMOPT_EINVAL,
                "prefill_diff: null q/out/cu_seqlens");
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
  const size_t need = tmopt_attn_prefill_diff_workspace_size(
      num_seqs, max_seqlen_q, HQ, HKV, paged ? bt_stride : 0, window);
  TMOPT_REQUIRE(need == 0 || !workspace ||
                    (workspace_bytes >= need &&
                     (uintptr_t)workspace % 16 == 0),
                TMOPT_EWORKSPACE,
                "prefill_diff: workspace %zu bytes < %zu needed (or unaligned)",
                workspace_bytes, need);
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
  a.num_pages = num_pages;
  a.HQ = HQ;
  a.HKV = HKV;
  a.S = num_seqs;
  a.window = window;
  a.scale = scale;
  a.w = DiffWeights{lam, lam_stride, norm_weight, norm_eps, out_scale};
  a.out = (__bf16*)out;
  a.o_st = o_stride_tok;
  a.o_sh = o_stride_head;
  a.lse = lse;
  a.lse_sh = lse_stride_head;
  a.reject = reject;
  TMOPT_REQUIRE(max_seqlen_q <= 65535, TMOPT_EUNSUPPORTED,
                "prefill_diff: max_seqlen_q=%d", max_seqlen_q);
  hipLaunchKernelGGL(prefill_diff_kernel, dim3(HQ / 2, max_seqlen_q, num_seqs),
                     dim3(256), 0, (hipStream_t)stream, a);
  return check_launch("prefill_diff");
}
