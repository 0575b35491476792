// C entry points of the scored prefill and of the prefill over the 4-bit cache,
// and the scored kernels of whole items (kernels: prefill_kernel.h; split keys:
// prefill_scored_split.hip, prefill_mx4_split.hip).
#define TMOPT_PREFILL_SHORT_PIECES
#define TMOPT_PREFILL_SCORED
#include "prefill_host.h"

namespace tmopt {
namespace {

template <int REP>
void launch(const PrefillArgs& a, int src, size_t lds, hipStream_t st) {
  const dim3 grid((unsigned)a.n_base);
#define TMOPT_LAUNCH(K)                                                  \
  case K:                                                                \
    hipLaunchKernelGGL((prefill_kernel<REP, false, K>), grid, dim3(512), \
                       lds, st, a);                                      \
    break;
  switch (scored_kind(a, src)) { TMOPT_SCORED_KINDS(TMOPT_LAUNCH) }
#undef TMOPT_LAUNCH
}

// Keys a query may see at most, for the decision to split: the runs' own, or
// what the block table's width and the caller's bound leave.
int levels_of(int64_t n_base, int BQ, int max_seqlen, int64_t max_context,
              int64_t bt_stride, int window) {
  if (bt_stride <= 0)
    return split_levels(n_base, BQ, max_seqlen, window, 48);
  int64_t keys = bt_stride > (1 << 26) ? 1ll << 30 : bt_stride * kPage;
  if (max_context > 0 && max_context < keys) keys = max_context;
  return split_levels(n_base, BQ, keys, window, kMinSplit);
}

size_t workspace_of(int num_seqs, int max_seqlen_q, int64_t max_context,
                    int HQ, int HKV, int64_t bt_stride, int window) {
  if (num_seqs <= 0 || max_seqlen_q <= 0 || HKV <= 0 || HQ <= 0 ||
      HQ % HKV != 0)
    return 0;
  const int rep = query_group(HQ / HKV);
  const int64_t hkv = HQ / rep;
  if (hkv > 65535) return 0;
  const int bq = 256 / rep;
  const int64_t n = level_wgs((int)hkv, bq, num_seqs, max_seqlen_q);
  const int levels =
      levels_of(n, bq, max_seqlen_q, max_context, bt_stride, window);
  return levels > 1 ? (size_t)workspace_bytes_of(levels, n) : 0;
}

// What the two entry points share. `src` and the key pointers of `a` are set.
int run(const char* what, PrefillArgs& a, int src, const void* q,
        int64_t q_stride_tok, int64_t q_stride_head, const int32_t* cu,
        const int32_t* prior, int num_seqs, int max_seqlen_q,
        int64_t max_context, const int32_t* block_table, int64_t bt_stride,
        int page_size, int64_t num_pages, int HQ, int HKV, int D, int window,
        float scale, float softcap, const float* slopes, void* out,
        int64_t o_stride_tok, int64_t o_stride_head, float* lse,
        int64_t lse_stride_head, const int32_t* reject, void* workspace,
        size_t workspace_bytes, hipStream_t st) {
  TMOPT_REQUIRE(num_seqs > 0 && num_seqs <= 65535 && max_seqlen_q > 0 &&
                    max_context >= 0,
                TMOPT_EINVAL, "%s: num_seqs=%d max_seqlen_q=%d max_context=%lld",
                what, num_seqs, max_seqlen_q, (long long)max_context);
  TMOPT_REQUIRE(q && out && cu, TMOPT_EINVAL, "%s: null q/out/cu_seqlens",
                what);
  TMOPT_REQUIRE(D == kD, TMOPT_EUNSUPPORTED, "%s: D=%d (only 128)", what, D);
  TMOPT_REQUIRE(HKV > 0 && HQ > 0 && HQ % HKV == 0 && HKV <= 65535,
                TMOPT_EINVAL, "%s: HQ=%d HKV=%d", what, HQ, HKV);
  const int rep = query_group(HQ / HKV);
  const int bq = 256 / rep;
  TMOPT_REQUIRE(HQ / rep <= 65535, TMOPT_EUNSUPPORTED,
                "%s: %d query-head groups exceed 65535", what, HQ / rep);
  TMOPT_REQUIRE(window >= 0 && scale > 0.0f && scale < INFINITY &&
                    good_cap(softcap, scale),
                TMOPT_EINVAL, "%s: window=%d scale=%g softcap=%g", what, window,
                scale, softcap);
  TMOPT_REQUIRE((int64_t)(HQ / rep) * num_seqs *
                            ((max_seqlen_q + bq - 1) / bq) + 64 <
                    0x7fffffffll,
                TMOPT_EUNSUPPORTED, "%s: the grid exceeds its limit", what);
  if (src != kPacked) {
    TMOPT_REQUIRE(block_table && bt_stride > 0 && num_pages > 0, TMOPT_EINVAL,
                  "%s: block table, bt_stride=%lld num_pages=%lld", what,
                  (long long)bt_stride, (long long)num_pages);
    TMOPT_REQUIRE(page_size == kPage, TMOPT_EUNSUPPORTED,
                  "%s: page_size=%d (only 16)", what, page_size);
    TMOPT_REQUIRE((int64_t)kPage * HKV * kD * 2 < (1ll << 31),
                  TMOPT_EUNSUPPORTED, "%s: page too large", what);
  }
  TMOPT_REQUIRE(((int64_t)max_seqlen_q * q_stride_tok + kD) * 2 < kOob,
                TMOPT_EUNSUPPORTED, "%s: a run's q span must stay below 2 GiB",
                what);
  TMOPT_REQUIRE(q_stride_tok >= 0 && q_stride_tok % 8 == 0 &&
                    q_stride_head % 8 == 0 && o_stride_tok % 4 == 0 &&
                    o_stride_head % 4 == 0 && (uintptr_t)q % 16 == 0 &&
                    (uintptr_t)out % 8 == 0,
                TMOPT_EINVAL, "%s: q/out rows misaligned", what);
  TMOPT_REQUIRE(lse_stride_head >= 0, TMOPT_EINVAL, "%s: lse_stride_head=%lld",
                what, (long long)lse_stride_head);
  a.q = (const __bf16*)q;
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_head;
  a.k_sd = a.v_sd = 1;
  a.cu = cu;
  a.prior = prior;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.bt_width = bt_stride > 0x7fffffff ? 0x7fffffff : (int)bt_stride;
  a.num_pages = num_pages > 0x7fffffff ? 0x7fffffff : (int)num_pages;
  a.page_size = kPage;
  a.HQ = HQ;
  a.HKV = HQ / rep;
  a.kv_div = a.HKV / HKV;
  a.HKV_stored = HKV;
  a.window = window;
  a.scale = scale;
  a.scale_log2 = scale * kLog2e;
  a.cap = make_cap(softcap, scale);
  a.slopes = slopes;
  a.out = (__bf16*)out;
  a.o_st = o_stride_tok;
  a.o_sh = o_stride_head;
  a.lse = lse;
  a.lse_sh = lse_stride_head;
  a.S = num_seqs;
  a.reject = reject;
  a.n_base = (int)level_wgs(a.HKV, bq, num_seqs, max_seqlen_q);
  a.split_wgs = device_cus();
  a.nsplit = workspace == nullptr
                 ? 1
                 : levels_of(a.n_base, bq, max_seqlen_q, max_context,
                             src == kPacked ? 0 : bt_stride, window);
  const int64_t slots = (int64_t)a.nsplit * a.n_base;
  const int64_t need = workspace_bytes_of(a.nsplit, a.n_base);
  TMOPT_REQUIRE(a.nsplit <= 1 || ((int64_t)workspace_bytes >= need &&
                                  (uintptr_t)workspace % 16 == 0),
                TMOPT_EWORKSPACE,
                "%s: workspace %zu bytes < %lld needed (or unaligned)", what,
                workspace_bytes, (long long)need);
  a.part_o = (float*)workspace;
  a.part_lse = a.part_o + slots * 256 * kD;
  a.part_n = (int*)(a.part_lse + slots * 256);
  a.nqb_max = (max_seqlen_q + bq - 1) / bq;
  const size_t lds = kNStage * kStage + (a.rel ? 8 * kBiasB : 0);
  const bool scored = src != kPaged4 || softcap > 0.0f || slopes ||
                      (scale > kMaxRaw && !a.rel);
  if (scored && a.nsplit > 1) {
    launch_prefill_scored_split(a, rep, src, lds, st);
  } else if (scored) {
    launch_prefill_scored(a, rep, src, lds, st);
  } else if (a.nsplit > 1) {
    launch_prefill_mx4_split(a, rep, lds, st);
  } else {
    launch_prefill_mx4(a, rep, lds, st);
  }
  return check_launch(what);
}

}  // namespace

void launch_prefill_scored(const PrefillArgs& a, int rep, int src, size_t lds,
                           hipStream_t st) {
  if (rep == 8)
    launch<8>(a, src, lds, st);
  else if (rep == 4)
    launch<4>(a, src, lds, st);
  else if (rep == 2)
    launch<2>(a, src, lds, st);
  else
    launch<1>(a, src, lds, st);
}

}  // namespace tmopt

using namespace tmopt;

extern "C" size_t tmopt_attn_prefill_scored_workspace_size(
    int num_seqs, int max_seqlen_q, int64_t max_context, int HQ, int HKV,
    int64_t bt_stride, int window) {
  return workspace_of(num_seqs, max_seqlen_q, max_context, HQ, HKV, bt_stride,
                      window);
}

extern "C" int tmopt_attn_prefill_scored_strided(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k,
    int64_t k_stride_tok, int64_t k_stride_head, const void* v,
    int64_t v_stride_tok, int64_t v_stride_head, const int32_t* cu_seqlens_q,
    const int32_t* prior_lens, int num_seqs, int max_seqlen_q,
    int64_t max_context, const void* k_pool, const void* v_pool,
    const int32_t* block_table, int64_t bt_stride, int page_size,
    int64_t num_pages, int HQ, int HKV, int D, int window, float scale,
    float softcap, const float* slopes, const int32_t* first_keys,
    const int32_t* prefix_lens, void* out, int64_t o_stride_tok,
    int64_t o_stride_head, float* lse, int64_t lse_stride_head,
    const int32_t* reject, void* workspace, size_t workspace_bytes,
    tmopt_stream_t stream) {
  clear_error();
  if (num_seqs == 0 || max_seqlen_q == 0) return TMOPT_OK;
  PrefillArgs a{};
  const bool pooled = block_table != nullptr;
  if (pooled) {
    TMOPT_REQUIRE(!k && !v && k_pool && v_pool, TMOPT_EINVAL,
                  "prefill_scored: keys come from k/v or from the pools");
    TMOPT_REQUIRE(((uintptr_t)k_pool | (uintptr_t)v_pool) % 16 == 0,
                  TMOPT_EINVAL, "prefill_scored: pools must be 16-byte aligned");
  } else {
    TMOPT_REQUIRE(k && v && !prior_lens, TMOPT_EINVAL,
                  "prefill_scored: k/v missing, or prior context without a "
                  "block table");
    const int64_t most =
        k_stride_tok > v_stride_tok ? k_stride_tok : v_stride_tok;
    TMOPT_REQUIRE(((uintptr_t)k | (uintptr_t)v) % 16 == 0 &&
                      k_stride_tok >= 0 && v_stride_tok >= 0 &&
                      k_stride_tok % 8 == 0 && v_stride_tok % 8 == 0 &&
                      k_stride_head % 8 == 0 && v_stride_head % 8 == 0,
                  TMOPT_EINVAL,
                  "prefill_scored: k/v rows must be 16-byte aligned");
    TMOPT_REQUIRE(max_seqlen_q < 0 ||
                      ((int64_t)max_seqlen_q * most + kD) * 2 < kOob,
                  TMOPT_EUNSUPPORTED,
                  "prefill_scored: a run's k/v span must stay below 2 GiB");
  }
  a.k = (const __bf16*)k;
  a.k_st = k_stride_tok;
  a.k_sh = k_stride_head;
  a.v = (const __bf16*)v;
  a.v_st = v_stride_tok;
  a.v_sh = v_stride_head;
  a.kpool = (const __bf16*)k_pool;
  a.vpool = (const __bf16*)v_pool;
  a.first = first_keys;
  a.prefix = prefix_lens;
  return run("prefill_scored", a, pooled ? kPaged : kPacked, q, q_stride_tok,
             q_stride_head, cu_seqlens_q, prior_lens, num_seqs, max_seqlen_q,
             max_context, block_table, bt_stride, page_size, num_pages, HQ,
             HKV, D, window, scale, softcap, slopes, out, o_stride_tok,
             o_stride_head, lse, lse_stride_head, reject, workspace,
             workspace_bytes, (hipStream_t)stream);
}

extern "C" int tmopt_attn_prefill_scored(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k,
    int64_t k_stride_tok, int64_t k_stride_head, const void* v,
    int64_t v_stride_tok, int64_t v_stride_head, const int32_t* cu_seqlens_q,
    const int32_t* prior_lens, int num_seqs, int max_seqlen_q,
    int64_t max_context, const void* k_pool, const void* v_pool,
    const int32_t* block_table, int64_t bt_stride, int page_size,
    int64_t num_pages, int HQ, int HKV, int D, int window, float scale,
    float softcap, const float* slopes, const int32_t* first_keys,
    const int32_t* prefix_lens, void* out, int64_t o_stride_tok,
    int64_t o_stride_head, float* lse, const int32_t* reject, void* workspace,
    size_t workspace_bytes, tmopt_stream_t stream) {
  return tmopt_attn_prefill_scored_strided(
      q, q_stride_tok, q_stride_head, k, k_stride_tok, k_stride_head, v,
      v_stride_tok, v_stride_head, cu_seqlens_q, prior_lens, num_seqs,
      max_seqlen_q, max_context, k_pool, v_pool, block_table, bt_stride,
      page_size, num_pages, HQ, HKV, D, window, scale, softcap, slopes,
      first_keys, prefix_lens, out, o_stride_tok, o_stride_head, lse, 0, reject,
      workspace, workspace_bytes, stream);
}

extern "C" size_t tmopt_attn_prefill_mx4_workspace_size(
    int num_seqs, int max_seqlen_q, int64_t max_context, int HQ, int HKV,
    int64_t bt_stride, int window) {
  return bt_stride <= 0 ? 0
                        : workspace_of(num_seqs, max_seqlen_q, max_context, HQ,
                                       HKV, bt_stride, window);
}

extern "C" int tmopt_attn_prefill_mx4_strided(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head,
    const int32_t* cu_seqlens_q, const int32_t* prior_lens, int num_seqs,
    int max_seqlen_q, int64_t max_context, const void* pool,
    const int32_t* block_table, int64_t bt_stride, int page_size,
    int64_t num_pages, int HQ, int HKV, int D, int window, float scale,
    float softcap, const float* slopes, const void* rel,
    int64_t rel_stride_tok, int64_t rel_stride_head, int rel_extent, void* out,
    int64_t o_stride_tok, int64_t o_stride_head, float* lse,
    int64_t lse_stride_head, const int32_t* reject, void* workspace,
    size_t workspace_bytes, tmopt_stream_t stream) {
  clear_error();
  if (num_seqs == 0 || max_seqlen_q == 0) return TMOPT_OK;
  TMOPT_REQUIRE(pool && (uintptr_t)pool % 16 == 0, TMOPT_EINVAL,
                "prefill_mx4: pool null or not 16-byte aligned");
  TMOPT_REQUIRE(rel == nullptr || (softcap == 0.0f && slopes == nullptr),
                TMOPT_EUNSUPPORTED,
                "prefill_mx4: a relative bias goes without softcap and slopes");
  TMOPT_REQUIRE(rel == nullptr || (rel_extent > 0 && (uintptr_t)rel % 2 == 0 &&
                                   !(scale < kMinRaw)),
                TMOPT_EINVAL, "prefill_mx4: rel_extent=%d scale=%g", rel_extent,
                scale);
  TMOPT_REQUIRE(rel == nullptr ||
                    (rel_stride_tok >= rel_extent && rel_stride_head >= 0 &&
                     64 * rel_stride_tok + 2 * (int64_t)rel_extent < kOob),
                TMOPT_EUNSUPPORTED,
                "prefill_mx4: rel rows must not overlap, and 32 rows must span "
                "less than 2 GiB (stride_tok=%lld, extent=%d)",
                (long long)rel_stride_tok, rel_extent);
  PrefillArgs a{};
  a.pool4 = (const uint8_t*)pool;
  a.rel = (const __bf16*)rel;
  a.r_st = rel_stride_tok;
  a.r_sh = rel_stride_head;
  a.rel_extent = rel ? rel_extent : 0;
  return run("prefill_mx4", a, kPaged4, q, q_stride_tok, q_stride_head,
             cu_seqlens_q, prior_lens, num_seqs, max_seqlen_q, max_context,
             block_table, bt_stride, page_size, num_pages, HQ, HKV, D, window,
             scale, softcap, slopes, out, o_stride_tok, o_stride_head, lse,
             lse_stride_head, reject, workspace, workspace_bytes,
             (hipStream_t)stream);
}

extern "C" int tmopt_attn_prefill_mx4(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head,
    const int32_t* cu_seqlens_q, const int32_t* prior_lens, int num_seqs,
    int max_seqlen_q, int64_t max_context, const void* pool,
    const int32_t* block_table, int64_t bt_stride, int page_size,
    int64_t num_pages, int HQ, int HKV, int D, int window, float scale,
    float softcap, const float* slopes, const void* rel,
    int64_t rel_stride_tok, int64_t rel_stride_head, int rel_extent, void* out,
    int64_t o_stride_tok, int64_t o_stride_head, float* lse,
    const int32_t* reject, void* workspace, size_t workspace_bytes,
    tmopt_stream_t stream) {
  return tmopt_attn_prefill_mx4_strided(
      q, q_stride_tok, q_stride_head, cu_seqlens_q, prior_lens, num_seqs,
      max_seqlen_q, max_context, pool, block_table, bt_stride, page_size,
      num_pages, HQ, HKV, D, window, scale, softcap, slopes, rel,
      rel_stride_tok, rel_stride_head, rel_extent, out, o_stride_tok,
      o_stride_head, lse, 0, reject, workspace, workspace_bytes, stream);
}
