// Split-KV paged decode attention over the 4-bit cache (format: mx4.h).
//
// One query token per sequence against its history; the balanced persistent
// grid, the pieces and their merge are the bf16 decode's (decode_kernel.h).
// What differs:
//
//  * A token costs 136 bytes a head instead of 512, so the same bandwidth
//    brings four times the keys to a compute unit, and what is done per key
//    counts. Nothing passes through LDS: lane (n, g) = (lane & 15, lane >> 4)
//    loads its MFMA operands of a page by itself, 16 bytes of K (block g of
//    token n) and 16 of V (dims 8n..8n+7 of tokens 4g..4g+3), the 64 of them a
//    contiguous KB, a byte of K scale and four of V scales. (Lanes 64 bytes
//    apart cost nothing measurable: the same loads with lane l at byte 16 l took
//    the same time, 45.1 us at 64 requests.)
//  * K becomes bf16 in registers (v_cvt_scalef32_pk_bf16_fp4: two elements
//    and their block's scale in one instruction, exact) and S^T = K.Q^T runs
//    on v_mfma_f32_16x16x32_bf16. (The f8f6f4 MFMA takes K as it is stored, and
//    a query's 8 bits as two e4m3 parts in 16 columns are exact; but it adds the
//    32 products of a block with some 13 bits below the largest: scores of
//    spread 20 came out wrong by 1e-3.)
//  * The 16 columns hold the up to 8 query heads of a KV head twice: column n
//    and n + 8 are one head. P.V uses the second copy to save the transpose
//    of V: two elements of a V byte are two dims of one token, while an MFMA's
//    k axis runs over tokens. So the k axis takes (token, parity of dim) pairs
//    as they lie, rows are pairs of dims, and column n holds the probability
//    at the pairs of even dims and zero at the odd ones, column n + 8 the other
//    way round: O^T of even dims comes out in column n, of odd ones in n + 8.
//    As many MFMAs as the plain form for 8 heads, and none of the 16 permutes
//    a page would need.
//  * Four pages (64 keys) a step; the next step's loads are out before a step
//    is computed. One wave per SIMD (256 ranges of 4 heads): a step is ~250
//    vector, ~100 scalar and 32 matrix instructions, 0.90 us of a SIMD with its
//    pages in the L2, and a second wave beside it adds nothing, since they share
//    the issue (512 ranges, or two waves that share a range's steps: 40.2 and
//    36.1 against 34.7 us at 64 requests). Nor do deeper prefetch (three
//    buffers 36.5) or steps of 2, 6 and 8 pages (40.0, 37.7, 39.1 against 35.7).
//
// What bounds it: 64 requests of 1K-8K tokens (32Q/4KV, 162 MB) 34.3 us a call
// with its merge, the kernel 28.4-30.4: HBM, 6.4 TB/s between ~5 us of start
// (lengths, page ids, first pages) and the last piece; where a KV head has four
// query heads or fewer, or there is a bias, the steps' instructions (96 requests,
// window 512, 64Q/16KV with bias: 35.1 us for 118 MB).
#include "decode_kernel.h"
#include "mx4.h"
#include "score.h"

namespace tmopt {
namespace {

constexpr int kMaxRep = 8;        // query heads per wave
constexpr int kPages = 4;         // pages of a step
constexpr int kIds4 = 400;        // steps of a range whose page ids LDS keeps
constexpr int kNt = 2;            // non-temporal: pages are read once

struct Mx4Args {
  DecodeArgs d;   // (first: the page lookups read it in the argument segment)
  const uint8_t* pool;
  Cap cap;
  const float* slopes;   // [HQ] or null
};

// Up to four pages of one sequence (wave-uniform).
struct Step4 {
  int b;       // sequence (-1: past the end of this work-group's range)
  int n;       // its context length
  int pg;      // first logical page
  int flags;   // kFirst, kLast, kFull, kWhole; page j is there: kHave << j
};
enum : int { kHave = 64 };   // (bit 6)

typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));

// What a lane loads of a step.
template <bool REL>
struct Buf4 {
  u32x4 k[kPages], v[kPages];
  uint32_t ks[kPages], vs[kPages];
  u32x3 bias[REL ? kPages : 1];         // the dwords that hold rel[d - 3 .. d]
};

// the value of lane n ^ 8 of each 16 lanes
__device__ __forceinline__ float other_half(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128,
                                         0xF, 0xF, true));   // row_ror 8
}

// SCORE: 1 with a score function, 2 with a cap above Cap::kNear (a kernel of its
// own: as a branch of the other's steps it cost these 1-2%)
template <bool REL, int SCORE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
void decode_mx4_kernel(Mx4Args args) {
  const DecodeArgs& a = args.d;
  extern __shared__ __align__(16) char smem[];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nw = blockDim.x >> 6;
  const int n16 = lane & 15;
  const int g = lane >> 4;
  const int wg = blockIdx.x;
  const int G = gridDim.x;
  const int kvh = blockIdx.y * nw + w;
  int* pref = reinterpret_cast<int*>(smem);  // [B + 1]
  int* wsum = pref + a.B + 1;                // [4]
  int* nlen = wsum + 4;                      // [B]
  int* ids = reinterpret_cast<int*>(smem + a.ids_off);   // [kIds4 * kPages]

  // ---- the steps of the batch: prefix sums, this work-group's range --------
  // A sequence has one step for every four of its visible pages, and a range is
  // C steps of the batch: a step of one page costs what one of four does, so
  // ranges of as many steps end together (ranges of pages gave eight requests of
  // a few tokens to one work-group: 64 of 16 tokens took 22.8 us, now 8.2).
  // (n - 1) / 16 + 1 pages: lengths may come up to 2^31 - 1. Pages past the
  // table's width have no entry and are not walked.
  auto first_page = [&](int n) { return vis_lo(n, a.window) / kPS; };
  auto pages_of = [&](int n) {
    int last = n <= 0 ? 0 : (n - 1) / kPS + 1;
    if (a.table_wrap == 0) last = min(last, a.bt_width);
    return max(0, last - first_page(n));
  };
  auto steps_of = [&](int n) { return (pages_of(n) + kPages - 1) / kPages; };
  if (a.B <= 64) {   // one wave's scan, one barrier
    const int nb = lane < a.B ? a.ctx_lens[lane] : 0;
    const int x = wave_scan(steps_of(nb));
    if (w == 0 && lane < a.B) {
      nlen[lane] = nb;
      pref[lane + 1] = x;
      if (lane == 0) pref[0] = 0;
    }
    __syncthreads();
  } else {
    int carry = 0;
    for (int b0 = 0; b0 < a.B; b0 += blockDim.x) {
      const int b = b0 + threadIdx.x;
      const int nb = b < a.B ? a.ctx_lens[b] : 0;
      if (b < a.B) nlen[b] = nb;
      const int x = wave_scan(steps_of(nb));
      if (lane == 63) wsum[w] = x;
      __syncthreads();
      int before = carry;
      for (int j = 0; j < w; ++j) before += wsum[j];
      if (b < a.B) pref[b + 1] = before + x;
      for (int j = 0; j < nw; ++j) carry += wsum[j];
      __syncthreads();
    }
    if (threadIdx.x == 0) pref[0] = 0;
    __syncthreads();
  }
  const int U = __builtin_amdgcn_readfirstlane(pref[a.B]);
  const int C = max((U + G - 1) / G, (a.min_pages - 1) / kPages + 1);
  if (wg == 0 && blockIdx.y == 0) {   // for the merge
    for (int i = threadIdx.x; i <= a.B; i += blockDim.x) a.geo[1 + i] = pref[i];
    if (threadIdx.x == 0) a.geo[0] = C;
  }
  const int u0 = (int)min((int64_t)wg * C, (int64_t)U);
  const int u1 = (int)min((int64_t)u0 + C, (int64_t)U);
  const int col = n16 & 7;               // this lane's query head of the group
  const int odd = n16 >> 3;
  const bool head_ok = col < a.rep;
  const int hq = kvh * a.rep + (head_ok ? col : 0);

  // ---- sequences without a key: output 0, LSE -inf --------------------------
  for (int b = wg; b < a.B; b += G) {
    if (pref[b + 1] != pref[b] || !head_ok) continue;
    u32x4* const o = reinterpret_cast<u32x4*>(
        a.out + ((int64_t)b * a.HQ + hq) * kD + 64 * odd + 16 * g);
    o[0] = o[1] = u32x4{0, 0, 0, 0};
    if (a.lse && g == 0 && !odd) a.lse[(int64_t)b * a.HQ + hq] = -INFINITY;
  }
  if (u0 >= u1) return;

  // ---- the page ids of the range, and its steps ----------------------------
  auto seq_of = [&](int u) {   // first sequence with pref[b + 1] > u
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (pref[mid + 1] > u) hi = mid; else lo = mid + 1;
    }
    return lo;
  };
  const int nids = min(u1 - u0, kIds4) * kPages;
  for (int i = threadIdx.x; i < nids; i += blockDim.x) {
    const int u = u0 + i / kPages;
    const int b = seq_of(u);
    const int pg = (u - pref[b]) * kPages + i % kPages;
    ids[i] = pg < pages_of(nlen[b])
                 ? page_id<0>(kernel_args(false), b, first_page(nlen[b]) + pg)
                 : -1;
    if (i == 0) wsum[0] = b;
  }
  __syncthreads();
  // the sequence of the next step, from step seq_start of the batch on
  int cb = __builtin_amdgcn_readfirstlane(wsum[0]);
  int seq_start = __builtin_amdgcn_readfirstlane(pref[cb]);
  int cur_n, cur_lo, seq_end, piece_end, seq_flags;
  auto enter = [&](int n) __attribute__((always_inline)) {
    cur_n = n;
    cur_lo = vis_lo(n, a.window);
    seq_end = seq_start + steps_of(n);
    piece_end = min(seq_end, u1);
    seq_flags = kFirst | (seq_start >= u0 && seq_end <= u1 ? kWhole : 0);
  };
  enter(__builtin_amdgcn_readfirstlane(nlen[cb]));
  int cu = u0;
  int cur_pg = first_page(cur_n) + (u0 - seq_start) * kPages;
  i32x4 id_next = reinterpret_cast<const i32x4*>(ids)[0];   // a step ahead
  auto next_step = [&](Step4& st, int (&phys)[kPages])
      __attribute__((always_inline)) {
    st.b = -1;
    st.n = st.pg = st.flags = 0;
#pragma unroll
    for (int j = 0; j < kPages; ++j) phys[j] = -1;
    if (cu >= u1) return;
    if (cu >= seq_end) {
      do {
        ++cb;
        seq_start = seq_end;
        enter(as_const(a.ctx_lens)[cb]);
      } while (seq_end <= cu);
      cur_pg = first_page(cur_n);
    }
    st.b = cb;
    st.n = cur_n;
    st.pg = cur_pg;
    const int at = cu - u0;
    if (at < kIds4) {
#pragma unroll
      for (int j = 0; j < kPages; ++j)
        phys[j] = __builtin_amdgcn_readfirstlane(id_next[j]);
      id_next = reinterpret_cast<const i32x4*>(ids)[min(at + 1, kIds4 - 1)];
    } else {
      const int last = first_page(cur_n) + pages_of(cur_n);
#pragma unroll
      for (int j = 0; j < kPages; ++j)
        if (cur_pg + j < last)
          phys[j] = page_id<0>(kernel_args(true), cb, cur_pg + j);
    }
    ++cu;
    // (a full step has its 64 keys below n, so cur_pg * 16 + 64 is in range)
    const bool full = (phys[0] | phys[1] | phys[2] | phys[3]) >= 0 &&
                      cur_n - cur_pg * kPS >= 64 && cur_pg * kPS >= cur_lo;
    st.flags = seq_flags | (cu == piece_end ? kLast : 0) | (full ? kFull : 0);
#pragma unroll
    for (int j = 0; j < kPages; ++j)
      st.flags |= (int)((uint32_t)~phys[j] >> 31) << (6 + j);
    seq_flags &= ~kFirst;
    cur_pg += kPages;
  };

  // ---- loads ----------------------------------------------------------------
  // A page's record is one buffer resource (an absent page: an empty one,
  // whose loads give zeros and fetch nothing), so every step issues the same
  // loads of pages and the waits for them need no branch. A piece's query rows
  // come before the pages of its first step.
  const int kvs = kvh / a.kv_div;
  const int rec_page = a.HKV_stored * kRecB;
  const int at_k = 64 * n16 + 16 * g;
  const int at_ks = kRecKs + 16 * g + n16;
  const int at_vs = kRecVs + 16 * (n16 >> 2) + 4 * g;
  const int at_q = (hq * kD + 32 * g) * 2;   // dims 32 g .. of the head's row
  u32x4 q_next[4];   // query rows of a piece, with its first step
  auto load = [&](Buf4<REL>& x, const Step4& st, const int (&phys)[kPages])
      __attribute__((always_inline)) {
    if (st.flags & kFirst) {
      const auto rq = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<__bf16*>(a.q + (int64_t)st.b * a.HQ * kD), (short)0,
          a.HQ * kD * 2, 0x00020000);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        q_next[kk] =
            __builtin_amdgcn_raw_buffer_load_b128(rq, at_q + 16 * kk, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<uint8_t*>(args.pool) +
              ((int64_t)max(phys[j], 0) * rec_page + kvs * kRecB),
          (short)0, phys[j] >= 0 ? kRecB : 0, 0x00020000);
      x.k[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, at_k, 0, kNt);
      x.ks[j] = __builtin_amdgcn_raw_buffer_load_b8(rs, at_ks, 0, 0);
      x.v[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, at_k + kRecV, 0, kNt);
      x.vs[j] = __builtin_amdgcn_raw_buffer_load_b32(rs, at_vs, 0, 0);
    }
    if constexpr (REL) {
      // rel[d - 3 .. d] of tokens 4g + 3 .. 4g of each page: three dwords from
      // the one that holds rel[d - 3], in a resource that starts at the dword of
      // the sequence's first value. (Before it there is nothing to read: a lane
      // whose keys come up to the query itself may start there instead, see
      // below.) What another head's values put into a score is masked or past
      // the band.
      const char* const row = reinterpret_cast<const char*>(a.rel) +
                              (int64_t)max(st.b, 0) * a.HQ * a.rel_extent * 2;
      const int mis = (int)((uintptr_t)row & 3);
      const int dist = st.n - 1 - st.pg * kPS;
      const bool band = st.b >= 0 && dist - 63 < a.rel_extent;
      const auto rr = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(row - mis), (short)0,
          band ? (a.HQ * a.rel_extent * 2 + mis + 3) & ~3 : 0, 0x00020000);
#pragma unroll
      for (int j = 0; j < kPages; ++j) {
        const int o = ((hq * a.rel_extent + dist - 16 * j - 4 * g - 3) * 2 +
                       mis) & ~3;
        x.bias[j] = __builtin_amdgcn_raw_buffer_load_b96(rr, max(o, 0), 0, 0);
      }
    }
  };

  // ---- per-piece state ------------------------------------------------------
  f32x4 o_acc[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) o_acc[m] = f32x4{0, 0, 0, 0};
  float m_run = -INFINITY, l_part = 0.0f;
  bf16x8 qf[4];
  // (v_perm: bytes 4..7 are the two probabilities, 0x0c a zero)
  const uint32_t p_sel0 = odd ? 0x05040c0cu : 0x0c0c0504u;
  const uint32_t p_sel1 = odd ? 0x07060c0cu : 0x0c0c0706u;
  [[maybe_unused]] float slope = 0.0f;
  if constexpr (SCORE != 0)
    if (args.slopes) slope = args.slopes[hq] * kLog2e;

  auto compute = [&](const Buf4<REL>& x, const Step4& st)
      __attribute__((always_inline)) {
    // ---- scores -------------------------------------------------------------
    float s[kPages][4];   // (without a cap the scale comes with the exponent)
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      f32x4 c = f32x4{0, 0, 0, 0};
      const float ks = scale_f32(x.ks[j]);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, dequantise8(x.k[j][kk], ks)), qf[kk], c,
            0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j][i] = c[i];
    }
    if constexpr (SCORE == 2) {
#pragma unroll
      for (int j = 0; j < kPages; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[j][i] = args.cap.far(s[j][i]);
    } else if constexpr (SCORE == 1) {
      if (args.cap.in != 0.0f) {
        if (__builtin_expect(!(st.flags & kFull), 0)) {
          // (the bytes of a key that is not there are nobody's: they do not
          // choose the form of the cap)
          const int lo = vis_lo(st.n, a.window) - st.pg * kPS;
          const int hi = st.n - st.pg * kPS;
#pragma unroll
          for (int j = 0; j < kPages; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int at = 16 * j + 4 * g + i;
              const bool ok =
                  (st.flags & (kHave << j)) && at >= lo && at < hi;
              s[j][i] = ok ? s[j][i] : 0.0f;
            }
        }
        float big = 0.0f;
#pragma unroll
        for (int j = 0; j < kPages; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) big = fmaxf(big, __builtin_fabsf(s[j][i]));
        if (__builtin_amdgcn_ballot_w64(big > args.cap.lim)) {
#pragma unroll
          for (int j = 0; j < kPages; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = args.cap(s[j][i]);
        } else {
#pragma unroll
          for (int j = 0; j < kPages; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = args.cap.small(s[j][i]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kPages; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[j][i] *= a.scale_log2;
      }
    }
    // distance of token 4g of the step's first page
    const int left = st.n - st.pg * kPS;   // keys from the step's first on
    if constexpr (SCORE != 0) {
      if (args.slopes) {
#pragma unroll
        for (int j = 0; j < kPages; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[j][i] -= slope * (float)(left - 1 - 16 * j - 4 * g - i);
      }
    }
    if constexpr (REL) {
      // the bias as part of q.k, divided by the scale that follows
      if (left - 64 < a.rel_extent) {
        const float inv_scale = kLog2e / a.scale_log2;
        const int mis = (int)(((uintptr_t)a.rel +
                               (int64_t)st.b * a.HQ * a.rel_extent * 2) & 3);
        // o is even; the lane's bytes within the first dword: 0 or 2
        const int o0 = (hq * a.rel_extent + left - 1 - 4 * g - 3) * 2 + mis;
        const int sh = o0 & 2;
#pragma unroll
        for (int j = 0; j < kPages; ++j) {
          u32x3 y = x.bias[j];
          if (left <= 64) {
            // loaded from the resource's start instead of 1 or 2 dwords
            // before it (which hold no value of a key that is there)
            const int o = (o0 - 32 * j) & ~3;
            const uint32_t y0 = y[0], y1 = y[1];
            y[2] = o == -4 ? y1 : o == -8 ? y0 : y[2];
            y[1] = o == -4 ? y0 : y1;
          }
          const uint32_t z0 = __builtin_amdgcn_alignbyte(y[1], y[0], sh);
          const uint32_t z1 = __builtin_amdgcn_alignbyte(y[2], y[1], sh);
          const uint32_t b[4] = {z1 & 0xffff0000u, z1 << 16, z0 & 0xffff0000u,
                                 z0 << 16};
          const int d0 = left - 1 - 16 * j - 4 * g;
          if (left - 1 < a.rel_extent) {   // every key inside the band
#pragma unroll
            for (int i = 0; i < 4; ++i)
              s[j][i] += __builtin_bit_cast(float, b[i]) * inv_scale;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              s[j][i] += d0 - i < a.rel_extent
                             ? __builtin_bit_cast(float, b[i]) * inv_scale
                             : 0.0f;
          }
        }
      }
    }
    uint32_t vs[kPages];
#pragma unroll
    for (int j = 0; j < kPages; ++j) vs[j] = x.vs[j];
    if (!(st.flags & kFull)) {
      // keys that are not there, and the scales of their values: a row that
      // was never written may hold a NaN's scale, which weight zero keeps
      const int lo = vis_lo(st.n, a.window) - st.pg * kPS;
#pragma unroll
      for (int j = 0; j < kPages; ++j) {
        const bool have = st.flags & (kHave << j);
        uint32_t keep = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = 16 * j + 4 * g + i;
          const bool ok = have && at >= lo && at < left;
          s[j][i] = ok ? s[j][i] : -INFINITY;
          keep |= ok ? 0xffu << (8 * i) : 0u;
        }
        vs[j] &= keep;
      }
    }
    // ---- online softmax -----------------------------------------------------
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < kPages; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[j][i]);
    mx = lane_pair(lane_pair(mx, 16, true), 32, true);
    const float to_log2 = SCORE ? 1.0f : a.scale_log2;
    if constexpr (SCORE == 0) mx *= to_log2;
    const bool move = mx > m_run;
    if (__builtin_amdgcn_ballot_w64(move)) {
      const float m_new = move ? mx : m_run;
      const float alpha = move ? fast_exp2(m_run - m_new) : 1.0f;
      m_run = m_new;
      l_part *= alpha;
#pragma unroll
      for (int m = 0; m < 4; ++m) o_acc[m] = o_acc[m] * alpha;
    }
    const float m_use = m_run == -INFINITY ? 0.0f : m_run;
#pragma unroll
    for (int j = 0; j < kPages; ++j) {
      float p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i] = fast_exp2(SCORE ? s[j][i] - m_use
                               : __builtin_fmaf(s[j][i], to_log2, -m_use));
        l_part += p[i];
      }
      // each probability in the low or the high half of its dword
      uint32_t pw[4];
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const uint32_t two = pack_bf16x2_rn(p[i], p[i + 1]);
        pw[i] = __builtin_amdgcn_perm(two, 0u, p_sel0);
        pw[i + 1] = __builtin_amdgcn_perm(two, 0u, p_sel1);
      }
      const bf16x8 pf =
          __builtin_bit_cast(bf16x8, u32x4{pw[0], pw[1], pw[2], pw[3]});
      // ---- O^T += V^T.P^T ---------------------------------------------------
      // scale of token 4g + i: byte i moved to the exponent (the conversion
      // reads nothing else)
      const float sc[4] = {__builtin_bit_cast(float, vs[j] << 23),
                           __builtin_bit_cast(float, vs[j] << 15),
                           __builtin_bit_cast(float, vs[j] << 7),
                           __builtin_bit_cast(float, vs[j] >> 1)};
      u32x4 vf[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 y = dequantise8(x.v[j][i], sc[i]);
#pragma unroll
        for (int m = 0; m < 4; ++m) vf[m][i] = y[m];
      }
#pragma unroll
      for (int m = 0; m < 4; ++m)
        o_acc[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8, vf[m]), pf, o_acc[m], 0, 0, 0);
    }
  };

  // End of a piece: o_acc[m][i] of lane (n, g) is dim 32g + 8i + 2m + odd of
  // head n & 7. The two lanes of a head swap halves, so that each has both
  // dims of every pair for two of the four i (0, 1 for the even lane).
  auto finish = [&](const Step4& st) {
    float l_tot = lane_pair(lane_pair(l_part, 16, false), 32, false);
    // (no number as a sum: no number as LSE)
    const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
    const float lse = l_tot == 0.0f ? -INFINITY
                                    : (m_run + fast_log2(l_tot)) * kLn2;
    const bool whole = st.flags & kWhole;
    const int64_t slot = whole ? st.b : (int64_t)st.b + wg;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float y[8];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const float keep = odd ? o_acc[m][2 + j] : o_acc[m][j];
        const float give = odd ? o_acc[m][j] : o_acc[m][2 + j];
        const float got = other_half(give);
        y[2 * m] = (odd ? got : keep) * inv;
        y[2 * m + 1] = (odd ? keep : got) * inv;
      }
      if (!head_ok) continue;
      const int64_t at =
          (slot * a.HQ + hq) * kD + 32 * g + 8 * (2 * odd + j);
      if (whole) {
        *reinterpret_cast<u32x4*>(a.out + at) =
            u32x4{pack_bf16x2_rn(y[0], y[1]), pack_bf16x2_rn(y[2], y[3]),
                  pack_bf16x2_rn(y[4], y[5]), pack_bf16x2_rn(y[6], y[7])};
      } else {
        f32x4* const o = reinterpret_cast<f32x4*>(a.part_o + at);
        o[0] = f32x4{y[0], y[1], y[2], y[3]};
        o[1] = f32x4{y[4], y[5], y[6], y[7]};
      }
    }
    float* const to = whole ? a.lse : a.part_lse;
    if (head_ok && to && g == 0 && !odd) to[slot * a.HQ + hq] = lse;
#pragma unroll
    for (int m = 0; m < 4; ++m) o_acc[m] = f32x4{0, 0, 0, 0};
    m_run = -INFINITY;
    l_part = 0.0f;
  };

  // ---- the walk ---------------------------------------------------------------
  Buf4<REL> buf[2];
  Step4 cur, nx;
  int phys[kPages];
  next_step(cur, phys);
  load(buf[0], cur, phys);
  // the next step's loads, then this step; false: that was the last one
  auto turn = [&](Buf4<REL>& now, Buf4<REL>& then)
      __attribute__((always_inline)) {
    if (cur.flags & kFirst) {
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        qf[kk] = __builtin_bit_cast(bf16x8, q_next[kk]);
    }
    next_step(nx, phys);
    load(then, nx, phys);
    compute(now, cur);
    if (cur.flags & kLast) finish(cur);
    cur = nx;
    return cur.b >= 0;
  };
  while (turn(buf[0], buf[1]) && turn(buf[1], buf[0])) {
  }
}

// Ranges of the grid by default: four waves per compute unit, one per SIMD.
int default_wgs4(int hkv) {
  const int g = 4 * device_cus() / hkv;
  return g > 0 ? g : 1;
}

// query heads per wave: the largest divisor of the ratio up to 8
int rep4(int HQ, int HKV) {
  int rep = HQ / HKV;
  while (rep > kMaxRep || (HQ / HKV) % rep != 0) --rep;
  return rep;
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" size_t tmopt_attn_decode_mx4_workspace_size(int B, int HQ, int HKV,
                                                       int D,
                                                       int num_workgroups) {
  (void)D;
  if (B <= 0 || HQ <= 0 || HKV <= 0 || HQ % HKV != 0) return 0;
  const int G =
      num_workgroups > 0 ? num_workgroups : default_wgs4(HQ / rep4(HQ, HKV));
  return ws_layout(B, HQ, G, nullptr, nullptr);
}

extern "C" int tmopt_attn_decode_mx4(
    const void* q, const void* pool, const int32_t* block_table,
    int64_t bt_stride, int table_wrap, const int32_t* ctx_lens, int B, int HQ,
    int HKV, int D, int page_size, int64_t num_pages, int window, float scale,
    float softcap, const float* slopes, const void* rel, int rel_extent,
    int min_pages, int num_workgroups, void* out, float* lse, void* workspace,
    size_t workspace_bytes, tmopt_stream_t stream) {
  clear_error();
  if (B == 0) return TMOPT_OK;
  TMOPT_REQUIRE(B > 0, TMOPT_EINVAL, "decode_mx4: B=%d", B);
  TMOPT_REQUIRE(B <= kMaxB, TMOPT_EUNSUPPORTED, "decode_mx4: B=%d above %d", B,
                kMaxB);
  TMOPT_REQUIRE(q && pool && out && block_table && ctx_lens, TMOPT_EINVAL,
                "decode_mx4: null tensor pointer");
  TMOPT_REQUIRE(D == kD && page_size == kPS, TMOPT_EUNSUPPORTED,
                "decode_mx4: D=%d page_size=%d (only 128, 16)", D, page_size);
  TMOPT_REQUIRE(HKV > 0 && HQ > 0 && HQ % HKV == 0, TMOPT_EINVAL,
                "decode_mx4: HQ=%d HKV=%d", HQ, HKV);
  const int rep = rep4(HQ, HKV);
  const int hkv = HQ / rep;
  TMOPT_REQUIRE(HQ <= 131072 && hkv <= 65535, TMOPT_EUNSUPPORTED,
                "decode_mx4: HQ=%d in %d groups", HQ, hkv);
  TMOPT_REQUIRE(num_pages > 0 && bt_stride > 0 && table_wrap >= 0 &&
                    table_wrap <= bt_stride && window >= 0,
                TMOPT_EINVAL,
                "decode_mx4: num_pages=%lld bt_stride=%lld table_wrap=%d "
                "window=%d",
                (long long)num_pages, (long long)bt_stride, table_wrap, window);
  TMOPT_REQUIRE(table_wrap == 0 ||
                    (window > 0 && (int64_t)window <= (int64_t)table_wrap * kPS),
                TMOPT_EINVAL, "decode_mx4: window=%d outside a ring of %d pages",
                window, table_wrap);
  TMOPT_REQUIRE(scale > 0.0f && scale < INFINITY && good_cap(softcap, scale),
                TMOPT_EINVAL, "decode_mx4: scale=%g softcap=%g", scale,
                softcap);
  TMOPT_REQUIRE(min_pages > 0 && num_workgroups >= 0 && num_workgroups <= 65535,
                TMOPT_EINVAL, "decode_mx4: min_pages=%d num_workgroups=%d",
                min_pages, num_workgroups);
  TMOPT_REQUIRE(rel == nullptr ||
                    (rel_extent > 0 && (int64_t)HQ * rel_extent < (1 << 29) &&
                     scale >= kMinRaw),
                TMOPT_EINVAL, "decode_mx4: rel_extent=%d scale=%g", rel_extent,
                scale);
  TMOPT_REQUIRE(rel == nullptr || (softcap == 0.0f && slopes == nullptr),
                TMOPT_EUNSUPPORTED,
                "decode_mx4: a relative bias goes without softcap and slopes");
  TMOPT_REQUIRE(((uintptr_t)q | (uintptr_t)pool | (uintptr_t)out) % 16 == 0 &&
                    (uintptr_t)rel % 2 == 0,
                TMOPT_EINVAL, "decode_mx4: tensors must be 16-byte aligned");
  const int G = num_workgroups > 0 ? num_workgroups : default_wgs4(hkv);
  size_t off_lse = 0, off_geo = 0;
  const size_t need = ws_layout(B, HQ, G, &off_lse, &off_geo);
  TMOPT_REQUIRE(workspace && workspace_bytes >= need &&
                    (uintptr_t)workspace % 16 == 0,
                TMOPT_EWORKSPACE,
                "decode_mx4: workspace %zu bytes < %zu needed (or unaligned)",
                workspace_bytes, need);
  Mx4Args x{};
  DecodeArgs& a = x.d;
  a.q = (const __bf16*)q;
  a.bt = block_table;
  a.bt_stride = bt_stride;
  a.bt_width = bt_stride > 0x7fffffff ? 0x7fffffff : (int)bt_stride;
  a.table_wrap = table_wrap;
  a.ctx_lens = ctx_lens;
  a.B = B;
  a.HQ = HQ;
  a.HKV = hkv;
  a.rep = rep;
  a.kv_div = hkv / HKV;
  a.HKV_stored = HKV;
  a.num_pages = num_pages > 0x7fffffff ? 0x7fffffff : (int)num_pages;
  a.window = window;
  a.scale_log2 = scale * kLog2e;
  a.rel = (const __bf16*)rel;
  a.rel_extent = rel ? rel_extent : 0;
  a.min_pages = min_pages;
  a.out = (__bf16*)out;
  a.lse = lse;
  a.part_o = (float*)workspace;
  a.part_lse = (float*)((char*)workspace + off_lse);
  a.geo = (int*)((char*)workspace + off_geo);
  x.pool = (const uint8_t*)pool;
  x.cap = make_cap(softcap, scale);
  x.slopes = slopes;
  const int nw = waves_per_wg(hkv);
  a.ids_off = (int)(((2 * (size_t)B + 1 + 4) * sizeof(int) + 15) & ~(size_t)15);
  const size_t lds = a.ids_off + kIds4 * kPages * sizeof(int);
  const dim3 grid(G, hkv / nw);
  hipStream_t st = (hipStream_t)stream;
  if (rel)
    hipLaunchKernelGGL((decode_mx4_kernel<true, 0>), grid, dim3(64 * nw),
                       lds, st, x);
  else if (x.cap.k != 0.0f)
    hipLaunchKernelGGL((decode_mx4_kernel<false, 2>), grid, dim3(64 * nw), lds,
                       st, x);
  else if (softcap > 0.0f || slopes || scale > kMaxRaw)
    hipLaunchKernelGGL((decode_mx4_kernel<false, 1>), grid, dim3(64 * nw),
                       lds, st, x);
  else
    hipLaunchKernelGGL((decode_mx4_kernel<false, 0>), grid, dim3(64 * nw),
                       lds, st, x);
  const int rc = check_launch("decode_mx4");
  if (rc) return rc;
  launch_combine<true>(a, G, st);
  return check_launch("decode_mx4 merge");
}
