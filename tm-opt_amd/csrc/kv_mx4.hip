// Rows into the 4-bit cache and back (format: mx4.h).
//
// A wave takes 16 consecutive tokens of one KV head, K and V: lane (t, c4) =
// (lane & 15, lane >> 4) holds 16-byte chunks c4, c4 + 4, c4 + 8, c4 + 12 of
// token t's row (dims 8c..8c+7), so a block's largest value is a maximum over
// the lanes t, t + 16, t + 32, t + 48 and one chunk each, and consecutive tokens
// of a page fill whole 64-byte lines of V's transposed elements. All eight loads
// of a lane are out before the first is used.
//
// What bounds them: small calls the launch (64 rows of 4 heads 3.7 us each),
// large ones HBM: 12,001 rows of 8 heads, parts of a fused projection's, 12.6 us
// in (49 MB read, 13 written) and 14.7 out (13 read, 49 written).
#include "mx4.h"

namespace tmopt {
namespace {

constexpr int kPS = 16, kD = 128;

struct Mx4Rows {
  const __bf16* k;
  const __bf16* v;
  int64_t k_st, k_sh, v_st, v_sh;
  const int64_t* slots;
  int64_t T, pool_rows;
  int HKV;
  uint8_t* pool;
  __bf16* k_out;   // [T, HKV, 128] of the way back
  __bf16* v_out;
};

// the larger of a lane pair's values (see lane_pair in common.h)
__device__ __forceinline__ uint32_t pair_max(uint32_t x, int dist) {
  const auto r = dist == 16
                     ? __builtin_amdgcn_permlane16_swap(x, x, false, false)
                     : __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max((uint32_t)r[0], (uint32_t)r[1]);
}

// Quantise the lane's four chunks of a row into its record: elements at
// el + c * el_step, the block's scale byte at sc + 16 block.
__device__ __forceinline__ void put_row(const u32x4 (&x)[4], bool ok, int c4,
                                        uint8_t* el, int el_step,
                                        uint8_t* sc) {
  int mine = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = x[j][i];
      m = max(m, max(w & 0x7fffu, w >> 16 & 0x7fffu));
    }
    const int e = block_scale(pair_max(pair_max(m, 16), 32));
    const uint32_t q = e == kNanE ? 0u : quantise8(x[j], scale_f32(e));
    if (ok) *reinterpret_cast<uint32_t*>(el + (4 * j + c4) * el_step) = q;
    mine = j == c4 ? e : mine;
  }
  if (ok) sc[16 * c4] = (uint8_t)mine;
}

__global__ __launch_bounds__(256) void write_mx4_kernel(Mx4Rows a) {
  const int lane = threadIdx.x & 63;
  const int64_t gw = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int h = (int)(gw % a.HKV);
  const int64_t t0 = gw / a.HKV * kPS;
  if (t0 >= a.T) return;
  const int c4 = lane >> 4;
  const int64_t t = min(t0 + (lane & 15), a.T - 1);
  const int64_t row = a.slots[t];
  const bool ok = t0 + (lane & 15) < a.T && row >= 0 && row < a.pool_rows;
  const u32x4* ks = reinterpret_cast<const u32x4*>(a.k + t * a.k_st + h * a.k_sh);
  const u32x4* vs = reinterpret_cast<const u32x4*>(a.v + t * a.v_st + h * a.v_sh);
  u32x4 k[4], v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) k[j] = ks[4 * j + c4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = vs[4 * j + c4];
  const int off = (int)(row & (kPS - 1));
  uint8_t* const rec =
      a.pool + ((ok ? row / kPS : 0) * a.HKV + h) * (int64_t)kRecB;
  put_row(k, ok, c4, rec + off * 64, 4, rec + kRecKs + off);
  put_row(v, ok, c4, rec + kRecV + off * 4, 64, rec + kRecVs + off);
}

__device__ __forceinline__ void get_row(u32x4 (&x)[4], bool ok, int c4,
                                        const uint8_t* el, int el_step,
                                        const uint8_t* sc) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t q =
        *reinterpret_cast<const uint32_t*>(el + (4 * j + c4) * el_step);
    x[j] = dequantise8(ok ? q : 0u, scale_f32(ok ? sc[16 * j] : kMinE));
  }
}

__global__ __launch_bounds__(256) void read_mx4_kernel(Mx4Rows a) {
  const int lane = threadIdx.x & 63;
  const int64_t gw = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int h = (int)(gw % a.HKV);
  const int64_t t = gw / a.HKV * kPS + (lane & 15);
  if (t >= a.T) return;
  const int c4 = lane >> 4;
  const int64_t row = a.slots[t];
  const bool ok = row >= 0 && row < a.pool_rows;
  const int off = ok ? (int)(row & (kPS - 1)) : 0;
  const uint8_t* const rec =
      a.pool + ((ok ? row / kPS : 0) * a.HKV + h) * (int64_t)kRecB;
  u32x4 k[4], v[4];
  get_row(k, ok, c4, rec + off * 64, 4, rec + kRecKs + off);
  get_row(v, ok, c4, rec + kRecV + off * 4, 64, rec + kRecVs + off);
  const int64_t at = (t * a.HKV + h) * kD;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    reinterpret_cast<u32x4*>(a.k_out + at)[4 * j + c4] = k[j];
    reinterpret_cast<u32x4*>(a.v_out + at)[4 * j + c4] = v[j];
  }
}

int check_rows(const char* what, const int64_t* slots, int64_t T, int HKV,
               int D, int page_size, const void* pool, int64_t num_pages) {
  TMOPT_REQUIRE(T >= 0 && HKV > 0 && slots && pool, TMOPT_EINVAL,
                "%s: T=%lld HKV=%d or null pointer", what, (long long)T, HKV);
  TMOPT_REQUIRE(D == kD && page_size == kPS, TMOPT_EUNSUPPORTED,
                "%s: D=%d page_size=%d (only 128, 16)", what, D, page_size);
  TMOPT_REQUIRE(num_pages > 0 && num_pages <= 0x7fffffff, TMOPT_EINVAL,
                "%s: num_pages=%lld", what, (long long)num_pages);
  TMOPT_REQUIRE((uintptr_t)pool % 16 == 0, TMOPT_EINVAL,
                "%s: the pool must be 16-byte aligned", what);
  TMOPT_REQUIRE(HKV <= 65535 && (T + 15) / 16 * HKV < (1ll << 31),
                TMOPT_EUNSUPPORTED, "%s: T=%lld HKV=%d", what, (long long)T,
                HKV);
  return TMOPT_OK;
}

dim3 rows_grid(int64_t T, int HKV) {
  return dim3((unsigned)(((T + 15) / 16 * HKV + 3) / 4));
}

}  // namespace
}  // namespace tmopt

using namespace tmopt;

extern "C" int tmopt_kv_write_mx4(const void* k, const void* v,
                                  int64_t k_stride_tok, int64_t k_stride_head,
                                  int64_t v_stride_tok, int64_t v_stride_head,
                                  const int64_t* slot_mapping, int64_t T,
                                  int HKV, int D, int page_size, void* pool,
                                  int64_t num_pages, tmopt_stream_t stream) {
  clear_error();
  if (T == 0) return TMOPT_OK;
  const int rc = check_rows("kv_write_mx4", slot_mapping, T, HKV, D, page_size,
                            pool, num_pages);
  if (rc) return rc;
  TMOPT_REQUIRE(k && v && ((uintptr_t)k | (uintptr_t)v) % 16 == 0 &&
                    k_stride_tok % 8 == 0 && k_stride_head % 8 == 0 &&
                    v_stride_tok % 8 == 0 && v_stride_head % 8 == 0,
                TMOPT_EINVAL,
                "kv_write_mx4: k/v null or rows not 16-byte aligned "
                "(strides %% 8)");
  Mx4Rows a{(const __bf16*)k, (const __bf16*)v, k_stride_tok, k_stride_head,
            v_stride_tok, v_stride_head, slot_mapping, T, num_pages * kPS, HKV,
            (uint8_t*)pool, nullptr, nullptr};
  hipLaunchKernelGGL(write_mx4_kernel, rows_grid(T, HKV), dim3(256), 0,
                     (hipStream_t)stream, a);
  return check_launch("kv_write_mx4");
}

extern "C" int tmopt_kv_read_mx4(const void* pool, int64_t num_pages,
                                 const int64_t* slot_mapping, int64_t T,
                                 int HKV, int D, int page_size, void* k,
                                 void* v, tmopt_stream_t stream) {
  clear_error();
  if (T == 0) return TMOPT_OK;
  const int rc = check_rows("kv_read_mx4", slot_mapping, T, HKV, D, page_size,
                            pool, num_pages);
  if (rc) return rc;
  TMOPT_REQUIRE(k && v && ((uintptr_t)k | (uintptr_t)v) % 16 == 0,
                TMOPT_EINVAL, "kv_read_mx4: k/v null or not 16-byte aligned");
  Mx4Rows a{nullptr, nullptr, 0, 0, 0, 0, slot_mapping, T, num_pages * kPS,
            HKV, (uint8_t*)const_cast<void*>(pool), (__bf16*)k, (__bf16*)v};
  hipLaunchKernelGGL(read_mx4_kernel, rows_grid(T, HKV), dim3(256), 0,
                     (hipStream_t)stream, a);
  return check_launch("kv_read_mx4");
}
