// The 4-bit cache: blocks of 32 values with one power-of-two scale.
//
// A token's head is 128 values, four blocks of 32 dims. A block keeps one byte,
// its scale 2^(E - 127), and 32 e2m1 elements (sign, 2 exponent bits, 1
// mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6), the nearest of value / scale, ties
// to the even code. The scale is the smallest power of two under which the
// block's largest magnitude is at most 7: it then rounds to 6 or is cut to it,
// and no value is off by more than the scale, half of the largest step.
// (6 instead of 7 would double the scale of every block whose largest value
// lies between: all its values then lose a bit.) E = 255: the block holds a
// value that is no number, infinite, or above 7 * 2^125; it reads as NaN.
//
// Pages are records of 2176 bytes per page and KV head, [num_pages, HKV, 2176]:
//      0  K elements   [16 tokens][64]: dims 2i, 2i + 1 in the low and the high
//                      half of byte i
//   1024  V elements   [16 dim groups][16 tokens][4]: group c = dims 8c..8c+7
//   2048  K scales     [4 blocks][16 tokens]
//   2112  V scales     [4 blocks][16 tokens]
// One head's part of a page is contiguous (17 cache lines), so a wave streams
// it by itself, and lane (r, g) = (lane & 15, lane >> 4) finds its MFMA operands
// at byte 64 r + 16 g of either half without any exchange: of K the block g of
// token r, of V the dims 8r..8r+7 of tokens 4g..4g+3. A new token touches bytes
// of its own only (V's bytes hold two dims of one token, so rows are written
// without reading what is there).
#pragma once

#include "common.h"

namespace tmopt {
namespace {

constexpr int kRecB = 2176;
constexpr int kRecV = 1024, kRecKs = 2048, kRecVs = 2112;
constexpr int kMinE = 2, kMaxE = 252, kNanE = 255;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Scale byte of a block whose largest magnitude has bf16 bits `amax` (an
// integer compare orders magnitudes, infinities and NaN last): 1.f * 2^x gives
// 2^(x - 2) up to 1.75 * 2^x = 7 * 2^(x - 2), else 2^(x - 1).
__device__ __forceinline__ int block_scale(uint32_t amax) {
  const int e = (int)((amax + 0x1f) >> 7) - 2;
  return e > kMaxE ? kNanE : max(e, kMinE);
}

__device__ __forceinline__ float scale_f32(uint32_t e) {
  return __builtin_bit_cast(float, e << 23);
}

// Eight bf16 -> eight elements (v_cvt_scalef32_pk_fp4_bf16: nearest, ties to
// even, cut to 6; checked for every bf16 value).
__device__ __forceinline__ uint32_t quantise8(u32x4 x, float scale) {
  uint32_t r = 0;
  const uint32_t x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      r, __builtin_bit_cast(bf16x2, x0), scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      r, __builtin_bit_cast(bf16x2, x1), scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      r, __builtin_bit_cast(bf16x2, x2), scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(
      r, __builtin_bit_cast(bf16x2, x3), scale, 3);
  return r;
}

// Elements 2 SEL, 2 SEL + 1 of a dword of eight, times the scale's power of two
// (its sign and mantissa are not read; exponent 255 gives NaN): two bf16,
// exact down to 2^-126.
template <int SEL>
__device__ __forceinline__ uint32_t dequantise2(uint32_t x, float scale) {
  return __builtin_bit_cast(
      uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(x, scale, SEL));
}
__device__ __forceinline__ u32x4 dequantise8(uint32_t x, float scale) {
  return u32x4{dequantise2<0>(x, scale), dequantise2<1>(x, scale),
               dequantise2<2>(x, scale), dequantise2<3>(x, scale)};
}

}  // namespace
}  // namespace tmopt
