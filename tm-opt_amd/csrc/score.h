// Score functions of the scored and of the 4-bit attention: what comes between
// q.k and the softmax, and which keys a query sees.
//
//   z = scale q.k;  x = softcap tanh(z / softcap)  (softcap 0: x = z)
//   x -= slope_h |pos_q - pos_k|                   (slopes given)
#pragma once

#include "common.h"

namespace tmopt {
namespace {

// cap tanh(z / cap), in units of log2(e), of s = q.k. With t = exp(2 z / cap) it
// is cap (1 - 2 / (1 + t)), whatever the sign; t = 0 and infinity give -cap and
// cap. fp32 throughout: 1 - 2 / (1 + t) is off by 5.5 x 2^-23 at most (t by
// 2^-23 of itself, the sum, the reciprocal and the difference by a rounding
// each), 2^-11 for caps up to kNear, an eighth of a probability's rounding to bf16.
// Above that the exponential form alone would lose the scores that are far below
// the cap (by 1 at a cap of 10^6): far() takes the polynomial for each of these.
//
// Minimax in y^2 of tanh(y) / y weighted by y over |y| <= 1/2: tanh is off by
// 2^-22.9, 2^-21 with the roundings, and by 2^-18.7 of y where that is less.
constexpr double kTanh[4] = {0.999997676192731, -0.33320655218286016,
                             0.13145145657253834, -0.04337248369819732};
struct Cap {
  static constexpr float kNear = 256.0f;
  float in;    // 2 log2(e) scale / cap; 0: no cap
  float out;   // cap log2(e)
  // up to |z| = cap / 2 also s (c0 + c1 s^2 + c2 s^4 + c3 s^6): five instructions
  // of one issue slot instead of eight slots
  float lim;   // the |s| up to which that holds
  float c0, c1, c2, c3;
  float k;     // caps above kNear: scale / cap; 0 for others
  __device__ __forceinline__ float operator()(float s) const {
    return out - 2.0f * out *
                     __builtin_amdgcn_rcpf(1.0f + fast_exp2(s * in));
  }
  __device__ __forceinline__ float small(float s) const {
    const float u = s * s;
    return s * __builtin_fmaf(
                   __builtin_fmaf(__builtin_fmaf(c3, u, c2), u, c1), u, c0);
  }
  // the same less m
  __device__ __forceinline__ float less(float s, float m) const {
    return (out - m) - 2.0f * out *
                           __builtin_amdgcn_rcpf(1.0f + fast_exp2(s * in));
  }
  __device__ __forceinline__ float small_less(float s, float m) const {
    const float u = s * s;
    return __builtin_fmaf(
        s,
        __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(c3, u, c2), u, c1), u, c0),
        -m);
  }
  // caps above kNear: y = z / cap up to 1/2 by the polynomial in y (whose powers
  // stay in fp32 whatever the cap), off by 2^-18 of z at most, as cap 2^-20 is
  // beyond
  __device__ __forceinline__ float far(float s) const {
    const float y = s * k, u = y * y;
    const float p =
        y * __builtin_fmaf(
                __builtin_fmaf(__builtin_fmaf((float)kTanh[3], u,
                                              (float)kTanh[2]),
                               u, (float)kTanh[1]),
                u, (float)kTanh[0]);
    const float e =
        1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + fast_exp2(s * in));
    return out * (__builtin_fabsf(y) <= 0.5f ? p : e);
  }
  // The |s| up to which the score stays below x (0 if no |s| does, infinity if
  // every one): 2^(in s) = (1 + r) / (1 - r), r = x / out.
  __device__ __forceinline__ float reach(float x) const {
    if (x >= out) return INFINITY;
    return x <= 0.0f ? 0.0f : fast_log2((out + x) / (out - x)) / in;
  }
  // How far (in log2) the prefill sets a query's reference point above the largest
  // score it has seen: keys below 2^-86 of the sum may count as nothing, and so may
  // products with values below 2^-86. (24 / 32 / 40 / 48, us: a chunk of 1,500 in
  // documents 94.6 / 92.0 / 91.0 / 91.0, where a query's first tile may show it a few
  // keys only; 4 prompts of 2K-8K 1,103 / 1,095 / 1,096 / 1,096.)
  static constexpr float kLead = 40.0f;
  // The prefill has kernels of its own for a cap up to kNear without slopes (4
  // prompts of 2K-8K with a cap of 60: 1,066 us there, 1,194 with the running
  // maximum and the exponential form that caps with slopes take).
  __host__ __device__ bool near() const { return in != 0.0f && k == 0.0f; }
};

// Scales for which a score may stay q.k up to the exponent, whose argument is then
// one fma of it and the rounded maximum: off by half a step of |x|, which passes
// fp32's exponents from |x| = 2^31 on. Above kMaxRaw scores are scaled first. A bias
// that joins q.k divided by the scale would leave fp32 below kMinRaw.
constexpr float kMinRaw = 0x1p-60f, kMaxRaw = 256.0f;

// A cap that fp32 can work with: 0, or 2 log2(e) scale / softcap in its range.
inline bool good_cap(float softcap, float scale) {
  return softcap == 0.0f || (softcap > 0.0f && softcap < INFINITY &&
                             scale / softcap < 1e37f && scale / softcap > 1e-37f);
}

inline Cap make_cap(float softcap, float scale) {
  Cap c{};
  if (!(softcap > 0.0f)) return c;
  c.in = 2.0f * kLog2e * scale / softcap;
  c.out = softcap * kLog2e;
  const double k = (double)scale / softcap;
  if (softcap > Cap::kNear) {
    c.k = (float)k;
    c.lim = -1.0f;
    return c;
  }
  double p = (double)scale * 1.4426950408889634;
  float* const to[4] = {&c.c0, &c.c1, &c.c2, &c.c3};
  for (int i = 0; i < 4; ++i, p *= k * k) *to[i] = (float)(kTanh[i] * p);
  // (outside this range the powers of k, or those of s up to 1 / 2k, leave fp32)
  const bool fits = k < 1e2 && c.c3 < -1e-36f;
  c.lim = fits ? (float)(0.5 / k) : -1.0f;
  return c;
}

}  // namespace
}  // namespace tmopt
