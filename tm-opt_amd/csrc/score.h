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
// each), less than a probability's rounding to bf16 for caps to 2^12.
struct Cap {
  float in;    // 2 log2(e) scale / cap; 0: no cap
  float out;   // cap log2(e)
  // up to |z| = cap / 2 also s (c0 + c1 s^2 + c2 s^4 + c3 s^6): five instructions
  // of one issue slot instead of eight slots
  float lim;   // the |s| up to which that holds
  float c0, c1, c2, c3;
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
  // The |s| up to which the score stays below x (0 if no |s| does, infinity if
  // every one): 2^(in s) = (1 + r) / (1 - r), r = x / out.
  __device__ __forceinline__ float reach(float x) const {
    if (x >= out) return INFINITY;
    return x <= 0.0f ? 0.0f : fast_log2((out + x) / (out - x)) / in;
  }
  // How far (in log2) the prefill sets a query's reference point above the largest
  // score it has seen: keys below 2^-102 of the sum may count as nothing.
  static constexpr float kLead = 24.0f;
  // caps that have a kernel of their own
  __host__ __device__ bool bounded() const {
    return in != 0.0f && out <= 77.0f;
  }
};

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
  // Minimax in s^2 of tanh(y) / y weighted by y over |y| <= 1/2: tanh is off by
  // 2^-22.9, 2^-21 with the roundings. (Outside these k its powers, or those of
  // s, leave fp32.)
  const double k = (double)scale / softcap;
  c.lim = k > 1e-4 && k < 1e2 ? (float)(0.5 / k) : -1.0f;
  const double a[4] = {0.999997676192731, -0.33320655218286016,
                       0.13145145657253834, -0.04337248369819732};
  double p = k * softcap * 1.4426950408889634;
  float* const to[4] = {&c.c0, &c.c1, &c.c2, &c.c3};
  for (int i = 0; i < 4; ++i, p *= k * k) *to[i] = (float)(a[i] * p);
  return c;
}

}  // namespace
}  // namespace tmopt
