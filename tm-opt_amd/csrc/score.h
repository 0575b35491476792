// Score functions of the scored and of the 4-bit attention: what comes between
// q.k and the softmax, and which keys a query sees.
//
//   z = scale q.k;  x = softcap tanh(z / softcap)  (softcap 0: x = z)
//   x -= slope_h |pos_q - pos_k|                   (slopes given)
#pragma once

#include "common.h"

namespace tmopt {
namespace {

// tanh(z / cap) cap, in units of log2(e), of s = q.k: with t = exp(2 z / cap) it
// is cap (1 - 2 / (1 + t)), whatever the sign; t = 0 and infinity give -cap and
// cap. fp32 throughout: near zero, where 1 - 2 / (1 + t) cancels, the result is
// off by 2^-23 cap, less than a probability's rounding to bf16 for caps to 2^14.
struct Cap {
  float in;    // 2 log2(e) scale / cap; 0: no cap
  float out;   // cap log2(e)
  __device__ __forceinline__ float operator()(float s) const {
    return out - 2.0f * out *
                     __builtin_amdgcn_rcpf(1.0f + fast_exp2(s * in));
  }
};

inline Cap make_cap(float softcap, float scale) {
  return softcap > 0.0f ? Cap{2.0f * kLog2e * scale / softcap,
                              softcap * kLog2e}
                        : Cap{0.0f, 0.0f};
}

}  // namespace
}  // namespace tmopt
