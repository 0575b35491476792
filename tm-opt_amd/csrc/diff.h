// Differential attention: what its decode (decode_diff.hip) and its prefill
// (prefill_diff.hip) share.
//
// Query heads 2h and 2h + 1 are the two maps of head pair h; stored heads
// 2g and 2g + 1, g = h / (HQ / HKV), hold their keys, and side by side the
// pair's 256-wide values:
//
//   O_h = softmax(s q_2h K_2g^T) V_g - lam_h softmax(s q_2h+1 K_2g+1^T) V_g
//   out_h = O_h / sqrt(mean(O_h^2) + eps) * weight * out_scale
//
// (without a weight: out_h = O_h * out_scale). A query that sees no key has
// O_h = 0.
#pragma once

#include "common.h"

namespace tmopt {

constexpr int kD = 128;      // dims of a stored head
constexpr int kDV = 256;     // dims of a pair's values
constexpr int kPage = 16;    // tokens per page

// the learned weights of a launch and what follows the difference
struct DiffWeights {
  const float* lam;      // [HQ / 2], or one value (lam_stride 0)
  int lam_stride;
  const float* weight;   // [256] of the norm over a pair's output; NULL: none
  float eps;
  float out_scale;
};

// Checks shared by the entry points; 0 or a status with its message.
inline int check_diff(const char* what, int HQ, int HKV, int D, int window,
                      float scale, const float* lam, int lam_stride,
                      const float* weight, float eps) {
  TMOPT_REQUIRE(D == kD, TMOPT_EUNSUPPORTED, "%s: D=%d (only 128)", what, D);
  TMOPT_REQUIRE(HKV > 0 && HQ > 0 && HKV % 2 == 0 && HQ % HKV == 0,
                TMOPT_EINVAL,
                "%s: HQ=%d HKV=%d (HKV even, HQ a multiple of it)", what, HQ,
                HKV);
  TMOPT_REQUIRE((int64_t)kPage * HKV * kD * 2 < (1ll << 31) &&
                    HQ <= (1 << 17),
                TMOPT_EUNSUPPORTED, "%s: HQ=%d HKV=%d too large", what, HQ,
                HKV);
  TMOPT_REQUIRE(window >= 0, TMOPT_EINVAL, "%s: window=%d", what, window);
  TMOPT_REQUIRE(scale > 0.0f, TMOPT_EINVAL, "%s: scale must be > 0", what);
  TMOPT_REQUIRE(lam && (lam_stride == 0 || lam_stride == 1) &&
                    (uintptr_t)lam % 4 == 0,
                TMOPT_EINVAL, "%s: lam null, misaligned or of stride %d",
                what, lam_stride);
  TMOPT_REQUIRE(!weight || (eps > 0.0f && (uintptr_t)weight % 16 == 0),
                TMOPT_EINVAL,
                "%s: the norm needs eps > 0 and a 16-byte aligned weight",
                what);
  return TMOPT_OK;
}

}  // namespace tmopt
