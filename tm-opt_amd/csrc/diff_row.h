// One query row of one head pair by one work-group of 256 threads: 256 keys
// at a time, a key per thread for the scores, a dimension per thread for the
// values, with the running maximum and sum of both softmaxes (fp32 throughout).
#pragma once

#include "diff.h"

namespace tmopt {
namespace {

__device__ __forceinline__ float dot128(const __bf16* k, const float* q) {
  float s = 0.0f;
  for (int d = 0; d < kD; d += 8) {
    const bf16x8 x = *reinterpret_cast<const bf16x8*>(k + d);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += (float)x[i] * q[d + i];
  }
  return s;
}

// sum or maximum over the work-group, to every thread
__device__ __forceinline__ float wg_reduce(float x, bool want_max,
                                           float* red) {
  for (int m = 1; m < 64; m <<= 1) {
    const float y = __shfl_xor(x, m);
    x = want_max ? fmaxf(x, y) : x + y;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  const float a = want_max ? fmaxf(red[0], red[1]) : red[0] + red[1];
  const float b = want_max ? fmaxf(red[2], red[3]) : red[2] + red[3];
  return want_max ? fmaxf(a, b) : a + b;
}

// rows(pos, kr, vr): element offsets of the position's rows (head 0) in k / v;
// left at -1 where there is none. ABSENT: such a key is masked; otherwise it
// counts as a key and a value of zeros. Head strides ksh / vsh.
template <bool ABSENT, class Rows>
__device__ __forceinline__ void diff_row(const __bf16* q1, const __bf16* q2,
                                         const __bf16* k, int64_t ksh,
                                         const __bf16* v, int64_t vsh,
                                         Rows rows,
                                         int g, int lo, int hi, float scale,
                                         const DiffWeights& w, int h,
                                         bool rejected, __bf16* out,
                                         float* lse1, float* lse2) {
  __shared__ float qs[2][kD];
  __shared__ float p[2][256];
  __shared__ int64_t vrow[256];
  __shared__ float red[4];
  const int t = threadIdx.x;
  qs[t >> 7][t & 127] = (float)(t < 128 ? q1[t] : q2[t - 128]);
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0, 0}, acc[2] = {0, 0};
  __syncthreads();
  for (int k0 = lo; k0 < hi; k0 += 256) {
    const int pos = k0 + t;
    int64_t kr = -1, vr = -1;
    if (pos < hi) rows(pos, kr, vr);
    vrow[t] = vr;
    for (int i = 0; i < 2; ++i) {
      const float s = kr >= 0 ? dot128(k + kr + (2 * g + i) * ksh, qs[i]) *
                                    (scale * kLog2e)
                              : (ABSENT || pos >= hi ? -INFINITY : 0.0f);
      const float mx = fmaxf(m[i], wg_reduce(s, true, red));
      const float mu = mx == -INFINITY ? 0.0f : mx;
      const float e = fast_exp2(s - mu);
      const float keep = fast_exp2(m[i] - mu);
      p[i][t] = e;
      l[i] = l[i] * keep + wg_reduce(e, false, red);
      acc[i] *= keep;
      m[i] = mx;
    }
    __syncthreads();
    const int n = min(256, hi - k0);
    for (int j = 0; j < n; ++j) {
      if (vrow[j] < 0) continue;
      const float x = (float)v[vrow[j] + (2 * g + (t >> 7)) * vsh + (t & 127)];
      acc[0] += p[0][j] * x;
      acc[1] += p[1][j] * x;
    }
    __syncthreads();
  }
  float o = (l[0] > 0 ? acc[0] / l[0] : 0.0f) -
            w.lam[(int64_t)h * w.lam_stride] * (l[1] > 0 ? acc[1] / l[1] : 0.0f);
  if (!(l[0] > 0)) o = 0.0f;
  if (w.weight) {
    const float ss = wg_reduce(o * o, false, red);
    o = o * (1.0f / sqrtf(ss * (1.0f / kDV) + w.eps)) * w.weight[t];
  }
  o *= w.out_scale;
  if (rejected) o = __builtin_nanf("");
  out[t] = (__bf16)o;
  if (t < 2 && lse1) {
    const float x = l[t] > 0 ? (m[t] + fast_log2(l[t])) * kLn2 : -INFINITY;
    *(t == 0 ? lse1 : lse2) = rejected ? __builtin_nanf("") : x;
  }
}

}  // namespace
}  // namespace tmopt
