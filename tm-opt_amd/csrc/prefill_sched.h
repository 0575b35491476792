// The order of a prefill's work items (KV head, run, block of queries) on its
// grid. A is the launch's arguments: S runs, cu [S + 1], prior [S] or null, HKV
// KV heads as scheduled, nqb_max blocks of the longest run.
#pragma once

#include "common.h"

namespace tmopt {
namespace {

// Sum over the wave, wave-uniform: within each 16-lane row by DPP (xor 1,
// xor 2, half-row mirror, row mirror: a few cycles each), then the four row
// sums by lane reads. (The schedule below takes ~10 of these per
// work-group; as ds_bpermute shuffles, 6 LDS round trips each, they cost
// microseconds of every work-group's start.)
__device__ __forceinline__ int wave_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);   // xor 1
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);   // xor 2
  v += __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);  // 7 - i
  v += __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false);  // 15 - i
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) +
         __builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48);
}

// query blocks of run s (lane-varying s)
template <class A>
__device__ __forceinline__ int run_blocks(const A& a, int s, int BQ) {
  const int len = a.cu[s + 1] - a.cu[s];
  return (len + BQ - 1) / BQ;
}

// items of one KV head in levels [0, z): a run with nb blocks has one item
// on each level z' >= nqb_max - nb. nb0: blocks of run `lane` (0 past S).
template <class A>
__device__ __forceinline__ int items_before(const A& a, int z, int BQ,
                                            int lane, int nb0) {
  int c = max(0, nb0 - a.nqb_max + z);
  for (int s = lane + 64; s < a.S; s += 64)
    c += max(0, run_blocks(a, s, BQ) - a.nqb_max + z);
  return __builtin_amdgcn_readfirstlane(wave_sum(c));
}

struct Work {
  int kvh, seq, qb;    // seq < 0: nothing to do
  int t0, len, prior;  // the run's first row, length and prior context
  int total;           // cu[S]: rows of the launch (the LSE row length)
};

// Work item of this work-group (computed by every wave, identically).
// Work-group L runs on XCD L % 8 as the L/8-th one there. KV heads are
// spread over the XCDs (8 % HKV == 0: 8/HKV XCDs per head; HKV % 8 == 0:
// HKV/8 heads per XCD; otherwise round robin), and each head's items, in
// level order, are dealt to its XCDs in turn.
template <class A>
__device__ __forceinline__ Work schedule(const A& a, int BQ, int lane,
                                         int L) {
  int kvh, i;
  if (a.HKV <= 8 && 8 % a.HKV == 0) {
    const int R = 8 / a.HKV;
    kvh = (L & 7) / R;
    i = (L >> 3) * R + (L & 7) % R;
  } else if (a.HKV % 8 == 0) {
    const int R = a.HKV / 8;
    kvh = (L & 7) + 8 * ((L >> 3) % R);
    i = (L >> 3) / R;
  } else {
    kvh = L % a.HKV;
    i = L / a.HKV;
  }
  Work w{kvh, -1, 0, 0, 0, 0, 0};
  // row start, end and prior context of the first 64 runs, one per lane:
  // the item's own values are then lane reads, not a second round trip to
  // memory after the search
  const int c0 = lane < a.S ? a.cu[lane] : 0;
  const int c1 = lane < a.S ? a.cu[lane + 1] : 0;
  const int p0 = a.prior != nullptr && lane < a.S ? a.prior[lane] : 0;
  const int nb0 = (c1 - c0 + BQ - 1) / BQ;
  const int total = items_before(a, a.nqb_max, BQ, lane, nb0);
  if (i >= total) return w;
  // level z: the last one with items_before(z) <= i
  int lo = 0, hi = a.nqb_max;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (items_before(a, mid, BQ, lane, nb0) <= i) lo = mid; else hi = mid;
  }
  int rem = i - items_before(a, lo, BQ, lane, nb0);
  const int need = a.nqb_max - lo;  // runs with at least this many blocks
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    const int s = s0 + lane;
    const bool act =
        s < a.S && (s0 == 0 ? nb0 : run_blocks(a, s, BQ)) >= need;
    const uint64_t m = __builtin_amdgcn_ballot_w64(act);
    const int pop = __builtin_popcountll(m);
    if (rem < pop) {
      const int rank = __builtin_amdgcn_mbcnt_hi(
          (uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
      const uint64_t hit = __builtin_amdgcn_ballot_w64(act && rank == rem);
      const int sl = __builtin_ctzll(hit);
      w.seq = s0 + sl;
      w.qb = a.nqb_max - 1 - lo;
      if (s0 == 0) {
        w.t0 = __builtin_amdgcn_readlane(c0, sl);
        w.len = __builtin_amdgcn_readlane(c1, sl) - w.t0;
        w.prior = __builtin_amdgcn_readlane(p0, sl);
      } else {
        w.t0 = as_const(a.cu)[w.seq];
        w.len = as_const(a.cu)[w.seq + 1] - w.t0;
        w.prior = a.prior != nullptr ? as_const(a.prior)[w.seq] : 0;
      }
      w.total = a.S <= 64 ? __builtin_amdgcn_readlane(c1, a.S - 1)
                          : as_const(a.cu)[a.S];
      return w;
    }
    rem -= pop;
  }
  return w;  // not reached for i < total
}

}  // namespace
}  // namespace tmopt
