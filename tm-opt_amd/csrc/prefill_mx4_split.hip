// Launches of the prefill over the 4-bit cache with split
// keys (prefill_split.h), without score functions
// (those: prefill_scored_split.hip), with and without the relative bias.
#define TMOPT_PREFILL_SHORT_PIECES
#include "prefill_split.h"

namespace tmopt {
namespace {

template <int REP>
void launch(const PrefillArgs& a, size_t lds, hipStream_t st) {
  const dim3 grid((unsigned)(a.n_base * a.nsplit));
  if (a.rel)
    hipLaunchKernelGGL((prefill_split_kernel<REP, true, kPaged4>), grid,
                       dim3(512), lds, st, a);
  else
    hipLaunchKernelGGL((prefill_split_kernel<REP, false, kPaged4>), grid,
                       dim3(512), lds, st, a);
  hipLaunchKernelGGL((prefill_merge_kernel<REP, true>), dim3(a.n_base, 8),
                     dim3(256), 0, st, a);
}

}  // namespace

void launch_prefill_mx4_split(const PrefillArgs& a, int rep, size_t lds,
                              hipStream_t st) {
  if (rep == 8)
    launch<8>(a, lds, st);
  else if (rep == 4)
    launch<4>(a, lds, st);
  else if (rep == 2)
    launch<2>(a, lds, st);
  else
    launch<1>(a, lds, st);
}

}  // namespace tmopt
