// Launches of the prefill over the 4-bit cache, without score functions
// (those: prefill_scored.hip), with and without the relative bias.
#include "prefill_kernel.h"

namespace tmopt {
namespace {

template <int REP>
void launch(const PrefillArgs& a, size_t lds, hipStream_t st) {
  const dim3 grid((unsigned)a.n_base);
  if (a.rel)
    hipLaunchKernelGGL((prefill_kernel<REP, true, kPaged4>), grid,
                       dim3(512), lds, st, a);
  else
    hipLaunchKernelGGL((prefill_kernel<REP, false, kPaged4>), grid,
                       dim3(512), lds, st, a);
}

}  // namespace

void launch_prefill_mx4(const PrefillArgs& a, int rep, size_t lds,
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
