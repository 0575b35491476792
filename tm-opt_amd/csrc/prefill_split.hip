// Launches of the split prefill (kernels: prefill_split.h).
#include "prefill_split.h"

namespace tmopt {
namespace {

template <int REP, bool REL>
void launch_src(const PrefillArgs& a, int src, dim3 grid, size_t lds,
                hipStream_t st) {
  if (src == kPacked)
    hipLaunchKernelGGL((prefill_split_kernel<REP, REL, kPacked>), grid, dim3(512), lds, st,
                       a);
  else if (src == kPaged)
    hipLaunchKernelGGL((prefill_split_kernel<REP, REL, kPaged>), grid, dim3(512), lds, st,
                       a);
  else if (src == kMixed)
    hipLaunchKernelGGL((prefill_split_kernel<REP, REL, kMixed>), grid, dim3(512), lds, st,
                       a);
  else
    hipLaunchKernelGGL((prefill_split_kernel<REP, REL, kPackedCM>), grid, dim3(512), lds, st,
                       a);
}

template <int REP>
void launch(const PrefillArgs& a, int src, size_t lds, hipStream_t st) {
  const dim3 grid((unsigned)(a.n_base * a.nsplit));
  if (a.rel)
    launch_src<REP, true>(a, src, grid, lds, st);
  else
    launch_src<REP, false>(a, src, grid, lds, st);
  hipLaunchKernelGGL((prefill_merge_kernel<REP>), dim3(a.n_base, 8), dim3(256),
                     0, st, a);
}

}  // namespace

void launch_prefill_split(const PrefillArgs& a, int rep, int src, size_t lds,
                          hipStream_t st) {
  if (rep == 8)
    launch<8>(a, src, lds, st);
  else if (rep == 4)
    launch<4>(a, src, lds, st);
  else if (rep == 2)
    launch<2>(a, src, lds, st);
  else
    launch<1>(a, src, lds, st);
}

}  // namespace tmopt
