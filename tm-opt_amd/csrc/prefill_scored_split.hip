// Launches of the scored prefill with split keys (kernels: prefill_split.h).
#define TMOPT_PREFILL_SHORT_PIECES
#define TMOPT_PREFILL_SCORED
#include "prefill_split.h"

namespace tmopt {
namespace {

template <int REP>
void launch(const PrefillArgs& a, int src, size_t lds, hipStream_t st) {
  const dim3 grid((unsigned)(a.n_base * a.nsplit));
#define TMOPT_LAUNCH(K)                                                        \
  case K:                                                                      \
    hipLaunchKernelGGL((prefill_split_kernel<REP, false, K>), grid, dim3(512), \
                       lds, st, a);                                            \
    break;
  switch (scored_kind(a, src)) { TMOPT_SCORED_KINDS(TMOPT_LAUNCH) }
#undef TMOPT_LAUNCH
  hipLaunchKernelGGL((prefill_merge_kernel<REP, true>), dim3(a.n_base, 8),
                     dim3(256), 0, st, a);
}

}  // namespace

void launch_prefill_scored_split(const PrefillArgs& a, int rep, int src,
                                 size_t lds, hipStream_t st) {
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
