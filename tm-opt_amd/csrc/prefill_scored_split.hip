// Launches of the scored prefill with split keys (kernels: prefill_split.h).
#define TMOPT_PREFILL_SHORT_PIECES
#define TMOPT_PREFILL_SCORED
#include "prefill_split.h"

namespace tmopt {
namespace {

template <int REP>
void launch(const PrefillArgs& a, int src, size_t lds, hipStream_t st) {
  const dim3 grid((unsigned)(a.n_base * a.nsplit));
  // a cap alone and slopes alone have kernels of their own
  const bool raw = a.scale >= kMinRaw && a.scale <= kMaxRaw;
  const int kind = src | (a.cap.in == 0.0f ? (a.slopes && raw ? kSloped : 0)
                          : a.cap.near() && !a.slopes ? kCapped : 0);
#define TMOPT_LAUNCH(K)                                                     \
  case K:                                                                   \
    hipLaunchKernelGGL((prefill_split_kernel<REP, false, K>), grid, dim3(512), \
                       lds, st, a);                                         \
    break
  switch (kind) {
    TMOPT_LAUNCH(kPacked);
    TMOPT_LAUNCH(kPaged);
    TMOPT_LAUNCH(kPaged4);
    TMOPT_LAUNCH(kPacked | kCapped);
    TMOPT_LAUNCH(kPaged | kCapped);
    TMOPT_LAUNCH(kPaged4 | kCapped);
    TMOPT_LAUNCH(kPacked | kSloped);
    TMOPT_LAUNCH(kPaged | kSloped);
    TMOPT_LAUNCH(kPaged4 | kSloped);
  }
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
