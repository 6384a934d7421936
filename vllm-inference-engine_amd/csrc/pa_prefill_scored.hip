// Paged prefill attention with capped, biased and masked scores: the forms of the kernel in
// pa_prefill_kernel.h that differ in what they add to a score. (A bias of 0 costs two
// instructions a score: windows and intervals without a cap take that form.)
#include "pa_prefill_kernel.h"

namespace pa {

hipError_t launch_prefill_scored(const PrefillScoredArgs& a, int D, hipStream_t s) {
  if (a.cap_log2 == 0.f) return launch_prefill<false, kScoreBias>(a, D, s);
  if (a.cap_t != 0.f) return launch_prefill<false, kScoreWideCapBias>(a, D, s);
  return a.slopes ? launch_prefill<false, kScoreCapBias>(a, D, s)
                  : launch_prefill<false, kScoreCap>(a, D, s);
}

}  // namespace pa
