// Paged prefill attention over the fp16 and the 8-bit pool: the forms of the kernel in
// pa_prefill_kernel.h with plain scores.
#include "pa_prefill_kernel.h"

namespace pa {

hipError_t launch_prefill_attn(const PrefillAttnArgs& a, int D, hipStream_t s) {
  return a.ks ? launch_prefill<true, 0>(a, D, s) : launch_prefill<false, 0>(a, D, s);
}

}  // namespace pa
