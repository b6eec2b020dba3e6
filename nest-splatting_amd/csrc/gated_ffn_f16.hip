// The gated feed-forward block for f16_t: see gated_calls.h.
#include "gated_calls.h"

namespace nest {

hipError_t gated_ffn_f16(const GatedParams& p, hipStream_t s, bool back) {
  return back ? gated_backward<f16_t>(p, s) : gated_forward<f16_t>(p, s);
}

}  // namespace nest
