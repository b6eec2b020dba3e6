// The gated feed-forward block for bf16_t: see gated_calls.h.
#include "gated_calls.h"

namespace nest {

hipError_t gated_ffn_bf16(const GatedParams& p, hipStream_t s, bool back) {
  return back ? gated_backward<bf16_t>(p, s) : gated_forward<bf16_t>(p, s);
}

}  // namespace nest
