// The gated feed-forward block for float: see gated_calls.h.
#include "gated_calls.h"

namespace nest {

hipError_t gated_ffn_f32(const GatedParams& p, hipStream_t s, bool back) {
  return back ? gated_backward<float>(p, s) : gated_forward<float>(p, s);
}

}  // namespace nest
