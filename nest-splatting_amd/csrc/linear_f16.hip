// The dense layer for f16_t: see linear_calls.h.
#include "linear_calls.h"

namespace nest {

hipError_t linear_f16(const LinearParams& p, hipStream_t s, bool back) {
  return back ? linear_backward<f16_t>(p, s) : linear_forward<f16_t>(p, s);
}

}  // namespace nest
