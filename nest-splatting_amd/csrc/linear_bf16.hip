// The dense layer for bf16_t: see linear_calls.h.
#include "linear_calls.h"

namespace nest {

hipError_t linear_bf16(const LinearParams& p, hipStream_t s, bool back) {
  return back ? linear_backward<bf16_t>(p, s) : linear_forward<bf16_t>(p, s);
}

}  // namespace nest
