// The dense layer for float: see linear_calls.h.
#include "linear_calls.h"

namespace nest {

hipError_t linear_f32(const LinearParams& p, hipStream_t s, bool back) {
  return back ? linear_backward<float>(p, s) : linear_forward<float>(p, s);
}

}  // namespace nest
