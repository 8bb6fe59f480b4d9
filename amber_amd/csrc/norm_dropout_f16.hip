// The row and elementwise kernels of norm_dropout.h for one element type (a translation unit each: they compile side by side).
#include "norm_dropout.h"

namespace amber {
hipError_t tail_forward_f16(const TailArgs& a, bool normalize, hipStream_t s) { return tail_forward_t<f16>(a, normalize, s); }
hipError_t tail_backward_f16(const TailArgs& a, bool normalize, hipStream_t s) { return tail_backward_t<f16>(a, normalize, s); }
}  // namespace amber
