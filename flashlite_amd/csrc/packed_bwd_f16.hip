// Gradients of attention over packed sequences, fp16: see packed_bwd.h.

#include "packed_bwd.h"

namespace fl {

hipError_t launch_packed_bwd_f16(const fl_packed_params& p, const fl_packed_grads& d, void* ws,
                                  hipStream_t stream) {
  return launch_bwd_type<_Float16>(p, d, ws, stream);
}

}  // namespace fl
