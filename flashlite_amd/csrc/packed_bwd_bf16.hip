// Gradients of attention over packed sequences, bf16: see packed_bwd.h.

#include "packed_bwd.h"

namespace fl {

hipError_t launch_packed_bwd_bf16(const fl_packed_params& p, const fl_packed_grads& d, void* ws,
                                  hipStream_t stream) {
  return launch_bwd_type<__bf16>(p, d, ws, stream);
}

}  // namespace fl
