// Attention over packed sequences, head dim 64, bf16: see packed_launch.h.

#include "packed_launch.h"

namespace fl {

hipError_t launch_packed_fwd_d64_bf16(const fl_packed_params& p, hipStream_t stream) {
  return launch_packed_fwd<64, __bf16>(p, stream);
}

}  // namespace fl
