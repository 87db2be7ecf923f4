// Attention over packed sequences, head dim 128, bf16: see packed_launch.h.

#include "packed_launch.h"

namespace fl {

hipError_t launch_packed_fwd_d128_bf16(const fl_packed_params& p, hipStream_t stream) {
  return launch_packed_fwd<128, __bf16>(p, stream);
}

}  // namespace fl
