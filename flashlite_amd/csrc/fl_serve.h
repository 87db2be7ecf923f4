// Internal interface between the C-ABI layer of the paged-cache operators
// (capi_serve.hip) and their kernels (cache_plan.hip, rotary.hip,
// tree_fwd.hip).  Sizes and pointers are validated before a launch.
#pragma once

#include "fl_internal.h"
#include "flashlite_attn.h"

namespace fl {

// Division of n < 2^31 by d, 1 <= d < 2^31 (Granlund and Montgomery's
// multiply and shift): q = (umulhi(mul, n) + n) >> shift.
struct FastDiv {
  uint32_t mul;
  int shift;
  int d;
};

inline FastDiv fast_div(int d) {
  FastDiv f;
  f.d = d;
  f.shift = 0;
  while (((int64_t)1 << f.shift) < d) ++f.shift;
  f.mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << f.shift) - (uint64_t)d)) /
                         (uint64_t)d +
                     1);
  return f;
}

__device__ __forceinline__ int divide(int n, const FastDiv& f) {
  return (int)((__umulhi(f.mul, (uint32_t)n) + (uint32_t)n) >> f.shift);
}

// Inclusive sum over a wave's lanes: within rows of 16, then over the rows.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);  // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);  // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);  // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true);  // row_bcast:31
  return x;
}

hipError_t launch_cache_plan(const fl_cache_plan_params& p, hipStream_t stream);  // cache_plan.hip
hipError_t launch_tree_plan(const fl_tree_plan_params& p, hipStream_t stream);    // cache_plan.hip

// With `store` the rows also go to the cache (rotary.hip).
hipError_t launch_rotary(const fl_rotary_params& p, const fl_cache_store* store,
                         hipStream_t stream);

// Norms and rotation (norm_rotary.hip): with `store` the rows also go to the
// cache, with `grads` the backward pass and its workspace.
int64_t norm_rotary_workspace_bytes(int64_t head_dim);
hipError_t launch_norm_rotary(const fl_rotary_params& p, const fl_norm_params& n,
                              const fl_cache_store* store, const fl_norm_grads* grads, void* ws,
                              hipStream_t stream);
// Zeros to the weights' gradients (each may be null).
hipError_t launch_norm_zero(const fl_rotary_params& p, float* dq, float* dk, hipStream_t stream);

// Bytes of the partial results of a call of these sizes, 0 where it is not
// split; launch_tree_fwd with ws == nullptr does without (tree_fwd.hip).
int64_t tree_workspace_bytes(const fl_tree_params& p);
hipError_t launch_tree_fwd(const fl_tree_params& p, void* ws, hipStream_t stream);

// Packed sequences, by head dim and element type (packed_fwd_*.hip) or by
// element type (packed_bwd_*.hip); dimensions of one entry have strides that fit.
hipError_t launch_packed_fwd_d64_f16(const fl_packed_params& p, hipStream_t stream);
hipError_t launch_packed_fwd_d64_bf16(const fl_packed_params& p, hipStream_t stream);
hipError_t launch_packed_fwd_d128_f16(const fl_packed_params& p, hipStream_t stream);
hipError_t launch_packed_fwd_d128_bf16(const fl_packed_params& p, hipStream_t stream);
hipError_t launch_packed_bwd_f16(const fl_packed_params& p, const fl_packed_grads& d, void* ws,
                                 hipStream_t stream);
hipError_t launch_packed_bwd_bf16(const fl_packed_params& p, const fl_packed_grads& d, void* ws,
                                  hipStream_t stream);

// The backward pass' workspace: {lse, delta} of every row, then with more than
// one part [parts][kv_heads][key_rows][2 head_dim] sums (capi_packed.hip).
int packed_bwd_parts(const fl_packed_params& p);
inline int64_t packed_stat_bytes(const fl_packed_params& p) {
  return (p.heads * p.rows * 8 + 255) / 256 * 256;
}

}  // namespace fl
