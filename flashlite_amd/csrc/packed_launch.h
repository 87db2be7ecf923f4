// Launches of the slot-scheduled kernels over packed sequences, one source file
// per element type (packed_fwd_f16.hip, packed_fwd_bf16.hip: the instances
// compile in parallel).
#pragma once

#include "fa2_d128_kernel.h"
#include "fa2_slot_kernel.h"

namespace fl {

namespace {

template <int D, int W, int SPLIT, class T>
hipError_t launch_packed(const fl_packed_params& p, const PackedGeom& g, const Scales& sc,
                         hipStream_t st) {
  const dim3 grid((unsigned)packed_groups(p.rows, p.sequences, 32 * W, p.heads));
  const dim3 block(64 * W * SPLIT);
  const T *q = static_cast<const T*>(p.q), *k = static_cast<const T*>(p.k),
          *v = static_cast<const T*>(p.v);
  T* o = static_cast<T*>(p.o);
  if constexpr (D == 128) {
    if (p.causal)
      hipLaunchKernelGGL((fa2_fwd_d128_kernel<W, 4, true, T, SPLIT, false, PackedGeom>), grid, block,
                         0, st, q, k, v, o, g, 0, sc.cq, sc.cr);
    else
      hipLaunchKernelGGL((fa2_fwd_d128_kernel<W, 4, false, T, SPLIT, false, PackedGeom>), grid,
                         block, 0, st, q, k, v, o, g, 0, sc.cq, sc.cr);
  } else {
    constexpr int kFv = W == 8 ? 4 : 2;
    if (p.causal)
      hipLaunchKernelGGL((fa2_fwd_slot_kernel<W, kFv, true, true, T, SPLIT, false, PackedGeom>),
                         grid, block, 0, st, q, k, v, o, g, 0, sc.cq, sc.cr);
    else
      hipLaunchKernelGGL((fa2_fwd_slot_kernel<W, kFv, false, true, T, SPLIT, false, PackedGeom>),
                         grid, block, 0, st, q, k, v, o, g, 0, sc.cq, sc.cr);
  }
  return hipGetLastError();
}

template <int D, class T>
hipError_t launch_packed_dim(const fl_packed_params& p, const PackedGeom& g, const Scales& sc,
                             hipStream_t st) {
  return launch_packed<D, 4, 1, T>(p, g, sc, st);
}

template <class T>
hipError_t launch_packed_type(const fl_packed_params& p, hipStream_t st) {
  PackedGeom g = {};
  g.q_sh = p.q_stride[0];
  g.k_sh = p.k_stride[0];
  g.v_sh = p.v_stride[0];
  g.o_sh = p.o_stride[0];
  g.q_sr = (int)p.q_stride[1];
  g.k_sr = (int)p.k_stride[1];
  g.v_sr = (int)p.v_stride[1];
  g.o_sr = (int)p.o_stride[1];
  g.starts = p.starts;
  g.key_starts = p.key_starts ? p.key_starts : p.starts;
  g.sequences = (int)p.sequences;
  g.rows = (int)p.rows;
  g.key_rows = (int)p.key_rows;
  g.heads = (int)p.heads;
  g.group = (int)(p.heads / p.kv_heads);
  g.xcds = device_xcds();
  g.lse = p.lse;
  const double s =
      p.sm_scale == 0.0 ? 1.0 / __builtin_sqrt((double)p.head_dim) : p.sm_scale;
  FwdArgs a = {};
  a.negate = s < 0.0;
  a.scale_log2 = (float)(__builtin_fabs(s) * 1.4426950408889634);
  const Scales sc(a);
  return p.head_dim == 128 ? launch_packed_dim<128, T>(p, g, sc, st)
                           : launch_packed_dim<64, T>(p, g, sc, st);
}

}  // namespace

}  // namespace fl
