// Launches of the slot-scheduled kernels over packed sequences, one source file
// per head dim and element type (packed_fwd_d64_f16.hip, ...: the instances
// compile in parallel).
#pragma once

#include "fa2_d128_kernel.h"
#include "fa2_slot_kernel.h"

namespace fl {

namespace {

// Rows of a work-group, and whether its key range is halved between two
// streams of waves or two blocks of a sequence are walked after one another.
enum class PackedShape { kRows128, kRows256, kSplit128, kSplit64, kPair128, kPair64 };

// The shape of a launch, from what the host knows of the lengths, their means
// (us, kRows128 against the rule's choice; fp16 D 64, bf16 D 128).  Work-groups
// of 128 rows, two a CU, are the rule; with few of them over long keys the
// walks are halved:
//   64-row groups fit the CUs once: B1 H8 N1024 D 64 12.6 against 10.2
//   128-row ones do, over keys of 768: 4 sequences of 500-1500, H8/2 D 128,
//     causal 23.6 against 20.7; of 2048, causal, as 64-row pairs: B1 H8 N4096
//     D 64 37.9 against 30.2; without a mask 42.8 against 41.4
//   twice, causal, as 128-row pairs: B2 H8 N4096 D 64 50.3 against 44.9
// and with many over very long keys 256 rows share a tile: B1 H16 N16384 D 64
// 584 against 567, B8 H16 N1000-3000 not causal 182 against 175.
inline PackedShape packed_shape(const fl_packed_params& p) {
  const int64_t cus = device_cus();
  const int64_t keys = p.key_rows / p.sequences;
  auto groups = [&](int64_t rows) { return (p.rows / rows + p.sequences) * p.heads; };
  // (an eighth more than a round: sequences end inside a block)
  if (keys >= 512 && groups(64) <= cus + cus / 8) return PackedShape::kSplit64;
  if (keys >= 768 && groups(128) <= cus + cus / 6) {
    if (p.causal) return keys >= 2048 ? PackedShape::kPair64 : PackedShape::kSplit128;
    if (keys >= 2048) return PackedShape::kSplit128;
  }
  if (p.causal && keys >= 2048 && groups(128) <= 2 * cus + cus / 4) return PackedShape::kPair128;
  if (keys >= (p.causal ? 4096 : 2000) && groups(256) >= cus) return PackedShape::kRows256;
  return PackedShape::kRows128;
}

template <int D, int W, int SPLIT, bool PAIR, class T>
hipError_t launch_packed(const fl_packed_params& p, const PackedGeom& g, const Scales& sc,
                         hipStream_t st) {
  const dim3 grid(
      (unsigned)packed_groups(p.rows, p.sequences, (PAIR ? 64 : 32) * W, p.heads));
  const dim3 block(64 * W * SPLIT);
  const T *q = static_cast<const T*>(p.q), *k = static_cast<const T*>(p.k),
          *v = static_cast<const T*>(p.v);
  T* o = static_cast<T*>(p.o);
  auto run = [&](auto causal) {
    constexpr bool kCausal = decltype(causal)::value != 0;
    if constexpr (D == 128)
      hipLaunchKernelGGL((fa2_fwd_d128_kernel<W, 4, kCausal, T, SPLIT, PAIR, PackedGeom>), grid,
                         block, 0, st, q, k, v, o, g, 0, sc.cq, sc.cr);
    else
      hipLaunchKernelGGL(
          (fa2_fwd_slot_kernel<W, W == 8 ? 4 : 2, kCausal, true, T, SPLIT, PAIR, PackedGeom>), grid,
          block, 0, st, q, k, v, o, g, 0, sc.cq, sc.cr);
  };
  if (PAIR || p.causal)  // (block pairs balance a causal mask)
    run(Ic<1>{});
  else if constexpr (!PAIR)
    run(Ic<0>{});
  return hipGetLastError();
}

template <int D, class T>
hipError_t launch_packed_fwd(const fl_packed_params& p, hipStream_t st) {
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
  switch (packed_shape(p)) {
    case PackedShape::kRows256: return launch_packed<D, 8, 1, false, T>(p, g, sc, st);
    case PackedShape::kSplit128: return launch_packed<D, 4, 2, false, T>(p, g, sc, st);
    case PackedShape::kSplit64: return launch_packed<D, 2, 2, false, T>(p, g, sc, st);
    case PackedShape::kPair128: return launch_packed<D, 4, 2, true, T>(p, g, sc, st);
    case PackedShape::kPair64: return launch_packed<D, 2, 2, true, T>(p, g, sc, st);
    default: return launch_packed<D, 4, 1, false, T>(p, g, sc, st);
  }
}

}  // namespace

}  // namespace fl
