// Slot-scheduled schedule (configurations br256_bc64_w8_slot,
// br128_bc64_w4_slot, the key-range splits br128_bc64_w4x2_slot and
// br64_bc64_w2x2_slot, and the block pairs br128_bc64_w4x2_pair), fp16 and
// bf16 at head_dim 64: launches of fa2_slot_kernel.h.

#include "fa2_slot_kernel.h"

namespace fl {

namespace {

template <int W, int FV, class T = _Float16, int SPLIT = 1, bool PAIR = false>
struct SlotLaunch {
  template <bool C, bool S>
  struct L {
    static hipError_t run(const FwdArgs& a, const Geom& g, dim3 grid, int nqb, float cq, float cr,
                          hipStream_t st) {
      if constexpr (PAIR) grid = dim3((unsigned)(a.batch_heads * ((nqb + 1) / 2)));
      hipLaunchKernelGGL((fa2_fwd_slot_kernel<W, FV, C, S, T, SPLIT, PAIR>), grid,
                         dim3(64 * W * SPLIT), 0, st,
                         static_cast<const T*>(a.q), static_cast<const T*>(a.k),
                         static_cast<const T*>(a.v), static_cast<T*>(a.o), g, nqb, cq, cr);
      return hipSuccess;
    }
  };
};

}  // namespace

// fp16 or bf16 by a.dtype; W = 8 (256-row groups, one per CU, V fetched 4
// tiles ahead) or 4 (128-row groups, two per CU, 2 tiles ahead: 64 KiB of
// rings, measured 0.3-4% faster than 3 from N 1024 to 8192, causal C2
// included).
hipError_t launch_slot(const FwdArgs& a, int waves, hipStream_t stream) {
  const bool bf = a.dtype == kDtypeBF16;
  if (waves == 8)
    return bf ? dispatch<SlotLaunch<8, 4, __bf16>::L>(a, stream, 256)
              : dispatch<SlotLaunch<8, 4>::L>(a, stream, 256);
  if (waves == 4)
    return bf ? dispatch<SlotLaunch<4, 2, __bf16>::L>(a, stream, 128)
              : dispatch<SlotLaunch<4, 2>::L>(a, stream, 128);
  return hipErrorInvalidValue;
}

// V fetch distance of the key-range splits: rings of 4 tiles (128 KiB per
// group), measured 1-6% faster than 3 (160 KiB) on the shapes the
// dispatcher sends to them; their walks are short, so the shorter prologue
// matters more than the deeper pipeline.
constexpr int kSplitFv = 2;

// fp16 or bf16 by a.dtype: groups of 2 x `waves` waves (4: 128-row blocks,
// 2: 64-row blocks) walking a pair of blocks of a head, p and nqb-1-p, each
// with its key range halved between the streams (grid B*H*ceil(nqb/2)).
hipError_t launch_slot_pair(const FwdArgs& a, int waves, hipStream_t stream) {
  const bool bf = a.dtype == kDtypeBF16;
  if (waves == 4)
    return bf ? dispatch<SlotLaunch<4, kSplitFv, __bf16, 2, true>::L>(a, stream, 128)
              : dispatch<SlotLaunch<4, kSplitFv, _Float16, 2, true>::L>(a, stream, 128);
  if (waves == 2)
    return bf ? dispatch<SlotLaunch<2, kSplitFv, __bf16, 2, true>::L>(a, stream, 64)
              : dispatch<SlotLaunch<2, kSplitFv, _Float16, 2, true>::L>(a, stream, 64);
  return hipErrorInvalidValue;
}

// fp16 or bf16 by a.dtype: groups of 2 x `waves` waves (4: 128 rows, 2: 64
// rows), the key range halved between them.
hipError_t launch_slot_split(const FwdArgs& a, int waves, hipStream_t stream) {
  const bool bf = a.dtype == kDtypeBF16;
  if (waves == 4)
    return bf ? dispatch<SlotLaunch<4, kSplitFv, __bf16, 2>::L>(a, stream, 128)
              : dispatch<SlotLaunch<4, kSplitFv, _Float16, 2>::L>(a, stream, 128);
  if (waves == 2)
    return bf ? dispatch<SlotLaunch<2, kSplitFv, __bf16, 2>::L>(a, stream, 64)
              : dispatch<SlotLaunch<2, kSplitFv, _Float16, 2>::L>(a, stream, 64);
  return hipErrorInvalidValue;
}

}  // namespace fl
