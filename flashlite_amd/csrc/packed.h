// Packed sequences (fl_attn_packed_fwd, fl_attn_packed_bwd): which rows a
// work-group has, from the sequences' starts on the GPU.
#pragma once

#include "fa2_common.h"
#include "fl_serve.h"

namespace fl {

namespace {

// One launch over packed sequences.  Sequence i has rows starts[i] ..
// starts[i + 1] - 1 of q and o, key_starts[i] .. of k and v.
struct PackedGeom {
  static constexpr bool kPacked = true;
  long long q_sh, k_sh, v_sh, o_sh;  // elements
  int q_sr, k_sr, v_sr, o_sr;
  const int32_t* starts;
  const int32_t* key_starts;
  int sequences, rows, key_rows;
  int heads, group;  // query heads, and those of a key head
  int xcds;
  float* lse;        // [heads][rows] or null
};

__device__ __forceinline__ int wave_sum(int x) {
  return __builtin_amdgcn_readlane(wave_scan(x), 63);
}

// The rows [begin, begin + count) of sequence i; starts out of [0, rows] or
// falling are brought into order, never followed.
__device__ __forceinline__ void sequence_rows(const int32_t* starts, int i, int rows, int& begin,
                                              int& count) {
  begin = min(max(starts[i], 0), rows);
  count = min(max(starts[i + 1], begin), rows) - begin;
}

// The largest of a wave's values, none negative (as wave_scan).
__device__ __forceinline__ int wave_max(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true));
  return __builtin_amdgcn_readlane(x, 63);
}

// A block of a sequence's rows (its j-th, of those that are cut into blocks), and
// the sequence's rows among those and among the others.
struct PackedAt {
  int j, begin, count, other, others;
};

// Block of rank r among the sequences' blocks of BLOCK rows, which is the same in
// every wave and needs no table.  False: no block.
//
// Under a causal mask, up to kRanked sequences, a lane each: the higher a
// block's index j, the earlier its rank (the heaviest first, over all
// sequences); f(l) = sum_i max(blocks_i - l, 0) blocks have j >= l.  More
// sequences, and any without that mask, follow one another, the last block of
// each first, which keeps neighbours in the L2 (us, ranked against one after
// the other; causal bf16 H32/8 D 128: gradients of 16 sequences of 500-1500 593
// and 649, of 32 of 64-2000 1402 and 1511, of 64 2945 and 2943, of 100 4879 and
// 4560; not causal, of 32 2617 and 2454, of 8 of 1000-3000 1936 and 1843, of one
// of 4096 844 and 863).
constexpr int kRanked = 64;

template <int BLOCK>
__device__ __forceinline__ bool packed_block(const int32_t* starts, int rows,
                                             const int32_t* other_starts, int others,
                                             int sequences, int r, bool ranked, PackedAt& x) {
  const int lane = threadIdx.x & 63;
  int begin = rows, count = 0;
  if (sequences > kRanked) {
    // Sequence i has the ranks from begin_i / BLOCK + i on, one more than it
    // may need: the last i that starts at or before r, 64 places a look.
    int lo = 0, hi = sequences;
    while (hi - lo > 1) {
      const int step = (hi - lo + 63) / 64, i = lo + step * lane;
      const bool past = i >= hi || min(max(starts[i], 0), rows) / BLOCK + i > r;
      const uint64_t at = __builtin_amdgcn_ballot_w64(past);
      if (at & 1) return false;
      lo += step * ((at == 0 ? 64 : __builtin_ctzll(at)) - 1);
      hi = min(hi, lo + step);
    }
    sequence_rows(starts, lo, rows, x.begin, x.count);
    sequence_rows(other_starts, lo, others, x.other, x.others);
    r -= x.begin / BLOCK + lo;
    x.j = (x.count + BLOCK - 1) / BLOCK - 1 - r;
    return r >= 0 && x.j >= 0;
  }
  // A lane a sequence: what the block needs of its own is then read across
  // lanes, not loaded behind the search.
  int other = 0, of_other = 0, seq;
  if (lane < sequences) {
    sequence_rows(starts, lane, rows, begin, count);
    sequence_rows(other_starts, lane, others, other, of_other);
  }
  const int nb = (count + BLOCK - 1) / BLOCK;
  if (ranked) {
    auto above = [&](int l) __attribute__((always_inline)) { return wave_sum(max(nb - l, 0)); };
    if (r >= above(0)) return false;
    int lo = 0, hi = wave_max(nb);  // above(lo) > r >= above(hi)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (above(mid) > r)
        lo = mid;
      else
        hi = mid;
    }
    r -= above(lo + 1);  // the r-th sequence with a block lo
    x.j = lo;
    const uint64_t has = __builtin_amdgcn_ballot_w64(nb > lo);
    const int before = (int)__builtin_amdgcn_mbcnt_hi(
        (uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
    seq = __builtin_ctzll(__builtin_amdgcn_ballot_w64(nb > lo && before == r));
  } else {
    const int first = begin / BLOCK + lane;
    const uint64_t past = __builtin_amdgcn_ballot_w64(lane >= sequences || first > r);
    if (past & 1) return false;
    seq = (past == 0 ? 64 : __builtin_ctzll(past)) - 1;
    x.j = __builtin_amdgcn_readlane(first + nb, seq) - 1 - r;
    if (x.j < 0) return false;
  }
  x.begin = __builtin_amdgcn_readlane(begin, seq);
  x.count = __builtin_amdgcn_readlane(count, seq);
  x.other = __builtin_amdgcn_readlane(other, seq);
  x.others = __builtin_amdgcn_readlane(of_other, seq);
  return true;
}

// Work-groups of blocks of `block` rows: at least what any sequences of these
// rows need.
inline int64_t packed_groups(int64_t rows, int64_t sequences, int64_t block, int64_t units) {
  return (rows / block + sequences) * units;
}

// Work-group -> (rank, unit) with `units` independent walks of a block (heads):
// neighbouring units, which share keys, on one XCD where they divide evenly.
__device__ __forceinline__ void packed_unit(int i, int units, int xcds, int& r, int& unit) {
  if (units % xcds == 0) {
    const int per = units / xcds, k = i / xcds;
    r = k / per;
    unit = (i - k * xcds) * per + (k - r * per);
  } else {
    r = i / units;
    unit = i - r * units;
  }
}

// The forward kernels' problem of this work-group: query block qb (of BLOCK
// rows) of head bh as a dense problem of one sequence, query heads that share
// a key head as a batch with key head stride 0.  False: no block.
template <int BLOCK, bool CAUSAL, class QPtr, class KPtr, class OPtr>
__device__ __forceinline__ bool packed_problem(const PackedGeom& p, QPtr& Q, KPtr& K, KPtr& V,
                                               OPtr& O, Geom& g, int& bh, int& qb) {
  int r;
  PackedAt x;
  packed_unit(blockIdx.x, p.heads, p.xcds, r, bh);
  if (!packed_block<BLOCK>(p.starts, p.rows, p.key_starts, p.key_rows, p.sequences, r, CAUSAL, x))
    return false;
  qb = x.j;
  const int q0 = x.begin, k0 = x.other;
  g.seq_q = x.count;
  g.seq_k = x.others;
  g.coff = g.seq_k - g.seq_q;
  g.heads = p.group;
  g.q_sb = p.q_sh * p.group;
  g.q_sh = p.q_sh;
  g.o_sb = p.o_sh * p.group;
  g.o_sh = p.o_sh;
  g.k_sb = p.k_sh;
  g.v_sb = p.v_sh;
  g.k_sh = g.v_sh = 0;
  g.q_sr = p.q_sr;
  g.k_sr = p.k_sr;
  g.v_sr = p.v_sr;
  g.o_sr = p.o_sr;
  Q += (long long)q0 * p.q_sr;
  K += (long long)k0 * p.k_sr;
  V += (long long)k0 * p.v_sr;
  O += (long long)q0 * p.o_sr;
  // (head_ptrs adds bh * seq_q)
  g.lse = p.lse ? p.lse + ((long long)bh * (p.rows - g.seq_q) + q0) : nullptr;
  return true;
}

__device__ __forceinline__ const Geom& problem_geom(const Geom& g, const Geom&) { return g; }
__device__ __forceinline__ const Geom& problem_geom(const PackedGeom&, const Geom& own) {
  return own;
}

template <int N>
__device__ __forceinline__ bool any_odd(const float16_t (&x)[N]) {
  float most = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) most += x[i][r] * 0.0f;
  return most != 0.0f;
}

// A tile's transposed operands `op` (of D columns and 8192 / 2D rows) before
// a product whose other factor is 0 for rows of the tile that a lane's own row
// does not see: NaN and infinities become 0, and are added to the lanes that
// see their row.
template <int D, class T, class Ops, class Sees, class Swizzle>
__device__ __forceinline__ void add_odd(const uint8_t* tile, Ops& ops, float16_t (&acc)[D / 32],
                                        int g, Sees&& sees, Swizzle&& swizzle) {
  using V8 = typename Elem<T>::v8;
  V8(&op)[8] = reinterpret_cast<V8(&)[8]>(ops);
  if (__builtin_amdgcn_ballot_w64(any_odd<T>(op)) == 0) return;
#pragma unroll
  for (int u = 0; u < 8; ++u) op[u] = finite_only<T>(op[u]);
#pragma unroll 1
  for (int j = 0; j < kTileBytes / (2 * D); ++j) {
    const bool mine = sees(j);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const V8 x = *reinterpret_cast<const V8*>(tile + j * 2 * D + 16 * ((2 * c + g) ^ swizzle(j)));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = (float)x[e];
        if (mine && !(__builtin_fabsf(y) < __builtin_huge_valf()))
          acc[c >> 1][8 * (c & 1) + e] += y;
      }
    }
  }
}

}  // namespace

}  // namespace fl
