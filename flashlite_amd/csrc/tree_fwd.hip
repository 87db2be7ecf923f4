// Attention of drafted tokens over a paged cache (fl_attn_tree_fwd), fp16 and
// bf16, head dim 64 and 128.  Shared building blocks: fa2_common.h, fa2_d128.h.
//
// The rows of one key/value head are its group of query heads times the drafts
// (row r: draft r / group, head r % group), so a cached key is read once for
// all of them.  A unit is 32 RW such rows of one (request, key/value head): a
// work-group's 4 (8) waves are RW row blocks times 4 / RW (1) key groups.
//
// One pass: o = sum p v, l = sum p with p = 2^(s - mc) and a stabiliser mc that
// a row takes from its first tile; parts of a row meet as
// sum_j 2^(mc_j - max mc) (o_j, l_j).  4 D flops a row and key against 4 D
// bytes a key: up to about 100 rows a key/value head are bound by memory (one
// token after 256-8192 of 32 requests, 32/8 heads, D 128: 5.3 TB/s), more by
// the matrix cores and what feeds them (64 drafts after 16000 of 8 requests,
// 32/8 heads: 0.7 PFLOP/s, matrix cores 42% busy), and short calls by the chain
// lengths, table entry, key row and by the second launch (one token after 4096,
// B2 H8 D 64: 12.1-12.9 us, of them the merge 3.1-3.8).

#include <algorithm>
#include <cmath>

#include "fa2_d128.h"
#include "fl_serve.h"

namespace fl {

namespace {

struct TreeGeom {
  long long q_sb, q_sh, q_sr, o_sb, o_sh, o_sr;  // elements
  long long k_head, v_head;             // bytes
  uint32_t k_blk, k_row, v_blk, v_row;  // bytes
  const int32_t* tables;
  long long table_stride;
  const int32_t* lengths;
  const int32_t* counts;
  const int64_t* mask;
  long long mask_stride;
  float* lse;
  int batch, heads, kv_units, drafts, rows, words, blocks_of_rows;
  int num_blocks, capacity;  // capacity: keys of a table row
  FastDiv block, group, by_drafts;
  // split launches: partial results, part_size floats each ([heads side by side]
  // [part_rows][kPartStride]), and per unit where they begin and end
  float* part;
  int2* parts;
  int part_rows, part_size;
  int xcds;
};

// The first n of 64 bits.
__device__ __forceinline__ uint64_t first_bits(int n) {
  return n <= 0 ? 0 : n >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << n) - 1;
}

// Where a lane's operands lie: those of Rows (head dim 64) and Rows128.
template <int D, class T>
struct TreeLayout;
template <class T>
struct TreeLayout<64, T> {
  using type = Rows<false, true, T>;
};
template <class T>
struct TreeLayout<128, T> {
  using type = Rows128<false, T>;
};

// One wave's 32 rows.  Scores stay raw in the accumulators and the stabiliser
// mc (base-2 logit units) is subtracted with the scale's multiply.  mc is the
// row max of the first tile in which the row sees a key, and later only moves
// when a tile would push p out of fp16's range; it never passes the running
// max.
template <int D, class T>
struct TreeRows : TreeLayout<D, T>::type {
  using Base = typename TreeLayout<D, T>::type;
  using E = Elem<T>;
  using V8 = typename E::v8;
  static constexpr int kBlocks = D == 64 ? 2 : 1;  // 32-key blocks of a tile
  static constexpr int kKeys = 32 * kBlocks, kSteps = D / 16;
  struct Scores {
    float16_t s[kBlocks];
  };
  struct Probs {
    V8 p[2 * kBlocks];
  };
  float mc;

  __device__ __forceinline__ void start(int lane, float cr) {
    Base::place(lane, 0, 0, 0, 0, cr);
    this->reset();
    mc = 0.0f;
  }
  __device__ __forceinline__ void scores(const uint8_t* kt, Scores& s) const {
    V8 ka[kBlocks][kSteps];
#pragma unroll
    for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
      for (int st = 0; st < kSteps; ++st) {
        if constexpr (D == 64)
          ka[kb][st] = this->read_k_op(kt, kb, st);
        else
          ka[kb][st] = this->read_k_op(kt, st);
      }
    const float16_t zero = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int st = 0; st < kSteps; ++st)
#pragma unroll
      for (int kb = 0; kb < kBlocks; ++kb)
        s.s[kb] = E::mfma(ka[kb][st], this->qf[st], st == 0 ? zero : s.s[kb]);
  }
  // Scores of hidden keys become -inf (bit j: key j of the tile is visible).
  __device__ __forceinline__ void hide(uint64_t seen, Scores& s) const {
    const uint64_t x = seen >> (4 * this->g);
#pragma unroll
    for (int kb = 0; kb < kBlocks; ++kb) {
      const uint32_t word = (uint32_t)(x >> (32 * kb));
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s.s[kb][r] = (word >> (8 * (r >> 2) + (r & 3))) & 1 ? s.s[kb][r] : ninf();
    }
  }
  // Row max of a tile in base-2 logit units (both halves of the row).
  __device__ __forceinline__ float tile_max(const Scores& s) const {
    float mx = ninf();
#pragma unroll
    for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s.s[kb][r]);
    return pair_max(mx) * this->cr;
  }
  // Rows without a stabiliser take the tile's row max, if they see a key.
  __device__ __forceinline__ bool settle(bool unset, const Scores& s) {
    const float mx = tile_max(s);
    const bool now = unset && mx != ninf();
    if (now) mc = mx;
    return unset && !now;
  }
  // p = 2^(s cr - mc); returns this lane's sum of the unrounded p.  For the
  // product with V p is rounded to the element type, half a step of it a key:
  // the matrix cores take 16-bit operands, and a second product with what the
  // rounding left would double half of the work.  Against 64 bits outputs are
  // off by 2.6-2.9e-4 (fp16) and 2.3e-3 (bf16) where their own rounding alone
  // makes 2.0e-4 and 1.7e-3.
  __device__ __forceinline__ float exponentiate(const Scores& s, Probs& p) const {
    float sum[2 * kBlocks];
#pragma unroll
    for (int h = 0; h < 2 * kBlocks; ++h) {
      sum[h] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x =
            __builtin_amdgcn_exp2f(__builtin_fmaf(s.s[h >> 1][8 * (h & 1) + e], this->cr, -mc));
        p.p[h][e] = (T)x;
        sum[h] += x;
      }
    }
    float all = sum[0] + sum[1];
    if constexpr (kBlocks == 2) all += sum[2] + sum[3];
    return all;
  }
  // Ends a tile's softmax: where a lane's sum left the range that keeps p
  // finite (or is NaN), mc moves up to the row max and p is taken again.
  __device__ __forceinline__ void settle_sum(float sum, const Scores& s, Probs& p) {
    if (__builtin_amdgcn_ballot_w64(!(sum <= kSumLimit)) != 0) {
      const float d = fmaxf(tile_max(s) - mc, 0.0f);
      const float alpha = __builtin_amdgcn_exp2f(-d);
      this->l *= alpha;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) this->o[db][r] *= alpha;
      mc += d;
      sum = exponentiate(s, p);
    }
    this->l += sum;
  }
  // V operand u of the tile: head-dim block u % (D / 32) at 16-key step
  // u / (D / 32).
  __device__ __forceinline__ V8 v_op(const uint8_t* vt, int u) const {
    return this->read_v_op(vt, u % (D / 32), u / (D / 32));
  }
  __device__ __forceinline__ void output(int u, const V8& v, const Probs& p) {
    this->o[u % (D / 32)] = E::mfma(v, p.p[u / (D / 32)], this->o[u % (D / 32)]);
  }
  __device__ __forceinline__ static int v_phys(int row, int chunk) {
    return chunk ^ (D == 64 ? v_swz(row) : v_swz128(row));
  }
};

// 16 (or 4) bytes a lane from a 64-bit address of its own into LDS at
// base + 16 (4) * lane, asynchronously (vmcnt).  Inline assembly, so that the
// compiler does not guard reads of other slots with waits on it.  The wait state
// before the load is the one that it needs behind the write of M0 (load_lds16).
__device__ __forceinline__ void fetch16(uint64_t address, const void* lds) {
  const uint32_t base = (uint32_t)(uintptr_t)lds;
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               : : "v"(address), "{m0}"(base) : "memory");
}
__device__ __forceinline__ void fetch4(uint64_t address, const void* lds) {
  const uint32_t base = (uint32_t)(uintptr_t)lds;
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off"
               : : "v"(address), "{m0}"(base) : "memory");
}

// Waves of a work-group of RW row blocks, and slots for tiles of each of its
// key groups.  DEEP: for long walks, see launch_rw.
constexpr int slots_of(int d, int rw, bool deep) { return rw == 2 && d == 128 && deep ? 4 : rw; }
constexpr int waves_of(int rw) { return rw == 8 ? 8 : 4; }
// Key/value heads of a work-group, side by side.
constexpr int heads_of(int rw, bool deep) { return rw == 1 && deep ? 4 : 1; }
constexpr int key_groups_of(int rw, bool deep) { return waves_of(rw) / (rw * heads_of(rw, deep)); }

// One request: its tokens and its drafts that are there.
struct Request {
  int length, count;
};

__device__ __forceinline__ Request request(const TreeGeom& g, int b) {
  Request r;
  r.length = g.lengths[b];
  r.count = g.drafts;
  if (g.counts) r.count = min(max(g.counts[b], 0), g.drafts);
  r.length = min(max(r.length, 0), g.capacity);
  return r;
}

// Drafts whose keys row block rb (of `block` rows) of a request walks; with a
// chain through its last row's draft.
__device__ __forceinline__ int unit_drafts(const TreeGeom& g, const Request& r, int rb,
                                           int block) {
  int drafts = min(r.count, g.capacity - r.length);
  if (g.mask == nullptr)
    drafts = min(drafts, divide(min((rb + 1) * block, g.rows) - 1, g.group) + 1);
  return drafts;
}

// Steps of a unit's walk, 0 where no draft of its rows is there.
template <int D, int RW, bool DEEP>
__device__ __forceinline__ int unit_steps(const TreeGeom& g, const Request& r, int rb) {
  constexpr int kStepKeys = key_groups_of(RW, DEEP) * (D == 64 ? kBc : kBc2);
  if (rb * 32 * RW >= r.count * g.group.d) return 0;
  return (r.length + unit_drafts(g, r, rb, 32 * RW) + kStepKeys - 1) / kStepKeys;
}

// A unit's cost to a split launch, in steps: its walk and what starting one
// takes (the first tiles' latency, the merge of partial results).
constexpr int start_of(int rw) { return rw == 1 ? 1 : rw == 2 ? 6 : 10; }

template <int RW>
__device__ __forceinline__ int cost_of(int steps) {
  return steps > 0 ? steps + start_of(RW) : 0;
}

// Costs of all row blocks of one key/value head of a request.
template <int D, int RW, bool DEEP>
__device__ __forceinline__ int head_cost(const TreeGeom& g, const Request& r) {
  int n = 0;
#pragma unroll 1
  for (int rb = 0; rb < g.blocks_of_rows; ++rb) n += cost_of<RW>(unit_steps<D, RW, DEEP>(g, r, rb));
  return n;
}

__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32));
  return (uint64_t)hi << 32 | lo;
}

// The work-group's LDS: key and value tiles, and per wave the row addresses of
// the next tile's keys and table entries fetched ahead.
template <int D, int RW, bool DEEP>
struct Shared {
  static constexpr int kWaves = waves_of(RW);
  static constexpr int kGroups = kWaves / RW;
  static constexpr int kSlots = slots_of(D, RW, DEEP);
  // Rows of a tile that a wave fetches, and tiles whose rows it looks up at
  // once, a row a lane.
  static constexpr int kRows = (D == 64 ? kBc : kBc2) / RW;
  static constexpr int kPer = 64 / kRows;
  uint8_t tile[kGroups][kSlots][2][kTileBytes];
  uint64_t where[kWaves][2][2][64];  // K and V row addresses of two lookups
  uint64_t good[kWaves][2];          // their keys that have a block
  int bad[kWaves];                   // whether a key so far had none
  int32_t ids[kWaves][2][64];
  float2 ml[kWaves][64];
};

// One unit's part over steps [s0, s1) by this work-group: the result goes to O
// (and lse) with part == nullptr, or unnormalised to `part`.
template <int D, class T, int RW, bool DEEP>
__device__ __forceinline__ void walk(const T* Q, const uint8_t* K, const uint8_t* V, T* O,
                                     const TreeGeom& g, Shared<D, RW, DEEP>& sh, int b, int kvh, int rb,
                                     const Request& req, int s0, int s1, float* part, float cq,
                                     float cr) {
  using RowsT = TreeRows<D, T>;
  using V8 = typename RowsT::V8;
  constexpr int kKeys = RowsT::kKeys, kRowB = 2 * D;
  constexpr int KW = key_groups_of(RW, DEEP);
  constexpr int kHeads = heads_of(RW, DEEP);
  constexpr int kLanes = kRowB / 16;      // lanes a row of a fetch
  constexpr int kSegRows = 64 / kLanes;   // rows a fetch
  constexpr int kSegs = 8 / RW;           // fetches of a tile by this wave
  constexpr int kSlots = Shared<D, RW, DEEP>::kSlots;
  constexpr int kAcc = D / 2;
  constexpr int kPart = D == 64 ? kPartStride : kPartStride128;
  static_assert(kKeys * kRowB == kTileBytes, "tile size");
  static_assert(kHeads == 1 || KW == 1, "key groups of one head meet in LDS");

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Row block, head of those side by side, key group, and which wave (of a row
  // block) or key group's tiles are its.
  const int rw = w % RW, hw = w / RW % kHeads, kg = w / (RW * kHeads), own = w / RW;
  kvh += hw;
  const int length = req.length;
  const int drafts = unit_drafts(g, req, rb, 32 * RW);
  const int keys = length + drafts;
  const int tiles = (keys + kKeys - 1) / kKeys;
  const int first = s0 * KW + kg;  // this key group's tiles: first, first + KW, ...
  const int last = min(s1 * KW, tiles);
  const int n = RW == 1 ? (last > first ? (last - first + KW - 1) / KW : 0) : s1 - s0;

  RowsT rows;
  rows.start(lane, cr);
  const int local = 32 * rw + g.part_rows * hw + rows.col;  // (of the unit's rows in a part)
  const int row = 32 * (RW * rb + rw) + rows.col;
  const int my_row = min(row, g.rows - 1);
  const int draft = divide(my_row, g.group);
  const int head = kvh * g.group.d + (my_row - draft * g.group.d);
  const bool mine = row < g.rows && draft < req.count;
  // Q, and whatever was fetched before it: the loads are waited for here, not
  // among the fetches.
  auto load_q = [&]() __attribute__((always_inline)) {
    const T* q = Q + (b * g.q_sb + head * g.q_sh + draft * g.q_sr) + 8 * rows.g;
    const uint32_t sign = cq < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int st = 0; st < RowsT::kSteps; ++st) {
      const u32x4_t raw = *reinterpret_cast<const u32x4_t*>(q + 16 * st);
      rows.qf[st] = __builtin_bit_cast(V8, raw ^ (u32x4_t){sign, sign, sign, sign});
    }
#pragma unroll
    for (int st = 0; st < RowsT::kSteps; ++st) asm volatile("" : "+v"(rows.qf[st]));
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  };
  const int64_t* const mask =
      g.mask ? g.mask + b * g.mask_stride + (long long)draft * g.words : nullptr;
  // This lane's row's visible keys of tile [k0, k0 + 64) that is not all prefix.
  auto seen_bits = [&](int k0) __attribute__((always_inline)) {
    const int d0 = k0 - length;  // the tile's first draft
    const int from = max(d0, 0);
    uint64_t x = first_bits(drafts - from);
    if (mask == nullptr) {
      x &= first_bits(draft + 1 - from);
    } else {
      const int w0 = from >> 6, shift = from & 63;
      uint64_t m = w0 < g.words ? (uint64_t)mask[w0] >> shift : 0;
      if (shift != 0 && w0 + 1 < g.words) m |= (uint64_t)mask[w0 + 1] << (64 - shift);
      x &= m;
    }
    return d0 >= 0 ? x : (d0 > -64 ? x << -d0 : 0) | first_bits(-d0);
  };

  // The keys that every row of this wave sees: the tokens, and in a chain the
  // drafts up to the first row's.
  const int open =
      mask != nullptr
          ? length
          : length + min(drafts, divide(min(32 * (RW * rb + rw), g.rows - 1), g.group) + 1);

  const uint64_t table = (uint64_t)(uintptr_t)(g.tables + b * g.table_stride);
  const uint64_t kbase = (uint64_t)(uintptr_t)(K + kvh * g.k_head);
  const uint64_t vbase = (uint64_t)(uintptr_t)(V + kvh * g.v_head);
  int32_t(*const ids)[64] = sh.ids[w];
  using Sh = Shared<D, RW, DEEP>;
  constexpr int kPer = Sh::kPer, kRows = Sh::kRows;
  // The key that lane l looks up for the key group's tiles kPer m ..: this
  // wave's row l % kRows of tile kPer m + l / kRows (past the last key: the
  // last again).
  auto key_of = [&](int m) __attribute__((always_inline)) {
    const int tile = first + KW * (kPer * m + lane / kRows);
    return min(tile * kKeys + rw * kRows + lane % kRows, keys - 1);
  };
  auto fetch_ids = [&](int m) __attribute__((always_inline)) {
    fetch4(table + 4 * (uint64_t)divide(key_of(m), g.block), ids[m & 1]);
  };
  // Their rows' addresses, from the table entries, and a bit per key with a
  // block; then the table entries of lookup m + 2.
  int bad = 0;
  auto look_up = [&](int m) __attribute__((always_inline)) {
    const int key = key_of(m);
    const uint32_t in = key - divide(key, g.block) * g.block.d;
    uint32_t id = ids[m & 1][lane];
    const bool good = id < (uint32_t)g.num_blocks;
    id = good ? id : 0;
    sh.where[w][m & 1][0][lane] = kbase + ((uint64_t)id * g.k_blk + (uint64_t)in * g.k_row);
    sh.where[w][m & 1][1][lane] = vbase + ((uint64_t)id * g.v_blk + (uint64_t)in * g.v_row);
    const uint64_t all = __builtin_amdgcn_ballot_w64(good);
    bad |= ~all != 0;
    sh.good[w][m & 1] = all;
    sh.bad[w] = bad;
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    fetch_ids(m + 2);
  };
  // Keys of the key group's tile i with a block.
  auto good_keys = [&](int i) __attribute__((always_inline)) {
    uint64_t x = 0;
#pragma unroll 1
    for (int q = 0; q < RW; ++q) {
      const uint64_t y = uniform(sh.good[own * RW + q][(i / kPer) & 1]) >> (i % kPer * kRows);
      x |= (y & (kRows == 64 ? ~(uint64_t)0 : ((uint64_t)1 << kRows) - 1)) << (q * kRows);
    }
    return x;
  };
  // This wave's share of the K (t = 0) or V (1) tile j.
  auto fetch = [&](int t, int j) __attribute__((always_inline)) {
    uint8_t* const tile = sh.tile[own][j & (kSlots - 1)][t];
    const uint64_t* const from = sh.where[w][(j / kPer) & 1][t] + j % kPer * kRows;
    uint64_t at[kSegs];
#pragma unroll
    for (int i = 0; i < kSegs; ++i) {
      const int r = kSegRows * (rw * kSegs + i) + lane / kLanes;
      const int phys = lane & (kLanes - 1);
      const int chunk = phys ^ (D == 64 ? (t ? v_swz(r) : k_swz(r))
                                        : (t ? v_swz128(r) : k_swz128(r)));
      at[i] = from[kSegRows * i + lane / kLanes] + 16 * chunk;
    }
#pragma unroll
    for (int i = 0; i < kSegs; ++i) fetch16(at[i], tile + 1024 * (rw * kSegs + i));
  };

  bool unset = true, fresh = true;  // this lane's row, some row has no stabiliser yet
  uint64_t seen = 0;
  bool checked = false;
  // Before tile i's exponentials: hidden keys, and rows' first stabilisers.
  // `some_bad`: a key of this walk may have no block.
  auto prepare = [&](int i, bool some_bad, typename RowsT::Scores& s)
                     __attribute__((always_inline)) {
    const int k0 = (first + KW * i) * kKeys;
    checked = k0 + kKeys > open || some_bad;
    if (checked) {
      seen = seen_bits(k0);
      if (some_bad) seen &= good_keys(i);
      rows.hide(seen, s);
    }
    if (fresh) {
      unset = rows.settle(unset, s);
      fresh = __builtin_amdgcn_ballot_w64(unset) != 0;
    }
  };
  auto read_v = [&](const uint8_t* vt, V8 (&va)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 8; ++u) va[u] = rows.v_op(vt, u);
  };
  auto output = [&](const uint8_t* vt, V8 (&va)[8], const typename RowsT::Probs& p)
                    __attribute__((always_inline)) {
    // What p = 0 meets must be finite; a visible NaN or infinity is added to
    // the rows that see it.
    if (checked) {
      if (__builtin_amdgcn_ballot_w64(any_odd<T>(va)) != 0) {
#pragma unroll
        for (int u = 0; u < 8; ++u) va[u] = finite_only<T>(va[u]);
#pragma unroll 1
        for (int j = 0; j < kKeys; ++j) {
          const bool sees = (seen >> j) & 1;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const int chunk = RowsT::v_phys(j, 2 * c + rows.g);
            const V8 x = *reinterpret_cast<const V8*>(vt + j * kRowB + 16 * chunk);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float y = (float)x[e];
              if (sees && !(__builtin_fabsf(y) < __builtin_huge_valf()))
                rows.o[c >> 1][8 * (c & 1) + e] += y;
            }
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) rows.output(u, va[u], p);
  };

  if constexpr (RW == 1) {
    // Every wave has tiles, and a K and a V slot, of its own: no barrier
    // orders the walk.  K(i + 1) is fetched as soon as the operands of K(i)
    // are read, V(i + 1) after those of V(i); table entries two tiles ahead.
    // (Two slots each, 128 KiB, measured 1 us slower for short calls and 3%
    // for long ones.)
    if (n > 0) {
      fetch_ids(0);
      fetch_ids(1);
      load_q();
      look_up(0);
      fetch(0, 0);
      fetch(1, 0);
    }
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      typename RowsT::Scores s;
      typename RowsT::Probs p;
      asm volatile("s_waitcnt vmcnt(8)" : : : "memory");  // K(i), and the next table entries
      rows.scores(sh.tile[own][0][0], s);
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // its operands are in registers
      const bool more = i + 1 < n, next = (i + 1) % kPer == 0;
      prepare(i, bad != 0, s);
      if (more) {
        if (next) look_up((i + 1) / kPer);
        fetch(0, i + 1);
      }
      rows.settle_sum(rows.exponentiate(s, p), s, p);
      if (!more)
        asm volatile("s_waitcnt vmcnt(0)" : : : "memory");  // V(i)
      else if (next)
        asm volatile("s_waitcnt vmcnt(9)" : : : "memory");
      else
        asm volatile("s_waitcnt vmcnt(8)" : : : "memory");
      V8 va[8];
      read_v(sh.tile[own][0][1], va);
      output(sh.tile[own][0][1], va, p);
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      if (more) fetch(1, i + 1);
    }
  } else {
    // RW waves share their key group's tiles, kSlots of K and of V in rings;
    // each fetches 1 / RW of a tile.  Step i multiplies K(i + 1) while it
    // exponentiates the scores of tile i, then V(i), and fetches V(i + kSlots
    // - 1) and K(i + kSlots).  One barrier a step: past it K(i + 1) and V(i)
    // have landed for all, and K(i) and V(i - 1) are read by none.
    fetch_ids(0);
    fetch_ids(1);
    load_q();
    look_up(0);
    fetch(0, 0);
#pragma unroll
    for (int j = 0; j < kSlots - 1; ++j) {
      fetch(1, j);
      fetch(0, j + 1);
    }
    sync_ring<(kSlots - 1) * 2 * kSegs>();
    typename RowsT::Scores s;
    rows.scores(sh.tile[own][0][0], s);
    int flag = sh.bad[own * RW + (lane & (RW - 1))];
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      sync_ring<(kSlots - 2) * 2 * kSegs>();
      prepare(i, __builtin_amdgcn_ballot_w64(flag != 0) != 0, s);
      const uint8_t* const vt = sh.tile[own][i & (kSlots - 1)][1];
      typename RowsT::Scores next;
      typename RowsT::Probs p;
      V8 va[8];
      rows.scores(sh.tile[own][(i + 1) & (kSlots - 1)][0], next);
      const float sum = rows.exponentiate(s, p);
      // Keeps the exponentials here, among the products (they would be sunk
      // past the next branch).
#pragma unroll
      for (int h = 0; h < 2 * RowsT::kBlocks; ++h) asm volatile("" : : "v"(p.p[h]));
      read_v(vt, va);
      // (of tile i + 1, or a later one's)
      flag = sh.bad[own * RW + (lane & (RW - 1))];
      fetch(1, i + kSlots - 1);
      if ((i + kSlots) % kPer == 0) look_up((i + kSlots) / kPer);
      fetch(0, i + kSlots);
      rows.settle_sum(sum, s, p);
      output(vt, va, p);
      s = next;
    }
  }
  // Nothing may still write the tiles: partial results of the key groups meet
  // there.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
  float mm, l_tot;
  float a[KW];
  if constexpr (KW > 1) {
    if constexpr (RW > 1) __syncthreads();  // (with RW == 1 a wave's slots are its own)
    // (16 KiB a wave: its own slots, with RW == 1)
    float4* const to = reinterpret_cast<float4*>(sh.tile) + 1024 * w;
#pragma unroll
    for (int c = 0; c < kAcc / 4; ++c) {
      const float16_t& x = rows.o[c >> 2];
      const int r = 4 * (c & 3);
      to[c * 64 + lane] = make_float4(x[r], x[r + 1], x[r + 2], x[r + 3]);
    }
    sh.ml[w][lane] = make_float2(rows.mc, rows.l);
    __syncthreads();
    // They meet at their largest stabiliser; one without a visible key (l = 0
    // across the lane pair) is passed over.
    mm = ninf();
    float lt = 0.0f;
    float2 ml[KW];
    bool has[KW];
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      ml[j] = sh.ml[j * RW + rw][lane];
      has[j] = pair_sum(ml[j].y) != 0.0f;
      if (has[j]) mm = fmaxf(mm, ml[j].x);
    }
#pragma unroll
    for (int j = 0; j < KW; ++j) {
      a[j] = has[j] ? __builtin_amdgcn_exp2f(ml[j].x - mm) : 0.0f;
      lt += a[j] * ml[j].y;
    }
    l_tot = pair_sum(lt);
  } else {
    l_tot = pair_sum(rows.l);
    mm = rows.mc;
  }
  const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
  T* const orow = O + (b * g.o_sb + head * g.o_sh + draft * g.o_sr);
  float* const prow = part ? part + (long long)local * kPart : nullptr;
  // 8 columns of a row: 32 (c / 2) + 16 (c % 2) + 8 g.
  auto put = [&](int c, const float (&acc)[8]) __attribute__((always_inline)) {
    const int col = 32 * (c >> 1) + 16 * (c & 1) + 8 * rows.g;
    if (prow) {
      *reinterpret_cast<float4*>(prow + col) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(prow + col + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
    } else {
      V8 out;
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = (T)(acc[e] * inv);
      *reinterpret_cast<V8*>(orow + col) = out;
    }
  };
  if constexpr (KW > 1) {
    for (int c = kg; c < D / 16; c += KW) {
      float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        const float4* const pj = reinterpret_cast<const float4*>(sh.tile) + 1024 * (j * RW + rw);
        const float4 x0 = pj[(2 * c) * 64 + lane], x1 = pj[(2 * c + 1) * 64 + lane];
        acc[0] += a[j] * x0.x;
        acc[1] += a[j] * x0.y;
        acc[2] += a[j] * x0.z;
        acc[3] += a[j] * x0.w;
        acc[4] += a[j] * x1.x;
        acc[5] += a[j] * x1.y;
        acc[6] += a[j] * x1.z;
        acc[7] += a[j] * x1.w;
      }
      if (mine) put(c, acc);
    }
  } else if (mine) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      float acc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = rows.o[c >> 1][8 * (c & 1) + e];
      put(c, acc);
    }
  }
  if (kg == 0 && rows.g == 0 && mine) {
    if (prow) {
      prow[D] = l_tot == 0.0f ? ninf() : mm;
      prow[D + 1] = l_tot;
    } else if (g.lse != nullptr) {
      g.lse[((long long)b * g.heads + head) * g.drafts + draft] =
          l_tot == 0.0f ? ninf() : 0.693147180559945309f * (mm + __builtin_amdgcn_logf(l_tot));
    }
  }
}

// The launch's work-group, counted so that neighbours run on one XCD.
__device__ __forceinline__ int group_index(int xcds) {
  const int per = gridDim.x / xcds;
  return per * xcds == (int)gridDim.x ? (blockIdx.x % xcds) * per + blockIdx.x / xcds : blockIdx.x;
}

// A unit a work-group.
template <int D, class T, int RW>
__global__ void __launch_bounds__(64 * waves_of(RW), 2)
tree_fwd_kernel(const T* Q, const uint8_t* K, const uint8_t* V, T* O, const TreeGeom g, float cq,
                float cr) {
  __shared__ __attribute__((aligned(16))) Shared<D, RW, false> sh;
  const int per = g.kv_units * g.blocks_of_rows;
  const int unit = group_index(g.xcds);
  const int b = unit / per, rest = unit - b * per;
  const int kvh = rest / g.blocks_of_rows, rb = rest - kvh * g.blocks_of_rows;
  const Request r = request(g, b);
  const int steps = unit_steps<D, RW, false>(g, r, rb);
  if (steps > 0)
    walk<D, T, RW, false>(Q, K, V, O, g, sh, b, kvh, rb, r, 0, steps, nullptr, cq, cr);
}

// The costs of all units, in order, are dealt evenly to the work-groups: each
// has the end of one unit, whole units, the start of one.  Whole units are
// stored; partial results go to slot 2 x of work-group x (its first unit's) or
// 2 x + 1 (its last's, if another).  Whoever has a unit's first step says in
// parts[unit].x in which slot its results begin, whoever has its last in .y
// which work-group that was; between them each work-group has one in its first
// slot.  (The sum is below 2^31: tree_plan.)
template <int D, class T, int RW, bool DEEP>
__global__ void __launch_bounds__(64 * waves_of(RW), 2)
tree_split_kernel(const T* Q, const uint8_t* K, const uint8_t* V, T* O, const TreeGeom g, float cq,
                  float cr) {
  constexpr int kHeads = heads_of(RW, DEEP);
  __shared__ __attribute__((aligned(16))) Shared<D, RW, DEEP> sh;
  const int lane = threadIdx.x & 63;
  // Cost of one key/value head of requests b0 .. b0 + 63, one a lane.
  Request c;
  int n, upto;
  auto chunk = [&](int b0) __attribute__((always_inline)) {
    c = request(g, min(b0 + lane, g.batch - 1));
    n = b0 + lane < g.batch ? head_cost<D, RW, DEEP>(g, c) : 0;
    upto = wave_scan(n);
  };
  auto last_lane = [](int x) __attribute__((always_inline)) {
    return __builtin_amdgcn_readlane(x, 63);
  };
  int all = 0;
#pragma unroll 1
  for (int b0 = (g.batch - 1) & ~63; b0 >= 0; b0 -= 64) {  // (ends with the first 64)
    chunk(b0);
    all += last_lane(upto);
  }
  all *= g.kv_units;
  // `busy` work-groups have a share, `even` or one more; neighbours run on one
  // XCD, all XCDs alike.
  const int busy = min((int)gridDim.x, all);
  const int apiece = (busy + g.xcds - 1) / g.xcds;
  const int k = blockIdx.x / g.xcds;
  const int x = (blockIdx.x - k * g.xcds) * apiece + k;
  if (k >= apiece || x >= busy) return;
  const int even = (uint32_t)all / (uint32_t)busy, more = all - even * busy;
  int at = x * even + min(x, more);
  const int end = at + even + (x < more ? 1 : 0);
  // The request of `at`, and where in it that is.
  int b0 = 0, before = 0;
  uint64_t past;
#pragma unroll 1
  while ((past = __builtin_amdgcn_ballot_w64(before + upto * g.kv_units > at)) == 0) {
    before += last_lane(upto) * g.kv_units;
    b0 += 64;
    chunk(b0);
  }
  const int l = __builtin_ctzll(past);
  int b = b0 + l;
  Request r;
  r.length = __builtin_amdgcn_readlane(c.length, l);
  r.count = __builtin_amdgcn_readlane(c.count, l);
  const int head = __builtin_amdgcn_readlane(n, l);
  int in = at - before - __builtin_amdgcn_readlane(upto - n, l) * g.kv_units;
  int kvh = 0, rb = 0, steps, cost;
#pragma unroll 1
  while (in >= head) {
    in -= head;
    ++kvh;
  }
#pragma unroll 1
  while (in >= (cost = cost_of<RW>(steps = unit_steps<D, RW, DEEP>(g, r, rb)))) {
    in -= cost;
    ++rb;
  }
  int slot = 2 * x;
#pragma unroll 1
  for (;;) {
    // Costs [in, upto) of the unit; its start comes first.
    const int to = min(cost, in + (end - at));
    const int s0 = max(in - start_of(RW), 0), s1 = to - start_of(RW);
    if (s1 > s0) {
      if (threadIdx.x == 0) {
        int2* const where = g.parts + (b * g.kv_units + kvh) * g.blocks_of_rows + rb;
        if (s0 == 0) where->x = slot;
        if (s1 == steps) where->y = x;
      }
      float* const part =
          s0 == 0 && s1 == steps ? nullptr : g.part + (long long)slot * g.part_size;
      walk<D, T, RW, DEEP>(Q, K, V, O, g, sh, b, kvh * kHeads, rb, r, s0, s1, part, cq, cr);
      slot = 2 * x + 1;
    }
    at += to - in;
    if (at >= end) return;
    in = 0;
    // The next unit with steps.
    do {
      if (++rb == g.blocks_of_rows) {
        rb = 0;
        if (++kvh == g.kv_units) {
          kvh = 0;
          r = request(g, ++b);
        }
      }
      cost = cost_of<RW>(steps = unit_steps<D, RW, DEEP>(g, r, rb));
    } while (cost == 0);
    __syncthreads();  // the tiles are free again
  }
}

// One wave a row: merges the partial results of its unit, if it was split.
template <int D, class T, int RW, int HEADS>
__global__ void __launch_bounds__(256) tree_merge_kernel(T* O, const TreeGeom g) {
  constexpr int kPart = D == 64 ? kPartStride : kPartStride128;
  constexpr int kCols = D / 64, kBatch = 8;
  const int lane = threadIdx.x & 63;
  const int b = blockIdx.y;
  const int rest = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (rest >= g.heads * g.drafts) return;
  const int head = divide(rest, g.by_drafts), draft = rest - head * g.drafts;
  const int kvh = divide(head, g.group);
  const int row = draft * g.group.d + (head - kvh * g.group.d);
  const int rb = row / (32 * RW);
  const int count = g.counts ? g.counts[b] : g.drafts;
  const int2 parts = g.parts[(b * g.kv_units + kvh / HEADS) * g.blocks_of_rows + rb];
  if (draft >= count) return;  // (its unit's entry may not be there either)
  // Part j: the first in slot parts.x, then the first slots of the work-groups
  // that follow.
  const int x0 = parts.x >> 1, n = parts.y - x0 + 1;
  if (n == 1) return;  // one work-group had all of it
  const float* const base =
      g.part + (long long)(row - rb * 32 * RW + kvh % HEADS * g.part_rows) * kPart;
  auto at = [&](int j) __attribute__((always_inline)) {
    return base + (long long)(j == 0 ? parts.x : 2 * (x0 + j)) * g.part_size;
  };
  float acc[kCols] = {}, l = 0.0f, mx = ninf();
#pragma unroll 1
  for (int j0 = 0; j0 < n; j0 += 64) {
    // Lane j's part's stabiliser and sum; O of the first parts meanwhile.
    float m = ninf(), lj = 0.0f, a = 0.0f;
    if (j0 + lane < n) {
      const float2 ml = *reinterpret_cast<const float2*>(at(j0 + lane) + D);
      m = ml.x;
      lj = ml.y;
    }
    const int most = min(n - j0, 64);
#pragma unroll 1
    for (int from = 0; from < most; from += kBatch) {
      float o[kBatch][kCols];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float* const p = at(j0 + min(from + u, most - 1));
#pragma unroll
        for (int c = 0; c < kCols; ++c) o[u][c] = p[lane + 64 * c];
      }
      if (from == 0) {
        float top = lj != 0.0f ? m : ninf();
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
        top = fmaxf(top, mx);
        const float again = mx == top ? 1.0f : __builtin_amdgcn_exp2f(mx - top);
        mx = top;
        l *= again;
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[c] *= again;
        // (weights are not negative: -1 marks a part without a visible key)
        a = lj != 0.0f ? __builtin_amdgcn_exp2f(m - mx) : -1.0f;
        float sum = a < 0.0f ? 0.0f : a * lj;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
        l += sum;
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const float w = from + u < most
                            ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), from + u))
                            : -1.0f;
#pragma unroll
        for (int c = 0; c < kCols; ++c) acc[c] += w < 0.0f ? 0.0f : w * o[u][c];
      }
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* const out = O + (b * g.o_sb + head * g.o_sh + draft * g.o_sr);
#pragma unroll
  for (int c = 0; c < kCols; ++c) out[lane + 64 * c] = (T)(acc[c] * inv);
  if (lane == 0 && g.lse != nullptr)
    g.lse[(long long)b * g.heads * g.drafts + rest] =
        l == 0.0f ? ninf() : 0.693147180559945309f * (mx + __builtin_amdgcn_logf(l));
}

// How a call of given sizes runs: row blocks a work-group, and whether the
// units' steps are dealt to a grid of one work-group a CU, of kMostParts to a
// unit on average at most.  The merge reads a row's partial results one batch
// after another, so past some parts it takes longer than the walks they
// shorten.  8 heads over one KV head (D 128, bf16), one token after 32000: 31
// us with 256 parts, 17.0 with 64, 18.6 with 32, 25.0 with 16; 64 drafts there
// (f16) 39.9, 35.7, 45.4 and 69.9.  (The host does not know the lengths: beside
// 3 requests of 1 token that one unit still gets some 250 parts, 30.3 us.)
constexpr int kMostParts = 64;
// Floats of a cache line, on which a partial result begins.
constexpr int kPartUnit = 32;

struct TreePlan {
  int rw, units, grid;
  int most_grid, heads;  // what the workspace has room for: work-groups, heads of each;
  int part_rows, part_size;  // rows of each, floats of a partial result
  bool split;
  int64_t parts_at, bytes;
};

TreePlan tree_plan(const fl_tree_params& p) {
  TreePlan t;
  const int64_t rows = p.heads / p.kv_heads * p.drafts;
  t.rw = rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
  t.units = (int)((rows + 32 * t.rw - 1) / (32 * t.rw) * p.kv_heads * p.batch);
  t.grid = (int)std::min<int64_t>(device_cus(), (int64_t)kMostParts * t.units);
  // (see launch_rw)
  t.most_grid = t.rw == 2 && p.head_dim == 64
                    ? (int)std::min<int64_t>(2 * device_cus(), (int64_t)kMostParts * t.units)
                    : t.grid;
  t.heads = t.rw == 1 && p.kv_heads % heads_of(1, true) == 0 && p.k_stride[1] < p.k_stride[2]
                ? heads_of(1, true)
                : 1;
  t.part_rows = (int)std::min<int64_t>(rows, 32 * t.rw);
  t.split = t.units < 2 * t.grid || t.heads > 1;
  const int64_t part = p.head_dim == 64 ? kPartStride : kPartStride128;
  t.part_size = (int)((t.part_rows * t.heads * part + kPartUnit - 1) / kPartUnit * kPartUnit);
  t.parts_at = 2LL * t.most_grid * t.part_size * (int64_t)sizeof(float);
  t.bytes = t.split ? t.parts_at + t.units * (int64_t)sizeof(int2) : 0;
  return t;
}

// One pass, or (grid > 0) the units' steps dealt to `grid` work-groups and
// joined.
template <int D, class T, int RW, bool DEEP>
hipError_t launch_walk(const fl_tree_params& p, const TreePlan& t, TreeGeom& g, int grid,
                       float cq, float cr, hipStream_t st) {
  const dim3 threads(64 * waves_of(RW));
  g.kv_units = (int)p.kv_heads / heads_of(RW, DEEP);
  if (grid % g.xcds != 0) g.xcds = 1;  // (all XCDs alike, or none told apart)
  const T* q = static_cast<const T*>(p.q);
  const uint8_t *k = static_cast<const uint8_t*>(p.k_cache),
                *v = static_cast<const uint8_t*>(p.v_cache);
  T* o = static_cast<T*>(p.o);
  if constexpr (!DEEP) {
    if (grid == 0) {
      hipLaunchKernelGGL((tree_fwd_kernel<D, T, RW>), dim3((unsigned)t.units), threads, 0, st, q, k,
                         v, o, g, cq, cr);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((tree_split_kernel<D, T, RW, DEEP>), dim3((unsigned)grid), threads, 0, st, q, k,
                     v, o, g, cq, cr);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const unsigned rows = (unsigned)(g.heads * g.drafts);
  hipLaunchKernelGGL((tree_merge_kernel<D, T, RW, heads_of(RW, DEEP)>), dim3((rows + 3) / 4, (unsigned)g.batch),
                     dim3(256), 0, st, o, g);
  return hipGetLastError();
}

template <int D, class T, int RW>
hipError_t launch_rw(const fl_tree_params& p, const TreePlan& t, TreeGeom& g, float cq, float cr,
                     hipStream_t st) {
  constexpr int kStepKeys = key_groups_of(RW, false) * (D == 64 ? kBc : kBc2);
  // Steps of the longest unit that the table has room for.
  const int64_t most = ((int64_t)g.capacity + g.drafts) / kStepKeys + 1;
  // A split launch adds up costs in 32 bits.
  const bool counted = t.units * (most + start_of(RW)) < (1LL << 30);
  // Splitting costs the partial results' way through memory and a second
  // launch, about four microseconds; it saves the steps by which the longest
  // unit passes an even share.  Up to kFewSaved one pass is no slower: 16
  // requests x 16 heads of 600 keys (D 128, f16) 15.5 us against 20.4, 4 x 16
  // drafts of 16/4 heads after 300 keys 9.4 against 13.3, 1 head of 1000 keys
  // 8.2 against 9.7; with twice that bound 8 drafts of 32/8 heads after 1000
  // keys lose, 12.8 against 11.8.  With as many units as work-groups the share
  // says nothing about requests of unlike lengths, so kMostSteps bounds what
  // waiting for the longest can cost: up to it 32 drafts of 32 x 32/8 heads
  // after 500 keys take 21.3 us against 26.5, while 16 heads and 1 to 16384
  // keys (128 steps) lose, 129 against 110.  The longest unit is taken to be as
  // long as the tables have room for: in tables 4 times as wide as the requests
  // need, short calls take the other side's time.
  constexpr int kFewSaved = 6, kMostSteps = 32;
  const int64_t share = (most * t.units + t.grid - 1) / t.grid;
  const bool can = g.part != nullptr && counted;
  const bool split = can && t.units < 2 * t.grid &&
                     (most > kMostSteps || most - share > kFewSaved);
  int grid = split ? t.grid : 0;
  // Long walks of 64 rows are bound by the keys on their way: at D 128 4 slots
  // instead of 2, at D 64 two work-groups a CU.  Short ones pay for the longer
  // start, or the parts.  12 drafts of 32/8 heads (bf16) for 16 requests of
  // 2000-4000 tokens 56.5 us against 64.7 (D 64: 35.9 against 42.6), for 8 of
  // 1000-2000 23.7 against 25.8 (D 64: 17.9 against 18.0), for 4 of 1500-3000
  // 21.9 against 20.7 (D 64: 17.8 against 16.6).
  if constexpr (RW == 2) {
    if (split && share * kStepKeys >= 512) {
      if constexpr (slots_of(D, RW, true) != slots_of(D, RW, false))
        return launch_walk<D, T, RW, true>(p, t, g, grid, cq, cr, st);
      grid = t.most_grid;
    }
  }
  // Up to 32 rows over long walks are bound by memory, and where a token's
  // heads lie side by side (the cache's rows first) a head's row is 128 or 256
  // bytes of it: 4 heads at once read 4 times that in one piece, a wave each.
  // One token after 8000 of 32 requests, 32/8 heads (bf16): D 64 98.7 us
  // against 109.7, D 128 181 against 191; 16 requests of 2000-4000: 26.5
  // against 29.9, 43.7 against 45.8.  Heads first they lose, 96 against 91, as
  // do shares (4 requests of 2000-4000: 16.2 against 14.1) or walks that are
  // short (512 of 100-500: 70 against 65), and units too few for kMostParts
  // each (1 of 64000: 39.2 against 36.3).
  if constexpr (RW == 1) {
    const int64_t units = t.units / heads_of(RW, true);
    if (can && t.heads > 1 && share * kStepKeys >= 2048 && most * kStepKeys > 2048 &&
        units * kMostParts >= t.grid)
      return launch_walk<D, T, RW, true>(p, t, g, t.grid, cq, cr, st);
  }
  return launch_walk<D, T, RW, false>(p, t, g, grid, cq, cr, st);
}

template <int D, class T>
hipError_t launch_t(const fl_tree_params& p, TreeGeom& g, float cq, float cr, hipStream_t st) {
  const TreePlan t = tree_plan(p);
  g.blocks_of_rows = (g.rows + 32 * t.rw - 1) / (32 * t.rw);
  g.part_rows = t.part_rows;
  g.part_size = t.part_size;
  g.parts = reinterpret_cast<int2*>(reinterpret_cast<uint8_t*>(g.part) + t.parts_at);
  return t.rw == 1   ? launch_rw<D, T, 1>(p, t, g, cq, cr, st)
         : t.rw == 2 ? launch_rw<D, T, 2>(p, t, g, cq, cr, st)
         : t.rw == 4 ? launch_rw<D, T, 4>(p, t, g, cq, cr, st)
                     : launch_rw<D, T, 8>(p, t, g, cq, cr, st);
}

}  // namespace

int64_t tree_workspace_bytes(const fl_tree_params& p) { return tree_plan(p).bytes; }

hipError_t launch_tree_fwd(const fl_tree_params& p, void* ws, hipStream_t st) {
  TreeGeom g = {};
  g.part = static_cast<float*>(ws);
  g.xcds = device_xcds();
  g.q_sb = p.q_stride[0];
  g.q_sh = p.q_stride[1];
  g.q_sr = p.q_stride[2];
  g.o_sb = p.o_stride[0];
  g.o_sh = p.o_stride[1];
  g.o_sr = p.o_stride[2];
  g.k_blk = (uint32_t)(2 * p.k_stride[0]);
  g.k_head = 2 * p.k_stride[1];
  g.k_row = (uint32_t)(2 * p.k_stride[2]);
  g.v_blk = (uint32_t)(2 * p.v_stride[0]);
  g.v_head = 2 * p.v_stride[1];
  g.v_row = (uint32_t)(2 * p.v_stride[2]);
  g.tables = p.block_tables;
  g.table_stride = p.table_stride;
  g.lengths = p.lengths;
  g.counts = p.counts;
  g.mask = p.mask;
  g.mask_stride = p.mask_stride;
  g.lse = p.lse;
  g.batch = (int)p.batch;
  g.heads = (int)p.heads;
  g.drafts = (int)p.drafts;
  g.group = fast_div((int)(p.heads / p.kv_heads));
  g.by_drafts = fast_div(g.drafts);
  g.rows = g.group.d * g.drafts;
  g.words = (g.drafts + 63) / 64;
  g.num_blocks = (int)p.num_blocks;
  g.capacity = (int)(p.max_blocks * p.block_size);
  g.block = fast_div((int)p.block_size);
  const double s = p.sm_scale == 0.0 ? (double)(1.0f / std::sqrt((float)p.head_dim)) : p.sm_scale;
  const float cr = (float)(std::fabs(s) * 1.44269504088896340736), cq = s < 0.0 ? -1.0f : 1.0f;
  const bool bf = p.dtype == FL_DTYPE_BF16;
  if (p.head_dim == 128)
    return bf ? launch_t<128, __bf16>(p, g, cq, cr, st) : launch_t<128, _Float16>(p, g, cq, cr, st);
  return bf ? launch_t<64, __bf16>(p, g, cq, cr, st) : launch_t<64, _Float16>(p, g, cq, cr, st);
}

}  // namespace fl
