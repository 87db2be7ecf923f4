// Gradients of attention over packed sequences (fl_attn_packed_bwd), one
// source file per element type (packed_bwd_f16.hip, packed_bwd_bf16.hip).
//
// With p = exp(s - lse), s = scale q.k, delta = dout . out a row and
// ds = p (dout v' - delta):
//   dv = p' dout    dk = scale ds' q    dq = scale ds k
// p is taken again from q, k and lse, so nothing of the size of the scores is
// kept.  Two kinds of work-groups, each of which owns what it sums, so no atomics
// and the same bits every time: one walks a query block's keys (3 products a
// pair: s, dout v', dq) and leaves -lse / scale and -delta of its rows for the
// other, which walks a key block's queries over all heads of its group (4
// products: s, dout v', dv, dk) in a launch behind it.  14 D flops a pair of a row
// and a key, 7 products where one kernel with atomics would do with 5.  Little
// work is one launch of both kinds, with delta taken by either.
//
// Bound by the matrix cores and what feeds them: B4 H32/8 N4096 D 128 bf16 causal
// 1780 us, 1.08 PFLOP/s of the 7 products, where a large library product has
// 1.2; 16 sequences of 64-2000, H32/8 675 (a block's triangle and the sequences'
// ends are walked whole), B2 H16/2 N7000-8192 fp16 1580; few short ones by
// launches and chains of loads (4 of 33-257, H8/2 D 64 17.5 us).
//
// Both kernels keep two waves a SIMD, the products of one among the exponentials
// of the other.  One wave with 64 bytes more registers a lane, dv and dk one
// block behind s and dout v' and the exponentials spread over all products, took
// 2020 where two waves then took 1810 (16 sequences 830 against 718: a work-group
// alone on its CU leaves it idle at its start and end).
//
// Operands as in the forward kernels: a wave's own 32 rows stay in registers
// as B operands, tiles of the others come into LDS by DMA and are read as rows
// (A of the score products) and transposed (A of the products that sum over
// the tile's rows), the scores' accumulators being in the order that the
// latter take.  Both reads of a tile go through one swizzle.
#pragma once

#include "packed.h"

namespace fl {

namespace {

struct BwdGeom {
  const void *q, *k, *v, *o, *dout;
  void *dq, *dk, *dv;
  const float* lse;       // [heads][rows]
  float2* stats;          // [heads][rows]: -lse / scale, -delta
  float* part;            // [parts][kv_heads][key_rows][2 D], or null
  long long q_sh, k_sh, v_sh, o_sh, do_sh, dq_sh, dk_sh, dv_sh;  // elements
  int q_sr, k_sr, v_sr, o_sr, do_sr, dq_sr, dk_sr, dv_sr;
  const int32_t* starts;
  const int32_t* key_starts;
  int sequences, rows, key_rows, heads, kv_heads, group, parts, causal, xcds;
  float scale, scale_log2;
};

// A tile: 8 KiB of rows of D columns, 16-byte chunks XOR-swizzled so that both
// reads are free of conflicts.  Rows (ds_read_b128, 16 rows at one chunk): 16
// different places of the 256 bytes that a sweep of the banks covers.
// Transposed (ds_read_b64_tr_b16, 4 rows of 4 chunks): 4 rows in different
// quarters of them.
template <int D>
__device__ __forceinline__ int both_swz(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3)
                  : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

template <int D, class T>
struct BwdLane {
  using E = Elem<T>;
  using V8 = typename E::v8;
  using V4 = typename E::v4;
  static constexpr int kRowB = 2 * D;
  static constexpr int kRows = kTileBytes / kRowB;  // of a tile
  static constexpr int kBlocks = kRows / 32, kSteps = D / 16, kCols = D / 32;
  int lane, g, col, tr_row, tr_col;

  __device__ __forceinline__ explicit BwdLane(int lane_) {
    lane = lane_;
    g = lane >> 5;
    col = lane & 31;
    const int G = lane >> 4, j = lane & 15, x = j & 3;
    tr_row = 4 * (G >> 1) + (j >> 2);
    tr_col = 16 * (G & 1) + 4 * (((x & 1) << 1) | (x >> 1));
  }
  // 32 rows of block b at columns 16 st ..
  __device__ __forceinline__ V8 rows_op(const uint8_t* tile, int b, int st) const {
    const int row = 32 * b + col;
    return *reinterpret_cast<const V8*>(tile + row * kRowB +
                                        16 * ((2 * st + g) ^ both_swz<D>(row)));
  }
  // Columns 32 c .. of rows 16 t .., transposed.
  __device__ __forceinline__ V8 cols_op(const uint8_t* tile, int c, int t) const {
    const int r1 = 16 * t + tr_row, r2 = r1 + 8, x = 32 * c + tr_col;
    const int ch = x >> 3, hb = ((x >> 2) & 1) * 8;
    const V4 lo = lds_read_tr<V4>(tile + r1 * kRowB + 16 * (ch ^ both_swz<D>(r1)) + hb);
    const V4 hi = lds_read_tr<V4>(tile + r2 * kRowB + 16 * (ch ^ both_swz<D>(r2)) + hb);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // Row `row` of x as a B operand (zeros past the last).
  __device__ __forceinline__ void own_rows(const T* x, long long sr, int row, int rows,
                                           V8 (&op)[kSteps]) const {
#pragma unroll
    for (int st = 0; st < kSteps; ++st) {
      op[st] = (V8){0, 0, 0, 0, 0, 0, 0, 0};
      if (row < rows) op[st] = *reinterpret_cast<const V8*>(x + row * sr + 16 * st + 8 * g);
    }
  }
  // acc (32 columns a block, times `scale`) to row `row`.
  __device__ __forceinline__ void store(T* x, long long sr, int row, int rows, float scale,
                                        const float16_t (&acc)[kCols]) const {
    if (row >= rows) return;
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        V8 out;
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = (T)(acc[c][8 * h + e] * scale);
        *reinterpret_cast<V8*>(x + row * sr + 32 * c + 16 * h + 8 * g) = out;
      }
  }
  __device__ __forceinline__ void store_part(float* x, int row, int rows,
                                             const float16_t (&acc)[kCols]) const {
    if (row >= rows) return;
#pragma unroll
    for (int c = 0; c < kCols; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 8; e += 4)
          *reinterpret_cast<float4*>(x + (long long)row * (2 * D) + 32 * c + 16 * h + 8 * g + e) =
              make_float4(acc[c][8 * h + e], acc[c][8 * h + e + 1], acc[c][8 * h + e + 2],
                          acc[c][8 * h + e + 3]);
  }
};

// The same operands by LDS address: what varies from lane to lane is kept in
// registers, a tile's place is added.
template <int D, class T>
struct TileOps {
  using L = BwdLane<D, T>;
  using V8 = typename L::V8;
  using V4 = typename L::V4;
  typedef const V8 __attribute__((address_space(3))) * LdsV8;
  typedef short4_t __attribute__((address_space(3))) * LdsTr;
  uint32_t row_at[L::kSteps], col_at[L::kCols][2];

  __device__ __forceinline__ explicit TileOps(const L& ln) {
#pragma unroll
    for (int st = 0; st < L::kSteps; ++st)
      row_at[st] = ln.col * L::kRowB + 16 * ((2 * st + ln.g) ^ both_swz<D>(ln.col));
#pragma unroll
    for (int c = 0; c < L::kCols; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = ln.tr_row + 8 * h, x = 32 * c + ln.tr_col;
        col_at[c][h] = row * L::kRowB + 16 * ((x >> 3) ^ both_swz<D>(row)) + 8 * ((x >> 2) & 1);
      }
  }
  // Rows 32 b .. at columns 16 st .., `off` bytes behind the tile.
  __device__ __forceinline__ V8 rows(uint32_t tile, int off, int b, int st) const {
    return *(LdsV8)(uintptr_t)(tile + row_at[st] + (off + 32 * b * L::kRowB));
  }
  // Columns 32 c .. of rows 16 t .., transposed.
  __device__ __forceinline__ V8 cols(uint32_t tile, int off, int c, int t) const {
    const uint32_t o = off + 16 * t * L::kRowB;
    const V4 a = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                            (LdsTr)(uintptr_t)(tile + col_at[c][0] + o)));
    const V4 b = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                            (LdsTr)(uintptr_t)(tile + col_at[c][1] + o)));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

__device__ __forceinline__ float16_t zero16() {
  return (float16_t){0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
}

// A resource of `n` rows, row_bytes apart, of kRowB bytes each, that the next
// instruction may load through: five wait states belong between a vector
// instruction that writes a scalar register and a load that reads it, and the
// compiler, which may take vector ones for this, does not add them before
// inline assembly.
template <int kRowB>
__device__ __forceinline__ i32x4_t rows_rsrc(const void* x, int n, int row_bytes) {
  i32x4_t rs = buffer_rsrc(x, n > 0 ? (n - 1) * row_bytes + kRowB : 0);
  asm volatile("s_nop 4" : "+s"(rs));
  return rs;
}

// At most `most` of the `left` rows (scalar: not a vector median).
__device__ __forceinline__ int tile_rows(int left, int most) {
  left = __builtin_amdgcn_readfirstlane(min(left, most));
  asm("" : "+s"(left));
  return max(left, 0);
}

// A pointer that is the same in every lane, in scalar registers.
__device__ __forceinline__ uint8_t* uniform(uint8_t* x) {
  const uint64_t a = (uint64_t)(uintptr_t)x;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
  return (uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// DMA of tiles: wave w moves kSegs segments of 1 KiB of a tile, each lane 16
// bytes.
template <int D, int kSegs>
struct TileFetch {
  int lane[kSegs];
  __device__ __forceinline__ TileFetch(int wave, int l, int row_bytes) {
    constexpr int kChunks = D / 8, kSegRows = 64 / kChunks;
#pragma unroll
    for (int i = 0; i < kSegs; ++i) {
      const int row = kSegRows * (wave * kSegs + i) + l / kChunks;
      lane[i] = row * row_bytes + 16 * ((l % kChunks) ^ both_swz<D>(row));
      asm volatile("" : "+v"(lane[i]));  // (kept, not derived again)
    }
  }
  __device__ __forceinline__ void seg(const i32x4_t& rs, const uint8_t* slot, int wave,
                                      int i) const {
    load_lds16(rs, lane[i], slot + 1024 * (wave * kSegs + i));
  }
  __device__ __forceinline__ void run(const i32x4_t& rs, const uint8_t* slot, int wave) const {
#pragma unroll
    for (int i = 0; i < kSegs; ++i) seg(rs, slot, wave, i);
  }
};

// Rows row0 .. of the `rows` rows of x, at most `most`, as a resource.
template <int kRowB, class T>
__device__ __forceinline__ i32x4_t tile_rsrc(const T* x, int row_bytes, int row0, int rows,
                                             int most) {
  return rows_rsrc<kRowB>(reinterpret_cast<const uint8_t*>(x) + (long long)row0 * row_bytes,
                          tile_rows(rows - row0, most), row_bytes);
}

// 4 bytes a lane into LDS at slot + 4 * lane (as load_lds16).
__device__ __forceinline__ void load_lds4(const i32x4_t& rs, int voff, const uint8_t* slot) {
  const uint32_t lds_base = (uint32_t)(uintptr_t)slot;
  asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
               : : "v"(voff), "s"(rs), "{m0}"(lds_base));
}

// A block's transposed operands (32 rows from `rows` on) before a product
// whose other factor is 0 for rows that a lane's own row does not see: NaN and
// infinities become 0, and are added to the lanes that see their row (as NaN
// where the factor may have any sign).
template <int D, class T, class Sees>
__device__ __forceinline__ void add_odd_block(const uint8_t* rows,
                                              typename Elem<T>::v8 (&op)[D / 16],
                                              float16_t (&acc)[D / 32], int g, Sees&& sees,
                                              bool as_nan) {
  using V8 = typename Elem<T>::v8;
#pragma unroll
  for (int u = 0; u < D / 16; ++u) op[u] = finite_only<T>(op[u]);
#pragma unroll 1
  for (int j = 0; j < 32; ++j) {
    const bool mine = sees(j);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const V8 x =
          *reinterpret_cast<const V8*>(rows + j * 2 * D + 16 * ((2 * c + g) ^ both_swz<D>(j)));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = (float)x[e];
        if (mine && !(__builtin_fabsf(y) < __builtin_huge_valf()))
          acc[c >> 1][8 * (c & 1) + e] += as_nan ? y - y : y;
      }
    }
  }
}

// A work-group's query block of the dq kernel.
struct DqTask {
  int head, kv, q0, nq, k0, nk, coff, first, tiles;
};

template <int D, int W>
__device__ __forceinline__ bool dq_task(const BwdGeom& p, int group, DqTask& x) {
  int r;
  PackedAt at;
  packed_unit(group, p.heads, p.xcds, r, x.head);
  if (!packed_block<32 * W>(p.starts, p.rows, p.key_starts, p.key_rows, p.sequences, r, p.causal,
                            at))
    return false;
  x.q0 = at.begin;
  x.nq = at.count;
  x.k0 = at.other;
  x.nk = at.others;
  x.coff = p.causal ? x.nk - x.nq : x.nk;  // query i sees keys up to i + coff
  x.kv = x.head / p.group;
  x.first = at.j * 32 * W;
  constexpr int kRows = kTileBytes / (2 * D);
  x.tiles = max((min(x.nk, min(x.first + 32 * W, x.nq) + x.coff) + kRows - 1) / kRows, 0);
  return true;
}

// This lane's rows of a query block: q and dout as B operands, lse in base 2
// and delta.
template <int D, class T>
struct DqRows {
  using L = BwdLane<D, T>;
  typename L::V8 qf[L::kSteps], df[L::kSteps];
  float lse, lse2, delta;

  __device__ __forceinline__ void load(const BwdGeom& p, const DqTask& x, const L& ln, int my) {
    typename L::V8 of[L::kSteps];
    ln.own_rows(static_cast<const T*>(p.q) + (x.head * p.q_sh + (long long)x.q0 * p.q_sr), p.q_sr,
                my, x.nq, qf);
    ln.own_rows(static_cast<const T*>(p.dout) + (x.head * p.do_sh + (long long)x.q0 * p.do_sr),
                p.do_sr, my, x.nq, df);
    ln.own_rows(static_cast<const T*>(p.o) + (x.head * p.o_sh + (long long)x.q0 * p.o_sr), p.o_sr,
                my, x.nq, of);
    float sum = 0.0f;
#pragma unroll
    for (int st = 0; st < L::kSteps; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = __builtin_fmaf((float)df[st][e], (float)of[st][e], sum);
    delta = pair_sum(sum);
    lse = my < x.nq ? p.lse[(long long)x.head * p.rows + x.q0 + my] : 0.0f;
    // (a row that sees nothing: p = 2^-inf)
    lse2 = lse == ninf() ? -ninf() : lse * 1.44269504088896341f;
  }
};

// The dq kernel's block walked again, with NaN and infinities of keys that rows
// do not see kept from them.  (A function of its own: its registers are not
// the kernel's.)
template <int D, int W, class T>
__device__ __attribute__((noinline)) void dq_checked(const void* geom, int group, uint8_t* lds) {
  using L = BwdLane<D, T>;
  using V8 = typename L::V8;
  using E = Elem<T>;
  lds = uniform(lds);
  group = __builtin_amdgcn_readfirstlane(group);
  BwdGeom p;
  __builtin_memcpy(&p, geom, sizeof p);
  DqTask x;
  if (!dq_task<D, W>(p, group, x)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const L ln(threadIdx.x & 63);
  const int my = x.first + 32 * wave + ln.col;
  const T* const K = static_cast<const T*>(p.k) + (x.kv * p.k_sh + (long long)x.k0 * p.k_sr);
  const T* const V = static_cast<const T*>(p.v) + (x.kv * p.v_sh + (long long)x.k0 * p.v_sr);
  const TileFetch<D, 8 / W> fk(wave, ln.lane, 2 * p.k_sr), fv(wave, ln.lane, 2 * p.v_sr);
  DqRows<D, T> rows;
  rows.load(p, x, ln, my);
  float16_t acc[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) acc[c] = zero16();
  const int lim = min(x.nk, my + x.coff + 1);  // keys that this lane's row sees
#pragma unroll 1
  for (int t = 0; t < x.tiles; ++t) {
    const int base = t * L::kRows;
    fk.run(tile_rsrc<2 * D>(K, 2 * p.k_sr, base, x.nk, L::kRows), lds, wave);
    fv.run(tile_rsrc<2 * D>(V, 2 * p.v_sr, base, x.nk, L::kRows), lds + kTileBytes, wave);
    sync_ring<0>();
#pragma unroll 1
    for (int b = 0; b < L::kBlocks; ++b) {
      float16_t s = zero16(), dp = zero16();
      V8 ds[2], ka[D / 16];
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st) s = E::mfma(ln.rows_op(lds, b, st), rows.qf[st], s);
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st)
        dp = E::mfma(ln.rows_op(lds + kTileBytes, b, st), rows.df[st], dp);
      auto sees = [&](int j) { return base + 32 * b + j < lim; };
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], p.scale_log2, -rows.lse2));
        const float y = e * (dp[i] - rows.delta);
        ds[i >> 3][i & 7] = (T)(sees(8 * (i >> 2) + 4 * ln.g + (i & 3)) ? y : 0.0f);
      }
#pragma unroll
      for (int u = 0; u < D / 16; ++u)
        ka[u] = ln.cols_op(lds, u % L::kCols, 2 * b + u / L::kCols);
      add_odd_block<D, T>(lds + 32 * b * L::kRowB, ka, acc, ln.g, sees, true);
#pragma unroll
      for (int u = 0; u < D / 16; ++u)
        acc[u % L::kCols] = E::mfma(ka[u], ds[u / L::kCols], acc[u % L::kCols]);
    }
    sync_ring<0>();
  }
  ln.store(static_cast<T*>(p.dq) + (x.head * p.dq_sh + (long long)x.q0 * p.dq_sr), p.dq_sr, my,
           x.nq, p.scale, acc);
}

// What a row's scores and dout v' start from.
__device__ __forceinline__ float2 row_stats(float lse, float delta, float scale) {
  // (a row that sees nothing: p = 2^-inf)
  return make_float2(lse == ninf() ? (scale > 0.0f ? ninf() : -ninf()) : -lse / scale, -delta);
}

using DqRing = uint8_t[3][2][kTileBytes];

// dq of W x 32 query rows, and with STATS the rows' {-lse / scale, -delta}.
template <int D, int W, bool STATS, class T>
__device__ __forceinline__ void dq_body(const BwdGeom& p, int group, DqRing& ring) {
  using L = BwdLane<D, T>;
  using V8 = typename L::V8;
  using E = Elem<T>;
  constexpr int kSegs = 8 / W, kAhead = 4;
  const void* const geom = (const void*)__builtin_amdgcn_kernarg_segment_ptr();
  DqTask x;
  if (!dq_task<D, W>(p, group, x)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const L ln(threadIdx.x & 63);
  const int qw = x.first + 32 * wave, my = qw + ln.col;
  const T* const K = static_cast<const T*>(p.k) + (x.kv * p.k_sh + (long long)x.k0 * p.k_sr);
  const T* const V = static_cast<const T*>(p.v) + (x.kv * p.v_sh + (long long)x.k0 * p.v_sr);
  const TileFetch<D, kSegs> fk(wave, ln.lane, 2 * p.k_sr), fv(wave, ln.lane, 2 * p.v_sr);
  auto fetch = [&](int t, int s) __attribute__((always_inline)) {
    const int rows = t < x.tiles ? x.nk : 0;
    fk.run(tile_rsrc<2 * D>(K, 2 * p.k_sr, t * L::kRows, rows, L::kRows), ring[s][0], wave);
    fv.run(tile_rsrc<2 * D>(V, 2 * p.v_sr, t * L::kRows, rows, L::kRows), ring[s][1], wave);
  };
  fetch(0, 0);
  fetch(1, 1);
  DqRows<D, T> rows;
  rows.load(p, x, ln, my);
  if (STATS && my < x.nq && ln.g == 0)
    p.stats[(long long)x.head * p.rows + x.q0 + my] = row_stats(rows.lse, rows.delta, p.scale);
  // (what the compiler sees of the loads is then done: no waits in the loop)
  __builtin_amdgcn_s_waitcnt(0);
  const TileOps<D, T> ops(ln);
  const uint32_t lds = (uint32_t)(uintptr_t)&ring[0][0][0];
  float16_t acc[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) acc[c] = zero16();
  const int lim = min(x.nk, my + x.coff + 1);  // keys that this lane's row sees
  int s = 0;
  for (int t = 0; t < x.tiles; ++t) {
    sync_ring<2 * kSegs>();
    fetch(t + 2, s == 0 ? 2 : s - 1);
    const int base = t * L::kRows;
    const uint32_t kt = lds + s * 2 * kTileBytes;
    s = s == 2 ? 0 : s + 1;
    if (base > min(qw + 31, x.nq - 1) + x.coff || qw >= x.nq) continue;  // nothing seen here
    const bool edge = base + L::kRows > min(x.nk, qw + x.coff + 1);
#pragma unroll
    for (int b = 0; b < L::kBlocks; ++b) {
      // 3 kSteps slots of a product each: s, dout v', dq.  A slot's operand is
      // read kAhead slots before; p is taken beside dout v'.
      constexpr int N = L::kSteps;
      float16_t sc = zero16(), dp = zero16();
      V8 op[3 * N], ds[2];
      auto read = [&](auto sl) __attribute__((always_inline)) {
        constexpr int i = decltype(sl)::value, of = i / N, u = i % N;
        if constexpr (of < 2)
          op[i] = ops.rows(kt, of * kTileBytes, b, u);
        else
          op[i] = ops.cols(kt, 0, u % L::kCols, 2 * b + u / L::kCols);
      };
      auto minus = [&](int e) __attribute__((always_inline)) {  // element e of ds
        ds[e >> 3][e & 7] = (T)(sc[e] * (dp[e] - rows.delta));
      };
      static_for(std::make_integer_sequence<int, kAhead>{}, read);
      static_for(std::make_integer_sequence<int, 3 * N>{}, [&](auto sl) __attribute__((always_inline)) {
        constexpr int i = decltype(sl)::value, of = i / N, u = i % N, kEach = 16 / N;
        constexpr int c = u % L::kCols, tt = u / L::kCols;
        if constexpr (of == 0)
          sc = E::mfma(op[i], rows.qf[u], sc);
        else if constexpr (of == 1)
          dp = E::mfma(op[i], rows.df[u], dp);
        else
          acc[c] = E::mfma(op[i], ds[tt], acc[c]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (i + kAhead < 3 * N) read(Ic<i + kAhead>{});
        if constexpr (i == N - 1) {
          if (edge) {
            const float hidden = p.scale > 0.0f ? ninf() : -ninf();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (base + 32 * b + 8 * (e >> 2) + 4 * ln.g + (e & 3) >= lim) sc[e] = hidden;
          }
        }
        if constexpr (of == 1) {
#pragma unroll
          for (int e = u * kEach; e < (u + 1) * kEach; ++e)
            sc[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], p.scale_log2, -rows.lse2));
        }
        // (the first 8 rows' before the products that take them, the others among those)
        if constexpr (i == 2 * N - 1) {
#pragma unroll
          for (int e = 0; e < 8; ++e) minus(e);
        } else if constexpr (of == 2 && tt == 0) {
          constexpr int kSome = 8 / L::kCols;
#pragma unroll
          for (int e = 8 + u * kSome; e < 8 + (u + 1) * kSome; ++e) minus(e);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    }
  }
  // A block with a row whose sum is not finite is walked again.
  __builtin_amdgcn_s_waitcnt(0);
  int* const redo = reinterpret_cast<int*>(ring);
  __syncthreads();
  if (threadIdx.x == 0) *redo = 0;
  __syncthreads();
  if (my < x.nq && any_odd(acc)) *redo = 1;
  __syncthreads();
  const bool again = *redo != 0;
  __syncthreads();
  if (again)
    dq_checked<D, W, T>(geom, group, &ring[0][0][0]);
  else
    ln.store(static_cast<T*>(p.dq) + (x.head * p.dq_sh + (long long)x.q0 * p.dq_sr), p.dq_sr, my,
             x.nq, p.scale, acc);
}

template <int D, int W, class T>
__global__ void __launch_bounds__(64 * W, 2) packed_dq_kernel(const BwdGeom p) {
  __shared__ __attribute__((aligned(16))) DqRing ring;
  dq_body<D, W, true, T>(p, blockIdx.x, ring);
}

// A work-group's key block, and its share of the queries that see it.
struct DkvTask {
  int kv, part, q0, nq, k0, nk, coff, first;
  int tbeg, per, steps, h0, t0;  // a head's first tile and tiles; steps from head h0, tile t0 on
};

constexpr int kDkvWaves = 4;

template <int R>  // query rows of a tile
__device__ __forceinline__ bool dkv_task(const BwdGeom& p, int group, DkvTask& x) {
  int r, unit;
  PackedAt at;
  packed_unit(group, p.kv_heads * p.parts, p.xcds, r, unit);
  constexpr int kBlock = 32 * kDkvWaves;
  if (!packed_block<kBlock>(p.key_starts, p.key_rows, p.starts, p.rows, p.sequences, r, p.causal,
                            at))
    return false;
  x.kv = unit / p.parts;
  x.part = unit - x.kv * p.parts;
  x.q0 = at.other;
  x.nq = at.others;
  x.k0 = at.begin;
  x.nk = at.count;
  // (the last index is the heaviest under a causal mask: the first keys)
  x.first = ((x.nk + kBlock - 1) / kBlock - 1 - at.j) * kBlock;
  x.coff = p.causal ? x.nk - x.nq : x.nk;
  x.tbeg = max(x.first - x.coff, 0) / R;
  x.per = max((x.nq + R - 1) / R - x.tbeg, 0);
  const int all = x.per * p.group;
  const int s0 = (int)((long long)all * x.part / p.parts);
  x.steps = (int)((long long)all * (x.part + 1) / p.parts) - s0;
  x.h0 = x.per > 0 ? s0 / x.per : 0;
  x.t0 = x.tbeg + (s0 - x.h0 * x.per);
  return true;
}

// The tiles of a walk, one after the other: the queries of a head, then those
// of the next.  A wave moves its share of q's and dout's rows and all of the
// statistics (every wave to the same place: its own wait then covers them), or
// with OWN none of those.
template <int D, int R, bool OWN, class T>
struct DkvFetch {
  static constexpr int kTileB = R * 2 * D, kSegs = kTileB / 1024 / kDkvWaves;
  static constexpr int kStats = OWN ? 0 : R / 32;
  static constexpr int kDma = 2 * kSegs + kStats;  // instructions of a wave
  const TileFetch<D, kSegs> fq, fd;
  int step, head, tile, wave, lane;
  i32x4_t rq, rd, rst;

  __device__ __forceinline__ DkvFetch(const BwdGeom& p, const DkvTask& x, int wave_, int lane_)
      : fq(wave_, lane_, 2 * p.q_sr), fd(wave_, lane_, 2 * p.do_sr) {
    wave = wave_;
    lane = lane_;
    step = 0;
    head = x.kv * p.group + x.h0;
    tile = x.t0;
  }
  // On to the next tile (past the last: zeros).
  __device__ __forceinline__ void next(const BwdGeom& p, const DkvTask& x) {
    const int rows = step < x.steps ? x.nq : 0;
    const long long h = min(head, p.heads - 1);
    rq = tile_rsrc<2 * D>(static_cast<const T*>(p.q) + (h * p.q_sh + (long long)x.q0 * p.q_sr),
                          2 * p.q_sr, tile * R, rows, R);
    rd = tile_rsrc<2 * D>(
        static_cast<const T*>(p.dout) + (h * p.do_sh + (long long)x.q0 * p.do_sr), 2 * p.do_sr,
        tile * R, rows, R);
    if constexpr (!OWN) rst = tile_rsrc<8>(p.stats + (h * p.rows + x.q0), 8, tile * R, rows, R);
    ++step;
    if (++tile == x.tbeg + x.per) {
      tile = x.tbeg;
      ++head;
    }
  }
  // Its i-th instruction.
  __device__ __forceinline__ void dma(const uint8_t* slot, const uint8_t* stat, int i) const {
    if (i < kSegs)
      fq.seg(rq, slot, wave, i);
    else if (i < 2 * kSegs)
      fd.seg(rd, slot + kTileB, wave, i - kSegs);
    else if constexpr (!OWN) {
      const int at = 64 * (i - 2 * kSegs) + lane;  // {starts of s, of dout v'} [R]
      load_lds4(rst, 8 * (at % R) + 4 * (at / R), stat + 256 * (i - 2 * kSegs));
    }
  }
  __device__ __forceinline__ void run(const BwdGeom& p, const DkvTask& x, const uint8_t* slot,
                                      const uint8_t* stat) {
    next(p, x);
#pragma unroll
    for (int i = 0; i < kDma; ++i) dma(slot, stat, i);
  }
};

// Tiles whose statistics a work-group takes at a time, where it does so itself.
constexpr int kOwnSteps = 16;

// The statistics {starts of s, of dout v'} [R] of the next tiles of a walk, at
// most kOwnSteps from `step` on, by all threads: D / 16 a row.  (Rows past the
// last: 0, as loads give.)
template <int D, int R, class T>
__device__ __forceinline__ void own_stats(const BwdGeom& p, const DkvTask& x, int step, int& head,
                                          int& t, float* stat) {
  using V8 = typename Elem<T>::v8;
  constexpr int kThreads = D / 16;
  static_assert(R * kThreads == 256);
  const int row = (int)threadIdx.x / kThreads, c = 16 * ((int)threadIdx.x % kThreads);
  const int count = min(x.steps - step, kOwnSteps);
  for (int i = 0; i < count; ++i) {
    const int r = t * R + row;
    float2 s = make_float2(0.0f, 0.0f);
    float sum = 0.0f, lse = 0.0f;
    if (r < x.nq) {
      const T* const d = static_cast<const T*>(p.dout) + (head * p.do_sh +
                                                          (long long)(x.q0 + r) * p.do_sr + c);
      const T* const o =
          static_cast<const T*>(p.o) + (head * p.o_sh + (long long)(x.q0 + r) * p.o_sr + c);
      lse = p.lse[(long long)head * p.rows + x.q0 + r];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const V8 a = *reinterpret_cast<const V8*>(d + 8 * h);
        const V8 b = *reinterpret_cast<const V8*>(o + 8 * h);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = __builtin_fmaf((float)a[e], (float)b[e], sum);
      }
    }
#pragma unroll
    for (int m = 1; m < kThreads; m *= 2) sum += __shfl_xor(sum, m);
    if (r < x.nq) s = row_stats(lse, sum, p.scale);
    if (c == 0) {
      stat[2 * R * i + row] = s.x;
      stat[2 * R * i + R + row] = s.y;
    }
    if (++t == x.tbeg + x.per) {
      t = x.tbeg;
      ++head;
    }
  }
  __syncthreads();
}

template <int D, class T>
__device__ __forceinline__ void dkv_store(const BwdGeom& p, const DkvTask& x,
                                          const BwdLane<D, T>& ln, int my,
                                          const float16_t (&dk)[D / 32],
                                          const float16_t (&dv)[D / 32]) {
  if (p.parts > 1) {
    float* const to =
        p.part + (((long long)x.part * p.kv_heads + x.kv) * p.key_rows + x.k0) * (2 * D);
    ln.store_part(to, my, x.nk, dk);
    ln.store_part(to + D, my, x.nk, dv);
  } else {
    ln.store(static_cast<T*>(p.dk) + (x.kv * p.dk_sh + (long long)x.k0 * p.dk_sr), p.dk_sr, my,
             x.nk, p.scale, dk);
    ln.store(static_cast<T*>(p.dv) + (x.kv * p.dv_sh + (long long)x.k0 * p.dv_sr), p.dv_sr, my,
             x.nk, 1.0f, dv);
  }
}

// The dk and dv kernel's block walked again, with NaN and infinities of queries
// that do not see a key kept from it.
template <int D, int R, bool OWN, class T>
__device__ __attribute__((noinline)) void dkv_checked(const void* geom, int group, uint8_t* lds,
                                                      uint8_t* stat) {
  using L = BwdLane<D, T>;
  using V8 = typename L::V8;
  using E = Elem<T>;
  lds = uniform(lds);
  stat = uniform(stat);
  group = __builtin_amdgcn_readfirstlane(group);
  BwdGeom p;
  __builtin_memcpy(&p, geom, sizeof p);
  DkvTask x;
  if (!dkv_task<R>(p, group, x)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const L ln(threadIdx.x & 63);
  const int my = x.first + 32 * wave + ln.col;
  DkvFetch<D, R, OWN, T> tiles(p, x, wave, ln.lane);
  V8 kf[L::kSteps], vf[L::kSteps];
  ln.own_rows(static_cast<const T*>(p.k) + (x.kv * p.k_sh + (long long)x.k0 * p.k_sr), p.k_sr, my,
              x.nk, kf);
  ln.own_rows(static_cast<const T*>(p.v) + (x.kv * p.v_sh + (long long)x.k0 * p.v_sr), p.v_sr, my,
              x.nk, vf);
  float16_t dk[L::kCols], dv[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) dk[c] = dv[c] = zero16();
  const int lo = my - x.coff;  // queries from lo on see this lane's key
  float* const st = reinterpret_cast<float*>(stat);
  const uint8_t *const qt = lds, *const dt = lds + DkvFetch<D, R, OWN, T>::kTileB;
  int t = x.t0, own_head = x.kv * p.group + x.h0, own_t = x.t0;
#pragma unroll 1
  for (int step = 0; step < x.steps; ++step) {
    tiles.run(p, x, lds, stat);
    if (OWN && step % kOwnSteps == 0) own_stats<D, R, T>(p, x, step, own_head, own_t, st);
    sync_ring<0>();
#pragma unroll 1
    for (int b = 0; b < R / 32; ++b) {
      const int base = t * R + 32 * b;
      float16_t sc, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = (OWN ? 2 * R * (step % kOwnSteps) : 0) + 32 * b + 8 * (i >> 2) + 4 * ln.g + (i & 3);
        sc[i] = st[at];
        dp[i] = st[R + at];
      }
#pragma unroll
      for (int u = 0; u < L::kSteps; ++u) sc = E::mfma(ln.rows_op(qt, b, u), kf[u], sc);
#pragma unroll
      for (int u = 0; u < L::kSteps; ++u) dp = E::mfma(ln.rows_op(dt, b, u), vf[u], dp);
      V8 pp[2], ds[2];
      auto sees = [&](int j) { return base + j >= lo && base + j < x.nq; };
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const bool seen = sees(8 * (i >> 2) + 4 * ln.g + (i & 3));
        const float e = __builtin_amdgcn_exp2f(sc[i] * p.scale_log2), y = e * dp[i];
        pp[i >> 3][i & 7] = (T)(seen ? e : 0.0f);
        ds[i >> 3][i & 7] = (T)(seen ? y : 0.0f);
      }
      auto add = [&](const uint8_t* tile, float16_t (&acc)[L::kCols], const V8 (&w)[2],
                     bool as_nan) __attribute__((always_inline)) {
        V8 a[D / 16];
#pragma unroll
        for (int u = 0; u < D / 16; ++u)
          a[u] = ln.cols_op(tile, u % L::kCols, 2 * b + u / L::kCols);
        add_odd_block<D, T>(tile + 32 * b * L::kRowB, a, acc, ln.g, sees, as_nan);
#pragma unroll
        for (int u = 0; u < D / 16; ++u)
          acc[u % L::kCols] = E::mfma(a[u], w[u / L::kCols], acc[u % L::kCols]);
      };
      add(dt, dv, pp, false);
      add(qt, dk, ds, true);
    }
    if (++t == x.tbeg + x.per) t = x.tbeg;
    sync_ring<0>();
  }
  dkv_store<D, T>(p, x, ln, my, dk, dv);
}

// dk and dv of 128 keys (4 waves of 32) over part `part` of the queries that
// see them, of all heads of the group one after the other, in tiles of R query
// rows.  K's operands stay in registers and V's in LDS, which leaves registers
// for two waves a SIMD: the products of one run among the exponentials of the
// other.  s and dout v' start from {-lse / scale, -delta} as accumulators, so p =
// 2^(s c) and ds = p dp' need no further subtraction, and where a block has
// hidden pairs those start from -inf.  With OWN the work-group takes the
// statistics of its few tiles itself, into LDS.
template <int D, int R, bool OWN>
struct DkvLds {
  static constexpr int kRing = D == 128 ? 2 : 3;
  uint8_t ring[kRing][2][R * 2 * D];
  uint8_t vblk[128 * 2 * D];
  uint8_t stat[OWN ? kOwnSteps : kRing][8 * R];
};

template <int D, int R, bool OWN, class T>
__device__ __forceinline__ void dkv_body(const BwdGeom& p, int group, DkvLds<D, R, OWN>& lds) {
  using L = BwdLane<D, T>;
  using V8 = typename L::V8;
  using E = Elem<T>;
  using F = DkvFetch<D, R, OWN, T>;
  constexpr int kTileB = F::kTileB, kRing = DkvLds<D, R, OWN>::kRing;
  auto& ring = lds.ring;
  auto& vblk = lds.vblk;
  auto& stat = lds.stat;
  constexpr int kVSegs = 128 * 2 * D / 1024 / 4, kAhead = 3;
  typedef const float4_t __attribute__((address_space(3))) * LdsF4;
  const void* const geom = (const void*)__builtin_amdgcn_kernarg_segment_ptr();
  DkvTask x;
  if (!dkv_task<R>(p, group, x)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const L ln(threadIdx.x & 63);
  const int kw = x.first + 32 * wave, my = kw + ln.col;
  float16_t dk[L::kCols], dv[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) dk[c] = dv[c] = zero16();
  bool again = false;
  if (x.steps > 0) {
    {
      const TileFetch<D, kVSegs> f(wave, ln.lane, 2 * p.v_sr);
      f.run(tile_rsrc<2 * D>(static_cast<const T*>(p.v) + (x.kv * p.v_sh + (long long)x.k0 * p.v_sr),
                             2 * p.v_sr, x.first, x.nk, 128),
            vblk, wave);
    }
    F tiles(p, x, wave, ln.lane);
#pragma unroll
    for (int i = 0; i < kRing - 1; ++i) tiles.run(p, x, ring[i][0], stat[i]);
    V8 kf[L::kSteps];
    ln.own_rows(static_cast<const T*>(p.k) + (x.kv * p.k_sh + (long long)x.k0 * p.k_sr), p.k_sr,
                my, x.nk, kf);
    __builtin_amdgcn_s_waitcnt(0);
    const TileOps<D, T> ops(ln);
    const uint32_t lds_ring = (uint32_t)(uintptr_t)&ring[0][0][0];
    const uint32_t lds_v = (uint32_t)(uintptr_t)&vblk[0] + wave * 32 * L::kRowB;
    const uint32_t lds_stat = (uint32_t)(uintptr_t)&stat[0][0] + 16 * ln.g;
    const int lo = my - x.coff;  // queries from lo on see this lane's key
    int t = x.t0, s = 0, own_head = x.kv * p.group + x.h0, own_t = x.t0;
#pragma unroll 1
    for (int step = 0; step < x.steps; ++step) {
      sync_ring<(kRing - 2) * F::kDma>();
      if (OWN && step % kOwnSteps == 0)
        own_stats<D, R, T>(p, x, step, own_head, own_t, reinterpret_cast<float*>(&stat[0][0]));
      {
        const int to = s == 0 ? kRing - 1 : s - 1;
        tiles.run(p, x, ring[to][0], stat[to]);
      }
      const uint32_t tile = lds_ring + s * 2 * kTileB, st = lds_stat + (OWN ? step % kOwnSteps : s) * 8 * R;
      s = s == kRing - 1 ? 0 : s + 1;
      const int first = t * R;
      if (++t == x.tbeg + x.per) t = x.tbeg;
      // (queries of the tile that see one of this wave's keys)
      if (min(first + R, x.nq) - 1 + x.coff < kw || kw >= x.nk) continue;
#pragma unroll
      for (int b = 0; b < R / 32; ++b) {
        const int base = first + 32 * b;
        float16_t S, X;
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
          const float4_t y = *(LdsF4)(uintptr_t)(st + 4 * (32 * b + 8 * g4));
          const float4_t z = *(LdsF4)(uintptr_t)(st + 4 * (R + 32 * b + 8 * g4));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            S[4 * g4 + e] = y[e];
            X[4 * g4 + e] = z[e];
          }
        }
        if (base + 32 > x.nq || base + x.coff < kw + 31) {
          const float hidden = p.scale > 0.0f ? ninf() : -ninf();
          const int from = lo - base - 4 * ln.g, end = x.nq - base - 4 * ln.g;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int at = 8 * (e >> 2) + (e & 3);
            if (at < from || at >= end) S[e] = hidden;
          }
        }
        // 4 kSteps slots of a product each: s, dout v', dv, dk.  A slot's operand
        // is read kAhead slots before; p is taken beside dout v', ds beside dv.
        constexpr int N = L::kSteps;
        V8 op[4 * N], vo[N], P[2], Q[2];
        auto read = [&](auto sl) __attribute__((always_inline)) {
          constexpr int i = decltype(sl)::value, of = i / N, u = i % N;
          if constexpr (of < 2) {
            op[i] = ops.rows(tile, of * kTileB, b, u);
            if constexpr (of == 1) vo[u] = ops.rows(lds_v, 0, 0, u);
          } else {
            op[i] = ops.cols(tile, (3 - of) * kTileB, u % L::kCols, 2 * b + u / L::kCols);
          }
        };
        static_for(std::make_integer_sequence<int, kAhead>{}, read);
        static_for(std::make_integer_sequence<int, 4 * N>{}, [&](auto sl) __attribute__((always_inline)) {
          constexpr int i = decltype(sl)::value, of = i / N, u = i % N;
          constexpr int c = u % L::kCols, tt = u / L::kCols, kEach = 16 / N;
          if constexpr (of == 0)
            S = E::mfma(op[i], kf[u], S);
          else if constexpr (of == 1)
            X = E::mfma(op[i], vo[u], X);
          else if constexpr (of == 2)
            dv[c] = E::mfma(op[i], P[tt], dv[c]);
          else
            dk[c] = E::mfma(op[i], Q[tt], dk[c]);
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (i + kAhead < 4 * N) read(Ic<i + kAhead>{});
#pragma unroll
          for (int e = u * kEach; e < (u + 1) * kEach; ++e) {
            if constexpr (of == 1) {
              S[e] = __builtin_amdgcn_exp2f(S[e] * p.scale_log2);
              P[e >> 3][e & 7] = (T)S[e];
            } else if constexpr (of == 2) {
              Q[e >> 3][e & 7] = (T)(S[e] * X[e]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        });
      }
    }
    // A block with a key whose sums are not finite is walked again.
    __builtin_amdgcn_s_waitcnt(0);
    int* const redo = reinterpret_cast<int*>(vblk);
    __syncthreads();
    if (threadIdx.x == 0) *redo = 0;
    __syncthreads();
    if (my < x.nk && (any_odd(dk) || any_odd(dv))) *redo = 1;
    __syncthreads();
    again = *redo != 0;
    __syncthreads();
  }
  if (again)
    dkv_checked<D, R, OWN, T>(geom, group, &ring[0][0][0], &stat[0][0]);
  else
    dkv_store<D, T>(p, x, ln, my, dk, dv);
}

template <int D, int R, class T>
__global__ void __launch_bounds__(256, 2) packed_dkv_kernel(const BwdGeom p) {
  __shared__ __attribute__((aligned(16))) DkvLds<D, R, false> lds;
  dkv_body<D, R, false, T>(p, blockIdx.x, lds);
}

// Little work: the work-groups of both kernels in one launch, `first` of them
// dq's, none of which waits for another.
template <int D, int R, class T>
__global__ void __launch_bounds__(256, 2) packed_both_kernel(const BwdGeom p, int first) {
  __shared__ __attribute__((aligned(16))) union {
    DqRing ring;
    DkvLds<D, R, true> lds;
  } u;
  if ((int)blockIdx.x < first)
    dq_body<D, 4, false, T>(p, blockIdx.x, u.ring);
  else
    dkv_body<D, R, true, T>(p, blockIdx.x - first, u.lds);
}

// Sums the parts: a thread 4 columns of a key's dk and dv.
template <int D, class T>
__global__ void __launch_bounds__(256) packed_join_kernel(const BwdGeom p) {
  constexpr int kThreads = D / 4;
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  const int c = 4 * (int)(x % kThreads);
  const long long row = x / kThreads;
  const int kv = (int)(row / p.key_rows), t = (int)(row - (long long)kv * p.key_rows);
  if (kv >= p.kv_heads) return;
  // rows of no sequence have no parts and are left as they were
  int lo = 0, hi = p.sequences;  // the last sequence that starts at or before t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.key_starts[mid + 1] <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  if (lo >= p.sequences || p.key_starts[lo] > t) return;
  const long long step = (long long)p.kv_heads * p.key_rows * (2 * D);
  const float* from = p.part + row * (2 * D) + c;
  float4 dk = {0, 0, 0, 0}, dv = {0, 0, 0, 0};
  for (int i = 0; i < p.parts; ++i, from += step) {
    const float4 a = *reinterpret_cast<const float4*>(from);
    const float4 b = *reinterpret_cast<const float4*>(from + D);
    dk.x += a.x, dk.y += a.y, dk.z += a.z, dk.w += a.w;
    dv.x += b.x, dv.y += b.y, dv.z += b.z, dv.w += b.w;
  }
  using V4 = typename Elem<T>::v4;
  const V4 k4 = {(T)(dk.x * p.scale), (T)(dk.y * p.scale), (T)(dk.z * p.scale),
                 (T)(dk.w * p.scale)};
  const V4 v4 = {(T)dv.x, (T)dv.y, (T)dv.z, (T)dv.w};
  *reinterpret_cast<V4*>(static_cast<T*>(p.dk) + (kv * p.dk_sh + (long long)t * p.dk_sr + c)) = k4;
  *reinterpret_cast<V4*>(static_cast<T*>(p.dv) + (kv * p.dv_sh + (long long)t * p.dv_sr + c)) = v4;
}

template <int D, class T>
hipError_t launch_bwd_dim(const BwdGeom& g, hipStream_t st) {
  constexpr int W = 4, R = D == 128 ? 32 : 64;
  const int64_t a = packed_groups(g.rows, g.sequences, 32 * W, g.heads);
  const int64_t b = packed_groups(g.key_rows, g.sequences, 32 * W, g.kv_heads * g.parts);
  // One launch up to two rounds of two work-groups a CU, one and a half without
  // a causal mask (us; two launches, one): 4 sequences of 33-257, H8/2 D 64 25.8,
  // 17.5; 4 of 300-700, H8 36.2, 26.2; one of 2048, H4 58.8, 42.7; of 1024, H32/8
  // D 128 81.9, 72.2; of 8192, H1 257, 218; above: 8 of 100-300, H32/8 60.2, 66.8;
  // 16 of 64-2000 686, 904; not causal, 4096, H8 D 64 159, 169.
  if (a + b <= (g.causal ? 4 : 3) * device_cus()) {
    hipLaunchKernelGGL((packed_both_kernel<D, R, T>), dim3((unsigned)(a + b)), dim3(64 * W), 0, st,
                       g, (int)a);
  } else {
    hipLaunchKernelGGL((packed_dq_kernel<D, W, T>), dim3((unsigned)a), dim3(64 * W), 0, st, g);
    hipLaunchKernelGGL((packed_dkv_kernel<D, R, T>), dim3((unsigned)b), dim3(64 * W), 0, st, g);
  }
  if (g.parts > 1)
    hipLaunchKernelGGL(
        (packed_join_kernel<D, T>),
        dim3((unsigned)(((long long)g.kv_heads * g.key_rows * (D / 4) + 255) / 256)), dim3(256), 0,
        st, g);
  return hipGetLastError();
}

template <class T>
hipError_t launch_bwd_type(const fl_packed_params& p, const fl_packed_grads& d, void* ws,
                           hipStream_t st) {
  BwdGeom g = {};
  g.q = p.q;
  g.k = p.k;
  g.v = p.v;
  g.o = p.o;
  g.dout = d.dout;
  g.dq = d.dq;
  g.dk = d.dk;
  g.dv = d.dv;
  g.lse = p.lse;
  g.stats = static_cast<float2*>(ws);
  g.q_sh = p.q_stride[0];
  g.k_sh = p.k_stride[0];
  g.v_sh = p.v_stride[0];
  g.o_sh = p.o_stride[0];
  g.do_sh = d.dout_stride[0];
  g.dq_sh = d.dq_stride[0];
  g.dk_sh = d.dk_stride[0];
  g.dv_sh = d.dv_stride[0];
  g.q_sr = (int)p.q_stride[1];
  g.k_sr = (int)p.k_stride[1];
  g.v_sr = (int)p.v_stride[1];
  g.o_sr = (int)p.o_stride[1];
  g.do_sr = (int)d.dout_stride[1];
  g.dq_sr = (int)d.dq_stride[1];
  g.dk_sr = (int)d.dk_stride[1];
  g.dv_sr = (int)d.dv_stride[1];
  g.starts = p.starts;
  g.key_starts = p.key_starts ? p.key_starts : p.starts;
  g.sequences = (int)p.sequences;
  g.rows = (int)p.rows;
  g.key_rows = (int)p.key_rows;
  g.heads = (int)p.heads;
  g.kv_heads = (int)p.kv_heads;
  g.group = (int)(p.heads / p.kv_heads);
  g.parts = packed_bwd_parts(p);
  g.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + packed_stat_bytes(p));
  g.causal = p.causal != 0;
  g.xcds = device_xcds();
  const double s = p.sm_scale == 0.0 ? 1.0 / __builtin_sqrt((double)p.head_dim) : p.sm_scale;
  g.scale = (float)s;
  g.scale_log2 = (float)(s * 1.4426950408889634);
  return p.head_dim == 128 ? launch_bwd_dim<128, T>(g, st) : launch_bwd_dim<64, T>(g, st);
}

}  // namespace

}  // namespace fl
