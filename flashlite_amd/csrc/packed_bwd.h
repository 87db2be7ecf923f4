// Gradients of attention over packed sequences (fl_attn_packed_bwd), one
// source file per element type (packed_bwd_f16.hip, packed_bwd_bf16.hip).
//
// With p = exp(s - lse), s = scale q.k, delta = dout . out a row and
// ds = p (dout v' - delta):
//   dv = p' dout    dk = scale ds' q    dq = scale ds k
// p is taken again from q, k and lse, so nothing of the size of the scores is
// kept.  Two kernels, each of which owns what it sums, so no atomics and the
// same bits every time: one walks a query block's keys (3 products a pair: s,
// dout v', dq) and leaves lse and delta in base 2 for the other, which walks a
// key block's queries over all heads of its group (4 products: s, dout v', dv,
// dk).  14 D flops a pair of a row and a key, 7 products where one kernel with
// atomics would do with 5.
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
  float2* stats;          // [heads][rows]: lse in base 2, delta
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
  left = min(left, most);
  asm("" : "+s"(left));
  return max(left, 0);
}

// DMA of tiles: wave w moves kSegs of a tile's 8 segments of 1 KiB, each lane
// 16 bytes.
template <int D, int kSegs>
struct TileFetch {
  int lane[kSegs];
  __device__ __forceinline__ TileFetch(int wave, int l, int row_bytes) {
    constexpr int kChunks = D / 8, kSegRows = 64 / kChunks;
#pragma unroll
    for (int i = 0; i < kSegs; ++i) {
      const int row = kSegRows * (wave * kSegs + i) + l / kChunks;
      lane[i] = row * row_bytes + 16 * ((l % kChunks) ^ both_swz<D>(row));
    }
  }
  // The rows row0 .. of x (those from `rows` on as zeros).
  template <class T>
  __device__ __forceinline__ void run(const T* x, int row_bytes, int row0, int rows,
                                      const uint8_t* slot, int wave) const {
    constexpr int kRows = kTileBytes / (2 * D);
    const i32x4_t rs =
        rows_rsrc<2 * D>(reinterpret_cast<const uint8_t*>(x) + (long long)row0 * row_bytes,
                         tile_rows(rows - row0, kRows), row_bytes);
#pragma unroll
    for (int i = 0; i < kSegs; ++i) load_lds16(rs, lane[i], slot + 1024 * (wave * kSegs + i));
  }
};

// 4 bytes a lane into LDS at slot + 4 * lane (as load_lds16).
__device__ __forceinline__ void load_lds4(const i32x4_t& rs, int voff, const uint8_t* slot) {
  const uint32_t lds_base = (uint32_t)(uintptr_t)slot;
  asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds"
               : : "v"(voff), "s"(rs), "{m0}"(lds_base));
}

constexpr int kBwdSlots = 3;

// dq of W x 32 query rows, and the rows' lse and delta.
template <int D, int W, class T>
__global__ void __launch_bounds__(64 * W, 2) packed_dq_kernel(const BwdGeom p) {
  using L = BwdLane<D, T>;
  using V8 = typename L::V8;
  using E = Elem<T>;
  constexpr int kSegs = 8 / W;
  __shared__ __attribute__((aligned(16))) uint8_t ring[kBwdSlots][2][kTileBytes];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const L ln(threadIdx.x & 63);
  int r, head, seq, qb;
  packed_unit(p.heads, p.xcds, r, head);
  if (!packed_block<32 * W>(p.starts, p.sequences, p.rows, r, seq, qb)) return;
  seq = __builtin_amdgcn_readfirstlane(seq);
  int q0, nq, k0, nk;
  sequence_rows(p.starts, seq, p.rows, q0, nq);
  sequence_rows(p.key_starts, seq, p.key_rows, k0, nk);
  const int coff = p.causal ? nk - nq : nk;  // query i sees keys up to i + coff
  const int kv = head / p.group;
  const T* const K = static_cast<const T*>(p.k) + (kv * p.k_sh + (long long)k0 * p.k_sr);
  const T* const V = static_cast<const T*>(p.v) + (kv * p.v_sh + (long long)k0 * p.v_sr);
  const int first = qb * 32 * W, qw = first + 32 * wave, my = qw + ln.col;
  int tiles = (min(nk, min(first + 32 * W, nq) + coff) + L::kRows - 1) / L::kRows;
  tiles = max(tiles, 0);

  const TileFetch<D, kSegs> fk(wave, ln.lane, 2 * p.k_sr), fv(wave, ln.lane, 2 * p.v_sr);
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const int s = t % kBwdSlots, rows = t < tiles ? nk : 0;
    fk.run(K, 2 * p.k_sr, t * L::kRows, rows, ring[s][0], wave);
    fv.run(V, 2 * p.v_sr, t * L::kRows, rows, ring[s][1], wave);
  };
  fetch(0);
  fetch(1);
  V8 qf[L::kSteps], df[L::kSteps];
  float lse2, delta;
  {
    V8 of[L::kSteps];
    ln.own_rows(static_cast<const T*>(p.q) + (head * p.q_sh + (long long)q0 * p.q_sr), p.q_sr, my,
                nq, qf);
    ln.own_rows(static_cast<const T*>(p.dout) + (head * p.do_sh + (long long)q0 * p.do_sr),
                p.do_sr, my, nq, df);
    ln.own_rows(static_cast<const T*>(p.o) + (head * p.o_sh + (long long)q0 * p.o_sr), p.o_sr, my,
                nq, of);
    float sum = 0.0f;
#pragma unroll
    for (int st = 0; st < L::kSteps; ++st)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = __builtin_fmaf((float)df[st][e], (float)of[st][e], sum);
    delta = pair_sum(sum);
    const long long at = (long long)head * p.rows + q0 + my;
    const float lse = my < nq ? p.lse[at] : 0.0f;
    // (a row that sees nothing: p = 2^-inf)
    lse2 = lse == ninf() ? -ninf() : lse * 1.44269504088896341f;
    if (my < nq && ln.g == 0) p.stats[at] = make_float2(lse2, delta);
  }
  // (what the compiler sees of the loads is then done: no waits in the loop)
  __builtin_amdgcn_s_waitcnt(0);
  float16_t acc[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) acc[c] = zero16();
  const int lim = min(nk, my + coff + 1);  // keys that this lane's row sees
  for (int t = 0; t < tiles; ++t) {
    sync_ring<2 * kSegs>();
    fetch(t + 2);
    const int base = t * L::kRows;
    if (base > min(qw + 31, nq - 1) + coff || qw >= nq) continue;  // nothing seen by this wave
    const uint8_t* const kt = ring[t % kBwdSlots][0];
    const uint8_t* const vt = ring[t % kBwdSlots][1];
    const bool edge = base + L::kRows > min(nk, qw + coff + 1);
    V8 ds[L::kBlocks][2];
#pragma unroll
    for (int b = 0; b < L::kBlocks; ++b) {
      float16_t s = zero16(), dp = zero16();
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st) s = E::mfma(ln.rows_op(kt, b, st), qf[st], s);
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st) dp = E::mfma(ln.rows_op(vt, b, st), df[st], dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], p.scale_log2, -lse2));
        float x = e * (dp[i] - delta);
        if (edge && base + 32 * b + 8 * (i >> 2) + 4 * ln.g + (i & 3) >= lim) x = 0.0f;
        ds[b][i >> 3][i & 7] = (T)x;
      }
    }
    V8 ka[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) ka[u] = ln.cols_op(kt, u % L::kCols, u / L::kCols);
    if (edge)
      add_odd<D, T>(
          kt, ka, acc, ln.g, [&](int j) { return base + j < lim; }, true,
          [](int row) { return both_swz<D>(row); });
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int tt = u / L::kCols;
      acc[u % L::kCols] = E::mfma(ka[u], ds[tt >> 1][tt & 1], acc[u % L::kCols]);
    }
  }
  __builtin_amdgcn_s_waitcnt(0);
  ln.store(static_cast<T*>(p.dq) + (head * p.dq_sh + (long long)q0 * p.dq_sr), p.dq_sr, my, nq,
           p.scale, acc);
}

// dk and dv of W x 32 keys over part `part` of the queries that see them, of
// all heads of the group one after the other.
template <int D, int W, class T, int OCC>
__global__ void __launch_bounds__(64 * W, OCC) packed_dkv_kernel(const BwdGeom p) {
  using L = BwdLane<D, T>;
  using V8 = typename L::V8;
  using E = Elem<T>;
  constexpr int kSegs = 8 / W;
  constexpr int kStatB = 2 * 4 * L::kRows, kStatLoads = L::kRows / 32;
  constexpr int kLoads = 2 * kSegs + kStatLoads;
  __shared__ __attribute__((aligned(16))) uint8_t ring[kBwdSlots][2][kTileBytes];
  __shared__ __attribute__((aligned(16))) uint8_t stat[kBwdSlots][kStatB];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const L ln(threadIdx.x & 63);
  int r, unit, seq, kb;
  packed_unit(p.kv_heads * p.parts, p.xcds, r, unit);
  if (!packed_block<32 * W>(p.key_starts, p.sequences, p.key_rows, r, seq, kb)) return;
  seq = __builtin_amdgcn_readfirstlane(seq);
  const int kv = unit / p.parts, part = unit - kv * p.parts;
  int q0, nq, k0, nk;
  sequence_rows(p.starts, seq, p.rows, q0, nq);
  sequence_rows(p.key_starts, seq, p.key_rows, k0, nk);
  // (the last index is the heaviest under a causal mask: the first keys)
  kb = (nk + 32 * W - 1) / (32 * W) - 1 - kb;
  const int coff = p.causal ? nk - nq : nk;
  const int first = kb * 32 * W, kw = first + 32 * wave, my = kw + ln.col;
  const int tbeg = max(first - coff, 0) / L::kRows;
  const int per = max((nq + L::kRows - 1) / L::kRows - tbeg, 0);  // tiles a head
  const int all = per * p.group;
  const int s0 = (int)((long long)all * part / p.parts);
  const int s1 = (int)((long long)all * (part + 1) / p.parts);
  const int h0 = per > 0 ? s0 / per : 0;

  const TileFetch<D, kSegs> fq(wave, ln.lane, 2 * p.q_sr), fd(wave, ln.lane, 2 * p.do_sr);
  // The fetched step's head of the group and tile, kFetch steps ahead.
  int fh = h0, ft = tbeg + (s0 - h0 * per), fs = s0;
  auto fetch = [&]() __attribute__((always_inline)) {
    const int s = (fs - s0) % kBwdSlots, rows = fs < s1 ? nq : 0;
    const long long head = kv * p.group + min(fh, p.group - 1);
    fq.run(static_cast<const T*>(p.q) + (head * p.q_sh + (long long)q0 * p.q_sr), 2 * p.q_sr,
           ft * L::kRows, rows, ring[s][0], wave);
    fd.run(static_cast<const T*>(p.dout) + (head * p.do_sh + (long long)q0 * p.do_sr),
           2 * p.do_sr, ft * L::kRows, rows, ring[s][1], wave);
    // every wave all of them, to the same place: its own wait then covers them
    const i32x4_t rs =
        rows_rsrc<8>(p.stats + (head * p.rows + q0 + (long long)ft * L::kRows),
                     tile_rows(rows - ft * L::kRows, L::kRows), 8);
#pragma unroll
    for (int i = 0; i < kStatLoads; ++i) {
      const int x = 64 * i + ln.lane;
      load_lds4(rs, 8 * (x % L::kRows) + 4 * (x / L::kRows), stat[s] + 256 * i);
    }
    ++fs;
    if (++ft == tbeg + per) {
      ft = tbeg;
      ++fh;
    }
  };
  fetch();
  fetch();
  V8 kf[L::kSteps], vf[L::kSteps];
  ln.own_rows(static_cast<const T*>(p.k) + (kv * p.k_sh + (long long)k0 * p.k_sr), p.k_sr, my, nk,
              kf);
  ln.own_rows(static_cast<const T*>(p.v) + (kv * p.v_sh + (long long)k0 * p.v_sr), p.v_sr, my, nk,
              vf);
  __builtin_amdgcn_s_waitcnt(0);
  float16_t dk[L::kCols], dv[L::kCols];
#pragma unroll
  for (int c = 0; c < L::kCols; ++c) dk[c] = dv[c] = zero16();
  int t = tbeg + (s0 - h0 * per);
  for (int step = s0; step < s1; ++step) {
    sync_ring<kLoads>();
    fetch();
    const int base = t * L::kRows, s = (step - s0) % kBwdSlots;
    if (++t == tbeg + per) t = tbeg;
    // (queries of the tile that see one of this wave's keys)
    if (min(base + L::kRows, nq) - 1 + coff < kw || kw >= nk) continue;
    const uint8_t* const qt = ring[s][0];
    const uint8_t* const dt = ring[s][1];
    const float* const st_lse = reinterpret_cast<const float*>(stat[s]);
    const float* const st_delta = st_lse + L::kRows;
    const bool edge = base + L::kRows > nq || base + coff < kw + 31;
    const int lo = my - coff;  // queries from lo on see this lane's key
    V8 pp[L::kBlocks][2], ds[L::kBlocks][2];
#pragma unroll
    for (int b = 0; b < L::kBlocks; ++b) {
      float16_t sc = zero16(), dp = zero16();
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st) sc = E::mfma(ln.rows_op(qt, b, st), kf[st], sc);
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st) dp = E::mfma(ln.rows_op(dt, b, st), vf[st], dp);
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const int at = 32 * b + 8 * i4 + 4 * ln.g;
        const float4 ls = *reinterpret_cast<const float4*>(st_lse + at);
        const float4 de = *reinterpret_cast<const float4*>(st_delta + at);
        const float lsv[4] = {ls.x, ls.y, ls.z, ls.w}, dev[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * i4 + e, q = base + at + e;
          float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], p.scale_log2, -lsv[e]));
          float y = x * (dp[i] - dev[e]);
          if (edge && (q < lo || q >= nq)) x = y = 0.0f;
          pp[b][i >> 3][i & 7] = (T)x;
          ds[b][i >> 3][i & 7] = (T)y;
        }
      }
    }
    auto add = [&](const uint8_t* tile, float16_t (&acc)[L::kCols], const V8 (&w)[L::kBlocks][2],
                   bool as_nan) __attribute__((always_inline)) {
      V8 a[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) a[u] = ln.cols_op(tile, u % L::kCols, u / L::kCols);
      if (edge)
        add_odd<D, T>(
            tile, a, acc, ln.g, [&](int j) { return base + j >= lo && base + j < nq; }, as_nan,
            [](int row) { return both_swz<D>(row); });
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int tt = u / L::kCols;
        acc[u % L::kCols] = E::mfma(a[u], w[tt >> 1][tt & 1], acc[u % L::kCols]);
      }
    };
    add(dt, dv, pp, false);
    add(qt, dk, ds, true);
  }
  __builtin_amdgcn_s_waitcnt(0);
  if (p.parts > 1) {
    float* const x =
        p.part + (((long long)part * p.kv_heads + kv) * p.key_rows + k0) * (2 * D);
    ln.store_part(x, my, nk, dk);
    ln.store_part(x + D, my, nk, dv);
  } else {
    ln.store(static_cast<T*>(p.dk) + (kv * p.dk_sh + (long long)k0 * p.dk_sr), p.dk_sr, my, nk,
             p.scale, dk);
    ln.store(static_cast<T*>(p.dv) + (kv * p.dv_sh + (long long)k0 * p.dv_sr), p.dv_sr, my, nk,
             1.0f, dv);
  }
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
  constexpr int W = 4;
  hipLaunchKernelGGL((packed_dq_kernel<D, W, T>),
                     dim3((unsigned)packed_groups(g.rows, g.sequences, 32 * W, g.heads)),
                     dim3(64 * W), 0, st, g);
  hipLaunchKernelGGL(
      (packed_dkv_kernel<D, W, T, 1>),
      dim3((unsigned)packed_groups(g.key_rows, g.sequences, 32 * W, g.kv_heads * g.parts)),
      dim3(64 * W), 0, st, g);
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
