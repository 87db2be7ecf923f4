// Rotary positions for q and k rows, their gradient, and the serving form that
// stores rotated k and v in a paged cache (fl_attn_rotary, fl_attn_rotary_cache).
//
// Bound by memory: a row is read and written once (B1 H16/16 N16384 D 128
// fp16 5.5-6.2 TB/s, fp32 5.3, into a cache B4 H32/8 N4096 5.4); small calls by
// their launch, and in fp32 by 64-bit sines (B2 H8/8 N1999 D 64 7.4 us, 6.9 with
// the hardware's, which are not exact enough for it).  A thread owns V pairs of
// one token and walks a few heads with their sines and cosines in registers,
// the loads of four heads at a time in flight.

#include <algorithm>

#include "fl_serve.h"

namespace fl {

namespace {

// Work-groups that a launch should have, by fewer heads a thread: the sines
// and cosines of a token are then computed more often, but the chip is full.
constexpr int kLeastBlocks = 256;
// Heads side by side, and lanes that they take at most.
constexpr int kAcross = 4, kAcrossLanes = 32;

struct RotaryGeom {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;  // k_out and v_out: the caches, with one
  long long q_st[3], k_st[3], v_st[3], qo_st[3];  // {batch, head, row} elements
  long long ko_st[3], vo_st[3];                   // the same, or {block, head, row}
  const void* positions;
  long long pos_sb, pos_sr;
  const int64_t* slots;
  long long slot_sb, slot_sr, num_slots;
  const double* freqs;
  int pos64, pairs, heads, kv_heads;
  uint32_t tokens;  // batch * rows
  int heads_per_thread, across_log2;
  float scale, sign;
  double scale64;
  FastDiv rows, block;
};

template <class T, int N>
__device__ __forceinline__ void load(const T* p, T (&x)[N]) {
  __builtin_memcpy(x, __builtin_assume_aligned(p, sizeof(T) * N), sizeof(T) * N);
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const T (&x)[N]) {
  __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T) * N), x, sizeof(T) * N);
}

// A thread owns V columns at c0 and V at c1 of one token, the V pairs between
// them (V / 2 within each when interleaved: neighbouring threads then read
// neighbouring columns in both layouts), or V of either half of the columns
// behind the rotated ones.  Head h of the launch: q heads, then k heads, then (with a cache) v
// heads.
template <class T, int D, bool INTER, int V, bool CACHE, int UNROLL>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryGeom g) {
  constexpr uint32_t kThreads = D / (2 * V);  // a row
  const uint32_t x = blockIdx.x * 256 + threadIdx.x;
  const uint32_t token = x / kThreads >> g.across_log2;
  const int j = (int)(x % kThreads);
  const int across = 1 << g.across_log2;  // heads side by side
  if (token >= g.tokens) return;
  const int b = divide((int)token, g.rows);
  const int i = (int)token - b * g.rows.d;
  long long blk = b, row = i;  // where k (and v) go
  if constexpr (CACHE) {
    const long long slot = g.slots[b * g.slot_sb + i * g.slot_sr];
    if (slot < 0 || slot >= g.num_slots) return;
    if (((uint64_t)slot >> 31) == 0)
      blk = divide((int)slot, g.block);
    else
      blk = slot / g.block.d;
    row = slot - blk * g.block.d;
  }
  const bool turns = j * V < g.pairs;
  constexpr bool kHalves = !INTER || V > 1;
  const int rest = D - 2 * g.pairs;  // columns that are copied
  const int c0 = turns ? (kHalves ? j * V : 2 * j) : g.pairs + j * V;
  const int c1 = turns ? (kHalves ? g.pairs + j * V : 2 * j + 1) : c0 + rest / 2;
  const long long q_in = b * g.q_st[0] + i * g.q_st[2], k_in = b * g.k_st[0] + i * g.k_st[2],
                  v_in = CACHE ? b * g.v_st[0] + i * g.v_st[2] : 0;
  const long long q_to = b * g.qo_st[0] + i * g.qo_st[2],
                  k_to = blk * g.ko_st[0] + row * g.ko_st[2],
                  v_to = CACHE ? blk * g.vo_st[0] + row * g.vo_st[2] : 0;
  const int total = g.heads + g.kv_heads * (CACHE ? 2 : 1);
  // This thread's heads: h, h + across, .. below h1.
  const int span = g.heads_per_thread << g.across_log2;
  int h = blockIdx.y * span + (int)(x / kThreads & (uint32_t)(across - 1));
  const int h1 = min((int)(blockIdx.y + 1) * span, total);
  if (h >= h1) return;
  T x0[UNROLL][V], x1[UNROLL][V];
  T* to[UNROLL];
  auto fetch = [&]() __attribute__((always_inline)) {  // (past h1: the first again)
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int hu = h + u * across, hh = hu < h1 ? hu : h, hk = hh - g.heads;
      const T* from;
      if (hk < 0) {
        from = static_cast<const T*>(g.q) + (q_in + hh * g.q_st[1]);
        to[u] = static_cast<T*>(g.q_out) + (q_to + hh * g.qo_st[1]);
      } else if (!CACHE || hk < g.kv_heads) {
        from = static_cast<const T*>(g.k) + (k_in + hk * g.k_st[1]);
        to[u] = static_cast<T*>(g.k_out) + (k_to + hk * g.ko_st[1]);
      } else {
        from = static_cast<const T*>(g.v) + (v_in + (hk - g.kv_heads) * g.v_st[1]);
        to[u] = static_cast<T*>(g.v_out) + (v_to + (hk - g.kv_heads) * g.vo_st[1]);
      }
      load<T, V>(from + c0, x0[u]);
      load<T, V>(from + c1, x1[u]);
    }
  };
  fetch();
  float cs[V], sn[V];
  if (turns) {
    const long long at = b * g.pos_sb + i * g.pos_sr;
    const double position = g.pos64 ? (double)static_cast<const int64_t*>(g.positions)[at]
                                    : (double)static_cast<const int32_t*>(g.positions)[at];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int pair = !INTER ? j * V + e
                       : V == 1 ? j
                                : (e < V / 2 ? c0 / 2 + e : c1 / 2 + e - V / 2);
      // Turns in 64 bits, reduced to [-1/2, 1/2], so that far positions keep
      // what 64 bits have of them.  16-bit rows take the hardware's sine and
      // cosine of the turns in 32 bits: at most 2^-22 off, of a half step of
      // 2^-11 or more.  32-bit rows round the scaled sine and cosine once from
      // 64 bits.
      double t = position * (g.freqs[pair] * 0.15915494309189533577);
      t -= rint(t);
      if constexpr (sizeof(T) == 4) {
        double s64, c64;
        sincospi(2.0 * t, &s64, &c64);
        cs[e] = (float)(g.scale64 * c64);
        sn[e] = g.sign * (float)(g.scale64 * s64);
      } else {
        cs[e] = g.scale * __builtin_amdgcn_cosf((float)t);
        sn[e] = g.scale * g.sign * __builtin_amdgcn_sinf((float)t);
      }
    }
  }
  for (;;) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int hu = h + u * across;
      if (turns && (!CACHE || hu < g.heads + g.kv_heads)) {
        if constexpr (INTER && V > 1) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            T* const y = e < V / 2 ? &x0[u][2 * e] : &x1[u][2 * e - V];
            const float a = (float)y[0], c = (float)y[1];
            y[0] = (T)(a * cs[e] - c * sn[e]);
            y[1] = (T)(a * sn[e] + c * cs[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float a = (float)x0[u][e], c = (float)x1[u][e];
            x0[u][e] = (T)(a * cs[e] - c * sn[e]);
            x1[u][e] = (T)(a * sn[e] + c * cs[e]);
          }
        }
      }
      if (hu < h1) {
        store<T, V>(to[u] + c0, x0[u]);
        store<T, V>(to[u] + c1, x1[u]);
      }
    }
    h += UNROLL * across;
    if (h >= h1) return;
    fetch();
  }
}

template <class T, bool CACHE, int D, int V, int UNROLL>
void launch_unroll(const RotaryGeom& g, bool inter, dim3 grid, hipStream_t stream) {
  if (inter)
    hipLaunchKernelGGL((rotary_kernel<T, D, true, V, CACHE, UNROLL>), grid, dim3(256), 0, stream, g);
  else
    hipLaunchKernelGGL((rotary_kernel<T, D, false, V, CACHE, UNROLL>), grid, dim3(256), 0, stream,
                       g);
}

// Neighbouring threads go on to the next token, or where a token's heads lie
// closer together than its rows (projections [B, N, H, D]) first to the next of
// up to kAcross heads, so that a wave's accesses are whole pieces of memory.
// Heads a thread: as many as leave kLeastBlocks work-groups, at most 8; four
// of them (or one) in flight.
template <class T, bool CACHE, int D, int V>
void launch(RotaryGeom& g, bool inter, hipStream_t stream) {
  const int total = g.heads + g.kv_heads * (CACHE ? 2 : 1);
  const long long* const st = g.heads > 0 ? g.q_st : g.k_st;
  g.across_log2 = 0;
  if (st[1] < st[2])
    while (1 << g.across_log2 < kAcross && 2 << g.across_log2 <= total &&
           (D / (2 * V)) << (g.across_log2 + 1) <= kAcrossLanes &&
           ((int64_t)g.tokens * (D / (2 * V)) << (g.across_log2 + 1)) < (1LL << 32) - 256)
      ++g.across_log2;  // (threads are counted in 32 bits)
  const int64_t blocks =
      (((int64_t)g.tokens << g.across_log2) * (D / (2 * V)) + 255) / 256;
  const int each = (total + (1 << g.across_log2) - 1) >> g.across_log2;
  int per = 8;
  while (per > 1 && blocks * ((each + per - 1) / per) < kLeastBlocks) per /= 2;
  g.heads_per_thread = per;
  const dim3 grid((unsigned)blocks, (unsigned)((each + per - 1) / per));
  if (per >= 4)
    launch_unroll<T, CACHE, D, V, 4>(g, inter, grid, stream);
  else
    launch_unroll<T, CACHE, D, V, 1>(g, inter, grid, stream);
}

template <class T, bool CACHE, int D>
void launch_dim(RotaryGeom& g, bool inter, hipStream_t stream) {
  constexpr int kMost = 16 / (int)sizeof(T);
  int v = kMost;  // columns a load: 16 bytes where the pairs divide
  while (g.pairs % v != 0) v /= 2;
  if (v == 8) {
    if constexpr (kMost == 8) launch<T, CACHE, D, 8>(g, inter, stream);
  } else if (v == 4) {
    launch<T, CACHE, D, 4>(g, inter, stream);
  } else if (v == 2) {
    launch<T, CACHE, D, 2>(g, inter, stream);
  } else {
    launch<T, CACHE, D, 1>(g, inter, stream);
  }
}

template <class T, bool CACHE>
void launch_any(RotaryGeom& g, int head_dim, bool inter, hipStream_t stream) {
  if (head_dim == 128)
    launch_dim<T, CACHE, 128>(g, inter, stream);
  else
    launch_dim<T, CACHE, 64>(g, inter, stream);
}

}  // namespace

hipError_t launch_rotary(const fl_rotary_params& p, const fl_cache_store* c, hipStream_t stream) {
  RotaryGeom g = {};
  g.q = p.q;
  g.k = p.k;
  g.q_out = p.q_out;
  g.k_out = p.k_out;
  for (int i = 0; i < 3; ++i) {
    g.q_st[i] = p.q_stride[i];
    g.k_st[i] = p.k_stride[i];
    g.qo_st[i] = p.q_out_stride[i];
    g.ko_st[i] = p.k_out_stride[i];
  }
  g.positions = p.positions;
  g.pos_sb = p.position_stride[0];
  g.pos_sr = p.position_stride[1];
  g.pos64 = p.position_bits == 64;
  g.freqs = p.freqs;
  g.pairs = (int)p.pairs;
  g.heads = (int)p.heads;
  g.kv_heads = p.k ? (int)p.kv_heads : 0;
  g.tokens = (uint32_t)(p.batch * p.rows);
  g.rows = fast_div((int)p.rows);
  g.scale = (float)p.scale;
  g.scale64 = p.scale;
  g.sign = p.transpose ? -1.0f : 1.0f;
  const bool inter = p.interleaved != 0;
  const int d = (int)p.head_dim;
  if (c != nullptr) {
    g.v = c->v;
    g.k_out = c->k_cache;
    g.v_out = c->v_cache;
    for (int i = 0; i < 3; ++i) {
      g.v_st[i] = c->v_stride[i];
      g.ko_st[i] = c->k_cache_stride[i];
      g.vo_st[i] = c->v_cache_stride[i];
    }
    g.slots = c->slots;
    g.slot_sb = c->slot_stride[0];
    g.slot_sr = c->slot_stride[1];
    g.num_slots = c->num_blocks * c->block_size;
    g.block = fast_div((int)c->block_size);
    if (p.dtype == FL_DTYPE_BF16)
      launch_any<__bf16, true>(g, d, inter, stream);
    else
      launch_any<_Float16, true>(g, d, inter, stream);
  } else if (p.dtype == FL_DTYPE_F32) {
    launch_any<float, false>(g, d, inter, stream);
  } else if (p.dtype == FL_DTYPE_BF16) {
    launch_any<__bf16, false>(g, d, inter, stream);
  } else {
    launch_any<_Float16, false>(g, d, inter, stream);
  }
  return hipGetLastError();
}

}  // namespace fl
