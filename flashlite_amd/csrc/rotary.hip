// Rotary positions for q and k rows, their gradient, and the serving form that
// stores rotated k and v in a paged cache (fl_attn_rotary, fl_attn_rotary_cache).
//
// Bound by memory: a row is read and written once.  A thread owns V pairs of
// one token (V columns of each half, or 2 V neighbours when interleaved) and
// walks a few heads with their sine and cosine in registers.

#include <algorithm>
#include <type_traits>

#include "fl_serve.h"

namespace fl {

namespace {

struct RotaryGeom {
  const void *q, *k, *v;
  void *q_out, *k_out;
  void *k_cache, *v_cache;
  long long q_st[3], k_st[3], v_st[3], qo_st[3], ko_st[3];  // {batch, head, row} elements
  long long kc_st[3], vc_st[3];                             // {block, head, row}
  const void* positions;
  long long pos_sb, pos_sr;
  const int64_t* slots;
  long long slot_sb, slot_sr, num_slots;
  const double* freqs;
  int pos64, pairs, batch, heads, kv_heads, rows, head_dim;
  int heads_per_thread;
  float scale, sign;
  FastDiv block;
};

template <class T, int N>
struct Vec {
  T x[N];
};
template <class T, int N>
using Aligned = Vec<T, N> __attribute__((aligned(sizeof(T) * N < 16 ? sizeof(T) * N : 16)));

template <class T, int N>
__device__ __forceinline__ void load(const T* p, T (&x)[N]) {
  __builtin_memcpy(x, __builtin_assume_aligned(p, sizeof(T) * N < 16 ? sizeof(T) * N : 16),
                   sizeof(T) * N);
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const T (&x)[N]) {
  __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T) * N < 16 ? sizeof(T) * N : 16), x,
                   sizeof(T) * N);
}

// Head h of the launch: q heads, then k heads, then (with a cache) v heads.
template <class T, bool INTER, int V, bool CACHE>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryGeom g) {
  const int groups = g.head_dim / (2 * V);  // of 2 V columns a row
  const long long x = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long token = x / groups;
  const int j = (int)(x - token * groups);
  if (token >= (long long)g.batch * g.rows) return;
  const int b = (int)(token / g.rows);
  const int i = (int)(token - (long long)b * g.rows);
  long long slot = 0;
  if constexpr (CACHE) {
    slot = g.slots[b * g.slot_sb + i * g.slot_sr];
    if (slot < 0 || slot >= g.num_slots) return;
  }
  const bool turns = j * V < g.pairs;
  float cs[V], sn[V];
  if (turns) {
    const long long at = b * g.pos_sb + i * g.pos_sr;
    const double position = g.pos64 ? (double)static_cast<const int64_t*>(g.positions)[at]
                                    : (double)static_cast<const int32_t*>(g.positions)[at];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // Half turns in 64 bits, reduced to [-1, 1] before the rounding to 32:
      // positions of 2^20 and more lose nothing.
      double half_turns = position * (g.freqs[j * V + e] * 0.31830988618379067154);
      half_turns -= 2.0 * rint(0.5 * half_turns);
      sincospif((float)half_turns, &sn[e], &cs[e]);
      cs[e] *= g.scale;
      sn[e] *= g.scale * g.sign;
    }
  }
  // Columns: V at c0 and V at c1 (neighbours but in a rotated half pair).
  const int c0 = turns && !INTER ? j * V : 2 * j * V;
  const int c1 = turns && !INTER ? g.pairs + j * V : 2 * j * V + V;
  const int total = g.heads + g.kv_heads * (CACHE ? 2 : 1);
  const int h0 = blockIdx.y * g.heads_per_thread;
  const int h1 = min(h0 + g.heads_per_thread, total);
  for (int h = h0; h < h1; ++h) {
    const T* src;
    T* dst;
    bool turn = turns;
    if (h < g.heads) {
      src = static_cast<const T*>(g.q) + (b * g.q_st[0] + h * g.q_st[1] + i * g.q_st[2]);
      dst = static_cast<T*>(g.q_out) + (b * g.qo_st[0] + h * g.qo_st[1] + i * g.qo_st[2]);
    } else if (h < g.heads + g.kv_heads) {
      const int hk = h - g.heads;
      src = static_cast<const T*>(g.k) + (b * g.k_st[0] + hk * g.k_st[1] + i * g.k_st[2]);
      if constexpr (CACHE) {
        const long long blk = slot / g.block.d, row = slot - blk * g.block.d;
        dst = static_cast<T*>(g.k_cache) + (blk * g.kc_st[0] + hk * g.kc_st[1] + row * g.kc_st[2]);
      } else {
        dst = static_cast<T*>(g.k_out) + (b * g.ko_st[0] + hk * g.ko_st[1] + i * g.ko_st[2]);
      }
    } else {
      const int hk = h - g.heads - g.kv_heads;
      const long long blk = slot / g.block.d, row = slot - blk * g.block.d;
      src = static_cast<const T*>(g.v) + (b * g.v_st[0] + hk * g.v_st[1] + i * g.v_st[2]);
      dst = static_cast<T*>(g.v_cache) + (blk * g.vc_st[0] + hk * g.vc_st[1] + row * g.vc_st[2]);
      turn = false;
    }
    T x0[V], x1[V];
    load<T, V>(src + c0, x0);
    load<T, V>(src + c1, x1);
    if (turn) {
      if constexpr (INTER) {
        T y[2 * V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          y[e] = x0[e];
          y[V + e] = x1[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float a = (float)y[2 * e], c = (float)y[2 * e + 1];
          y[2 * e] = (T)(a * cs[e] - c * sn[e]);
          y[2 * e + 1] = (T)(a * sn[e] + c * cs[e]);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x0[e] = y[e];
          x1[e] = y[V + e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float a = (float)x0[e], c = (float)x1[e];
          x0[e] = (T)(a * cs[e] - c * sn[e]);
          x1[e] = (T)(a * sn[e] + c * cs[e]);
        }
      }
    }
    store<T, V>(dst + c0, x0);
    store<T, V>(dst + c1, x1);
  }
}

template <class T, bool CACHE, int V>
void launch(const RotaryGeom& g, bool inter, dim3 grid, hipStream_t stream) {
  if (inter)
    hipLaunchKernelGGL((rotary_kernel<T, true, V, CACHE>), grid, dim3(256), 0, stream, g);
  else
    hipLaunchKernelGGL((rotary_kernel<T, false, V, CACHE>), grid, dim3(256), 0, stream, g);
}

template <class T, bool CACHE>
void launch_any(RotaryGeom& g, bool inter, hipStream_t stream) {
  constexpr int kMost = 16 / (int)sizeof(T);
  int v = kMost;
  while (g.pairs % v != 0) v /= 2;
  const long long threads = (long long)g.batch * g.rows * (g.head_dim / (2 * v));
  const int total = g.heads + g.kv_heads * (CACHE ? 2 : 1);
  const long long blocks = (threads + 255) / 256;
  int per = 8;
  while (per > 1 && blocks * ((total + per - 1) / per) < 2048) per /= 2;
  g.heads_per_thread = per;
  const dim3 grid((unsigned)blocks, (unsigned)((total + per - 1) / per));
  if (v == 8) {
    if constexpr (kMost == 8) launch<T, CACHE, 8>(g, inter, grid, stream);
  } else if (v == 4) {
    launch<T, CACHE, 4>(g, inter, grid, stream);
  } else if (v == 2) {
    launch<T, CACHE, 2>(g, inter, grid, stream);
  } else {
    launch<T, CACHE, 1>(g, inter, grid, stream);
  }
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
  g.batch = (int)p.batch;
  g.heads = (int)p.heads;
  g.kv_heads = p.k ? (int)p.kv_heads : 0;
  g.rows = (int)p.rows;
  g.head_dim = (int)p.head_dim;
  g.scale = (float)p.scale;
  g.sign = p.transpose ? -1.0f : 1.0f;
  const bool inter = p.interleaved != 0;
  if (c != nullptr) {
    g.v = c->v;
    g.k_cache = c->k_cache;
    g.v_cache = c->v_cache;
    for (int i = 0; i < 3; ++i) {
      g.v_st[i] = c->v_stride[i];
      g.kc_st[i] = c->k_cache_stride[i];
      g.vc_st[i] = c->v_cache_stride[i];
    }
    g.slots = c->slots;
    g.slot_sb = c->slot_stride[0];
    g.slot_sr = c->slot_stride[1];
    g.num_slots = c->num_blocks * c->block_size;
    g.block = fast_div((int)c->block_size);
    if (p.dtype == FL_DTYPE_BF16)
      launch_any<__bf16, true>(g, inter, stream);
    else
      launch_any<_Float16, true>(g, inter, stream);
  } else if (p.dtype == FL_DTYPE_F32) {
    launch_any<float, false>(g, inter, stream);
  } else if (p.dtype == FL_DTYPE_BF16) {
    launch_any<__bf16, false>(g, inter, stream);
  } else {
    launch_any<_Float16, false>(g, inter, stream);
  }
  return hipGetLastError();
}

}  // namespace fl
