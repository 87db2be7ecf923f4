// Norms of query and key rows for each head with the rotary positions in the
// same pass, their gradients, and the serving form that stores k and v in a
// paged cache (fl_attn_norm_rotary, fl_attn_norm_rotary_bwd,
// fl_attn_norm_rotary_cache).
//
//   y = R(x r w),  r = 1 / sqrt(mean(x x) + eps), R the rotation of the pairs
//   g = R' dy,  dw = sum over the rows of g x r,
//   dx = r (g w - x r^2 mean(g w x))
//
// Bound by memory: every row is read and written once (the gradient reads the
// row and dy): B2 H32/8 N4096 D 128 bf16 with three axes 37.8 us (4.4 TB/s),
// back 56.5 (4.5), into a cache B4 H32/8 N4096 fp16 80 (5.0), where torch's
// copy_ reaches 5.15; small calls by their launch and the chain of loads
// (B1 H8/2 N333 D 64 4.7 us).  A thread owns V pairs of one token and walks
// heads with their sines and cosines in registers; the D / 2V threads of a row,
// neighbours in a wave, add up its sums across lanes in 32 bits, and each value
// is rounded once, at the end.  dw is summed in a work-group's registers and
// LDS, then over the work-groups by a second kernel in a fixed order: no
// atomics, the same bits every time.

#include <algorithm>
#include <type_traits>

#include "fl_serve.h"

namespace fl {

namespace {

constexpr int kAcross = 4, kAcrossLanes = 32;

enum { kForward, kStore, kBackward };

// Most work-groups of a gradient's launch: the partial sums of the weights.
constexpr int kBackGroups = 2048;
// Up to so many steps of tiles are a work-group each (norm_rotary_step_kernel):
// B1 H32/8 N1000 D 128 8.0 us, 8.7 with the other kernel.
constexpr int kStepGroups = 2048;
// Otherwise a launch has at least this many work-groups, by shares of the heads
// (B1 H32/8 N2500 D 128 back 23.2 us, with 256 work-groups 28.2).
constexpr int kLeastGroups = 512;

struct NormRows {
  const void* in;   // x; backward: dy
  const void* x;    // backward: x
  void* out;        // y, a cache, or dx
  const void* weight;  // null: neither normed nor scaled
  long long in_st[3], x_st[3];
  long long out_st[3];  // {batch, head, row}, or {block, head, row} of a cache
  int heads, steps;  // steps of a walk over the heads
};

struct NormGeom {
  NormRows rows[3];  // q, k, v
  const void* positions;
  long long pos_sa, pos_sb, pos_sr;
  const int32_t* axes;
  int num_axes;
  const int64_t* slots;
  long long slot_sb, slot_sr, num_slots;
  const double* freqs;
  float* part;  // backward: [q, k][work-groups][D]
  int pos64, pairs, weight32;
  uint32_t tokens;  // batch * rows
  int tile, tiles, across_log2, share;
  float scale, sign, eps, offset;
  double scale64;
  FastDiv by_rows, by_pairs, block;
};

template <class T, int N>
__device__ __forceinline__ void load(const T* p, T (&x)[N]) {
  __builtin_memcpy(x, __builtin_assume_aligned(p, sizeof(T) * N), sizeof(T) * N);
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const T (&x)[N]) {
  __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T) * N), x, sizeof(T) * N);
}

// N bytes as they are.
template <int N>
struct Raw {
  typedef uint32_t type __attribute__((ext_vector_type(N / 4)));
};
template <>
struct Raw<4> {
  using type = uint32_t;
};
template <>
struct Raw<2> {
  using type = uint16_t;
};

// Sum over groups of N neighbouring lanes (a power of two), in all of them.
template <int N>
__device__ __forceinline__ float group_sum(float x) {
  auto dpp = [&](auto ctrl) __attribute__((always_inline)) {
    const int y = __builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, 0xf, 0xf,
                                              true);
    x += __int_as_float(y);
  };
  if constexpr (N >= 2) dpp(std::integral_constant<int, 0xB1>{});   // quad_perm 1 0 3 2
  if constexpr (N >= 4) dpp(std::integral_constant<int, 0x4E>{});   // quad_perm 2 3 0 1
  if constexpr (N >= 8) dpp(std::integral_constant<int, 0x141>{});  // row_half_mirror
  if constexpr (N >= 16) dpp(std::integral_constant<int, 0x140>{});  // row_mirror
  if constexpr (N >= 32) x += __shfl_xor(x, 16);
  if constexpr (N >= 64) x += __shfl_xor(x, 32);
  return x;
}

// Sum over the lanes l, l + N, l + 2N, .. of a wave.
template <int N>
__device__ __forceinline__ float stride_sum(float x) {
#pragma unroll
  for (int d = N; d < 64; d *= 2) x += __shfl_xor(x, d);
  return x;
}

// A thread's columns of a row, V at c0 and V at c1 (as in rotary_kernel).
template <int D, bool INTER, int V>
struct Columns {
  int c0, c1;
  bool paired;  // they turn
  __device__ __forceinline__ Columns(int j, int pairs) {
    constexpr bool kHalves = !INTER || V > 1;
    paired = j * V < pairs;
    c0 = paired ? (kHalves ? j * V : 2 * j) : pairs + j * V;
    c1 = paired ? (kHalves ? pairs + j * V : 2 * j + 1) : c0 + (D - 2 * pairs) / 2;
  }
  // The pair of its e-th sine and cosine.
  __device__ __forceinline__ int pair(int j, int e) const {
    return !INTER ? j * V + e : V == 1 ? j : (e < V / 2 ? c0 / 2 + e : c1 / 2 + e - V / 2);
  }
};

template <class T, int V>
__device__ __forceinline__ void load_weight(const NormGeom& g, const void* w, int c0, int c1,
                                            float (&w0)[V], float (&w1)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) w0[e] = w1[e] = 1.0f;
  if (w == nullptr) return;
  if (g.weight32) {
    load<float, V>(static_cast<const float*>(w) + c0, w0);
    load<float, V>(static_cast<const float*>(w) + c1, w1);
  } else {
    T t0[V], t1[V];
    load<T, V>(static_cast<const T*>(w) + c0, t0);
    load<T, V>(static_cast<const T*>(w) + c1, t1);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w0[e] = (float)t0[e];
      w1[e] = (float)t1[e];
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    w0[e] += g.offset;
    w1[e] += g.offset;
  }
}

// {cosine, sine} of a token's pair.  Turns in 64 bits, reduced to [-1/2, 1/2];
// 16-bit rows take the hardware's sine and cosine of them in 32 bits, 32-bit
// rows round the scaled ones once from 64 bits (rotary.hip).
template <class T>
__device__ __forceinline__ float2 turn_of(const NormGeom& g, int b, int i, int pair) {
  long long at = b * g.pos_sb + i * g.pos_sr;
  if (g.axes != nullptr) at += min(max(g.axes[pair], 0), g.num_axes - 1) * g.pos_sa;
  const double position = g.pos64 ? (double)static_cast<const int64_t*>(g.positions)[at]
                                  : (double)static_cast<const int32_t*>(g.positions)[at];
  double t = position * (g.freqs[pair] * 0.15915494309189533577);
  t -= rint(t);
  if constexpr (sizeof(T) == 4) {
    double s64, c64;
    sincospi(2.0 * t, &s64, &c64);
    return make_float2((float)(g.scale64 * c64), g.sign * (float)(g.scale64 * s64));
  } else {
    return make_float2(g.scale * __builtin_amdgcn_cosf((float)t),
                       g.scale * g.sign * __builtin_amdgcn_sinf((float)t));
  }
}

// One row's columns in y (forward: x, to y; backward: dy, to dx, x its row and
// s the weight's gradient).
template <class T, int D, bool INTER, int V, bool BACK>
__device__ __forceinline__ void norm_row(T (&y0)[V], T (&y1)[V], const T (&x0)[V], const T (&x1)[V],
                                         const float (&w0)[V], const float (&w1)[V],
                                         const float (&cs)[V], const float (&sn)[V], bool norm,
                                         bool paired, float eps, bool live, float (&s0)[V],
                                         float (&s1)[V]) {
  constexpr int kThreads = D / (2 * V);
  float a[V], c[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    a[e] = (float)y0[e];
    c[e] = (float)y1[e];
  }
  auto turn = [&]() __attribute__((always_inline)) {
    if (!paired) return;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float* const p = INTER && V > 1 ? (e < V / 2 ? &a[2 * e] : &c[2 * e - V]) : &a[e];
      float* const q = INTER && V > 1 ? p + 1 : &c[e];
      const float u = *p, v = *q;
      *p = u * cs[e] - v * sn[e];
      *q = u * sn[e] + v * cs[e];
    }
  };
  if constexpr (!BACK) {
    if (norm) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) ss += a[e] * a[e] + c[e] * c[e];
      ss = group_sum<kThreads>(ss);
      const float r = __builtin_amdgcn_rsqf(ss * (1.0f / D) + eps);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        a[e] *= r * w0[e];
        c[e] *= r * w1[e];
      }
    }
    turn();
  } else {
    turn();  // g
    if (norm) {
      float p[V], q[V], ss = 0.0f, dot = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        p[e] = (float)x0[e];
        q[e] = (float)x1[e];
        ss += p[e] * p[e] + q[e] * q[e];
        dot += a[e] * w0[e] * p[e] + c[e] * w1[e] * q[e];
      }
      ss = group_sum<kThreads>(ss);
      dot = group_sum<kThreads>(dot);
      const float r = __builtin_amdgcn_rsqf(ss * (1.0f / D) + eps);
      const float along = dot * (1.0f / D) * r * r;
      const float mine = live ? r : 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (live) {
          s0[e] += a[e] * (p[e] * mine);
          s1[e] += c[e] * (q[e] * mine);
        }
        a[e] = r * (a[e] * w0[e] - p[e] * along);
        c[e] = r * (c[e] * w1[e] - q[e] * along);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    y0[e] = (T)a[e];
    y1[e] = (T)c[e];
  }
}

// A thread's token, and where its rows go.
struct NormToken {
  int b, i;
  bool there;
  long long blk, row;  // of k and v
};

template <int MODE>
__device__ __forceinline__ NormToken norm_token(const NormGeom& g, uint32_t token) {
  NormToken t;
  t.there = token < g.tokens;
  t.b = divide((int)(t.there ? token : 0u), g.by_rows);
  t.i = (int)(t.there ? token : 0u) - t.b * g.by_rows.d;
  t.blk = t.b;
  t.row = t.i;
  if constexpr (MODE == kStore) {
    const long long slot = t.there ? g.slots[t.b * g.slot_sb + t.i * g.slot_sr] : -1;
    t.there = slot >= 0 && slot < g.num_slots;
    if (t.there) {
      t.blk = ((uint64_t)slot >> 31) == 0 ? divide((int)slot, g.block) : slot / g.block.d;
      t.row = slot - t.blk * g.block.d;
    }
  }
  return t;
}

template <class T, int MODE>
__device__ __forceinline__ T* norm_out(const NormRows& n, const NormToken& t, bool to_cache) {
  return static_cast<T*>(n.out) +
         (MODE == kStore && to_cache ? t.blk * n.out_st[0] + t.row * n.out_st[2]
                                     : t.b * n.out_st[0] + t.i * n.out_st[2]);
}

// The work-group's share of the weights' gradients, s[t] of q's (0) and k's.
template <int D, int V>
__device__ __forceinline__ void store_sums(const NormGeom& g, float (&sums)[8][D], int c0, int c1,
                                           const float (&s0)[2][V], const float (&s1)[2][V]) {
  constexpr int kThreads = D / (2 * V);
  if (g.part == nullptr) return;  // (no weight's gradient is wanted)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = stride_sum<kThreads>(s0[t][e]), c = stride_sum<kThreads>(s1[t][e]);
      if (lane < kThreads) {
        sums[4 * t + wave][c0 + e] = a;
        sums[4 * t + wave][c1 + e] = c;
      }
    }
  __syncthreads();
  const long long groups = (long long)gridDim.x * gridDim.y;
  const long long me = (long long)blockIdx.y * gridDim.x + blockIdx.x;
  for (int x = threadIdx.x; x < 2 * D; x += 256) {
    const int t = x / D, c = x % D;
    g.part[(t * groups + me) * D + c] =
        (sums[4 * t][c] + sums[4 * t + 1][c]) + (sums[4 * t + 2][c] + sums[4 * t + 3][c]);
  }
}

// Few rows: a work-group one step of one tile of tokens, blockIdx.y its step
// (q's heads, then k's, then v's); everything it needs is loaded at once.
template <class T, int D, bool INTER, int V, int MODE>
__global__ void __launch_bounds__(256) norm_rotary_step_kernel(const NormGeom g) {
  constexpr int kThreads = D / (2 * V);  // a row
  constexpr bool kBack = MODE == kBackward;
  const int j = (int)threadIdx.x % kThreads, group = (int)threadIdx.x / kThreads;
  const Columns<D, INTER, V> at(j, g.pairs);
  int step = blockIdx.y, tensor = 0;
  while (tensor < 2 && step >= g.rows[tensor].steps) step -= g.rows[tensor++].steps;
  const NormRows& n = g.rows[tensor];
  const bool norm = n.weight != nullptr, turns = at.paired && tensor < 2;
  const NormToken t = norm_token<MODE>(
      g, (uint32_t)blockIdx.x * (uint32_t)g.tile + (uint32_t)(group >> g.across_log2));
  const int head = (step << g.across_log2) + (group & ((1 << g.across_log2) - 1));
  const int h = min(head, n.heads - 1);
  T y0[V], y1[V], x0[V], x1[V];
  const T* const in = static_cast<const T*>(n.in) + (t.b * n.in_st[0] + t.i * n.in_st[2] +
                                                     h * n.in_st[1]);
  load<T, V>(in + at.c0, y0);
  load<T, V>(in + at.c1, y1);
#pragma unroll
  for (int e = 0; e < V; ++e) x0[e] = x1[e] = (T)0.0f;
  if (kBack && norm) {
    const T* const x = static_cast<const T*>(n.x) + (t.b * n.x_st[0] + t.i * n.x_st[2] +
                                                     h * n.x_st[1]);
    load<T, V>(x + at.c0, x0);
    load<T, V>(x + at.c1, x1);
  }
  float w0[V], w1[V], cs[V], sn[V], s0[2][V], s1[2][V];
  load_weight<T, V>(g, n.weight, at.c0, at.c1, w0, w1);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s0[0][e] = s0[1][e] = s1[0][e] = s1[1][e] = 0.0f;
    const float2 x = turns ? turn_of<T>(g, t.b, t.i, at.pair(j, e)) : make_float2(1.0f, 0.0f);
    cs[e] = x.x;
    sn[e] = x.y;
  }
  const bool live = t.there && head < n.heads;
  if (tensor < 2) {
    float a0[V], a1[V];
#pragma unroll
    for (int e = 0; e < V; ++e) a0[e] = a1[e] = 0.0f;
    norm_row<T, D, INTER, V, kBack>(y0, y1, x0, x1, w0, w1, cs, sn, norm, turns, g.eps, live, a0,
                                    a1);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s0[0][e] = tensor == 0 ? a0[e] : 0.0f;
      s1[0][e] = tensor == 0 ? a1[e] : 0.0f;
      s0[1][e] = tensor == 0 ? 0.0f : a0[e];
      s1[1][e] = tensor == 0 ? 0.0f : a1[e];
    }
  }
  if (live) {
    T* const out = norm_out<T, MODE>(n, t, tensor > 0) + h * n.out_st[1];
    store<T, V>(out + at.c0, y0);
    store<T, V>(out + at.c1, y1);
  }
  if constexpr (kBack) {
    __shared__ float sums[8][D];
    store_sums<D, V>(g, sums, at.c0, at.c1, s0, s1);
  }
}

// Many rows: a work-group walks the heads of a tile of tokens (g.tile of
// them), q's, then k's, then v's, 1 << g.across_log2 side by side, or blockIdx.y's
// share of them.  The tile's sines and cosines are computed once, into LDS: done
// by each thread for its own pairs, with the loads of positions and frequencies,
// they cost as much as the rows of several heads.
template <class T, int D, bool INTER, int V, int MODE>
__global__ void __launch_bounds__(256, 4) norm_rotary_kernel(const NormGeom g) {
  constexpr int kThreads = D / (2 * V);  // a row
  constexpr bool kBack = MODE == kBackward;
  __shared__ float2 table[256 * V];  // {cosine, sine} [token][pair]
  const int j = (int)threadIdx.x % kThreads, group = (int)threadIdx.x / kThreads;
  const int side = group & ((1 << g.across_log2) - 1), own = group >> g.across_log2;
  const Columns<D, INTER, V> at(j, g.pairs);
  float s0[2][V], s1[2][V];  // gradients of q's and k's weights
#pragma unroll
  for (int e = 0; e < V; ++e) s0[0][e] = s0[1][e] = s1[0][e] = s1[1][e] = 0.0f;

  for (int tile = blockIdx.x; tile < g.tiles; tile += gridDim.x) {
    const uint32_t first = (uint32_t)tile * (uint32_t)g.tile;
    const NormToken t = norm_token<MODE>(g, first + (uint32_t)own);
    if (tile != (int)blockIdx.x) __syncthreads();  // the last tile's table has been read
    for (int x = threadIdx.x; x < g.tile * g.pairs; x += 256) {
      const int of = divide(x, g.by_pairs), pair = x - of * g.by_pairs.d;
      const uint32_t tk = min(first + (uint32_t)of, g.tokens - 1);
      const int b = divide((int)tk, g.by_rows);
      table[x] = turn_of<T>(g, b, (int)tk - b * g.by_rows.d, pair);
    }
    __syncthreads();
    float cs[V], sn[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float2 x = at.paired ? table[own * g.pairs + at.pair(j, e)] : make_float2(1.0f, 0.0f);
      cs[e] = x.x;
      sn[e] = x.y;
    }
    const int s_from = blockIdx.y * g.share, s_to = s_from + g.share;
    int before = 0;  // steps of the tensors before
    auto walk = [&](auto tensor) __attribute__((always_inline)) {
      constexpr int N = decltype(tensor)::value;
      const NormRows& n = g.rows[N];
      const bool norm = N < 2 && n.weight != nullptr;
      const T* const in = static_cast<const T*>(n.in) + (t.b * n.in_st[0] + t.i * n.in_st[2]);
      const T* const x_in =
          kBack ? static_cast<const T*>(n.x) + (t.b * n.x_st[0] + t.i * n.x_st[2]) : nullptr;
      T* const out = norm_out<T, MODE>(n, t, N > 0);
      float w0[V], w1[V];
      if constexpr (N < 2) load_weight<T, V>(g, n.weight, at.c0, at.c1, w0, w1);
      int step = max(s_from - before, 0);
      const int end = min(s_to - before, n.steps);
      before += n.steps;
      auto steps = [&](auto count) __attribute__((always_inline)) {
        constexpr int U = decltype(count)::value;  // heads in flight
        if constexpr (N == 2) {  // v: copied
          using R = typename Raw<V * (int)sizeof(T)>::type;
          R y0[U], y1[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int h = min(((step + u) << g.across_log2) + side, n.heads - 1);
            y0[u] = *reinterpret_cast<const R*>(in + h * n.in_st[1] + at.c0);
            y1[u] = *reinterpret_cast<const R*>(in + h * n.in_st[1] + at.c1);
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int h = ((step + u) << g.across_log2) + side;
            if (!t.there || h >= n.heads) continue;
            *reinterpret_cast<R*>(out + h * n.out_st[1] + at.c0) = y0[u];
            *reinterpret_cast<R*>(out + h * n.out_st[1] + at.c1) = y1[u];
          }
        } else {
          T y0[U][V], y1[U][V], x0[U][V], x1[U][V];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int h = min(((step + u) << g.across_log2) + side, n.heads - 1);
            load<T, V>(in + h * n.in_st[1] + at.c0, y0[u]);
            load<T, V>(in + h * n.in_st[1] + at.c1, y1[u]);
            if (kBack && norm) {
              load<T, V>(x_in + h * n.x_st[1] + at.c0, x0[u]);
              load<T, V>(x_in + h * n.x_st[1] + at.c1, x1[u]);
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int h = ((step + u) << g.across_log2) + side;
            const bool live = t.there && h < n.heads;
            norm_row<T, D, INTER, V, kBack>(y0[u], y1[u], x0[u], x1[u], w0, w1, cs, sn, norm,
                                            at.paired, g.eps, live, s0[N], s1[N]);
            if (live) {
              store<T, V>(out + h * n.out_st[1] + at.c0, y0[u]);
              store<T, V>(out + h * n.out_st[1] + at.c1, y1[u]);
            }
          }
        }
        step += U;
      };
      constexpr int kMost = kBack ? 2 : 4;
#pragma unroll 1
      while (end - step >= kMost) steps(std::integral_constant<int, kMost>{});
      if constexpr (kMost == 4)
        if (end - step >= 2) steps(std::integral_constant<int, 2>{});
      if (end > step) steps(std::integral_constant<int, 1>{});
    };
    walk(std::integral_constant<int, 0>{});
    walk(std::integral_constant<int, 1>{});
    if constexpr (MODE == kStore) walk(std::integral_constant<int, 2>{});
  }
  if constexpr (kBack) {
    __shared__ float sums[8][D];
    store_sums<D, V>(g, sums, at.c0, at.c1, s0, s1);
  }
}

// Sums `rows` rows of D partial sums: a work-group 16 columns of q's or k's
// (blockIdx.y), 64 threads a column.
__global__ void __launch_bounds__(1024) norm_weight_kernel(const float* part, int rows, int D,
                                                           float* q, float* k) {
  __shared__ float sums[64][16];
  float* const out = blockIdx.y == 0 ? q : k;
  if (out == nullptr) return;
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
  const float* const from = part + (long long)blockIdx.y * rows * D + c;
  float x = 0.0f;
#pragma unroll 8
  for (int i = r; i < rows; i += 64) x += from[(long long)i * D];
  sums[r][threadIdx.x & 15] = x;
  __syncthreads();
  for (int d = 32; d > 0; d >>= 1) {
    if (r < d) sums[r][threadIdx.x & 15] += sums[r + d][threadIdx.x & 15];
    __syncthreads();
  }
  if (r == 0) out[c] = sums[0][threadIdx.x];
}

// Neighbouring threads go on to the next token, or where heads lie closer
// together than rows first to the next of up to kAcross heads, so that a wave's
// accesses are whole pieces of memory.
template <class T, int D, int V, int MODE>
void launch(NormGeom& g, int tensors, bool inter, float* dq, float* dk, hipStream_t st) {
  constexpr int kThreads = D / (2 * V);
  const NormRows& n = g.rows[0].heads > 0 ? g.rows[0] : g.rows[1];
  g.across_log2 = 0;
  if (n.in_st[1] < n.in_st[2])
    while (1 << g.across_log2 < kAcross && 2 << g.across_log2 <= n.heads &&
           kThreads << (g.across_log2 + 1) <= kAcrossLanes)
      ++g.across_log2;
  g.tile = (256 / kThreads) >> g.across_log2;
  g.tiles = (int)((g.tokens + (uint32_t)g.tile - 1) / (uint32_t)g.tile);
  int steps = 0;
  for (int i = 0; i < tensors; ++i) {
    g.rows[i].steps = (g.rows[i].heads + (1 << g.across_log2) - 1) >> g.across_log2;
    steps += g.rows[i].steps;
  }
  const int64_t groups = (int64_t)g.tiles * std::max(steps, 1);
  dim3 grid((unsigned)g.tiles, (unsigned)steps);
  if (groups <= kStepGroups) {
    if (inter)
      hipLaunchKernelGGL((norm_rotary_step_kernel<T, D, true, V, MODE>), grid, dim3(256), 0, st, g);
    else
      hipLaunchKernelGGL((norm_rotary_step_kernel<T, D, false, V, MODE>), grid, dim3(256), 0, st,
                         g);
  } else {
    int shares = 1;
    while (shares < steps && g.tiles * shares < kLeastGroups) shares *= 2;
    g.share = (steps + shares - 1) / shares;
    shares = (steps + g.share - 1) / g.share;
    grid = dim3((unsigned)(MODE == kBackward ? std::min(g.tiles, kBackGroups / shares) : g.tiles),
                (unsigned)shares);
    if (inter)
      hipLaunchKernelGGL((norm_rotary_kernel<T, D, true, V, MODE>), grid, dim3(256), 0, st, g);
    else
      hipLaunchKernelGGL((norm_rotary_kernel<T, D, false, V, MODE>), grid, dim3(256), 0, st, g);
  }
  if (MODE == kBackward && (dq || dk))
    hipLaunchKernelGGL(norm_weight_kernel, dim3(D / 16, 2), dim3(1024), 0, st, g.part,
                       (int)(grid.x * grid.y), D, dq, dk);
}

template <class T, int D, int MODE>
void launch_dim(NormGeom& g, int tensors, bool inter, float* dq, float* dk, hipStream_t st) {
  // 16 bytes a load where the pairs divide; 8 in the backward pass, whose sums
  // and two rows then leave registers for four waves a SIMD (B2 H32/8 N4096
  // D 128 bf16 57 us against 65).
  constexpr int kMost = (MODE == kBackward ? 8 : 16) / (int)sizeof(T);
  int v = kMost;  // columns a load
  while (g.pairs % v != 0) v /= 2;
  if (v == 8) {
    if constexpr (kMost >= 8) launch<T, D, 8, MODE>(g, tensors, inter, dq, dk, st);
  } else if (v == 4) {
    if constexpr (kMost >= 4) launch<T, D, 4, MODE>(g, tensors, inter, dq, dk, st);
  } else if (v == 2) {
    launch<T, D, 2, MODE>(g, tensors, inter, dq, dk, st);
  } else {
    launch<T, D, 1, MODE>(g, tensors, inter, dq, dk, st);
  }
}

template <class T, int MODE>
void launch_any(NormGeom& g, int tensors, int d, bool inter, float* dq, float* dk, hipStream_t st) {
  if (d == 128)
    launch_dim<T, 128, MODE>(g, tensors, inter, dq, dk, st);
  else
    launch_dim<T, 64, MODE>(g, tensors, inter, dq, dk, st);
}

void strides(long long (&to)[3], const int64_t (&from)[3]) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

}  // namespace

hipError_t launch_norm_zero(const fl_rotary_params& p, float* dq, float* dk, hipStream_t stream) {
  // (sums of no rows)
  hipLaunchKernelGGL(norm_weight_kernel, dim3((unsigned)p.head_dim / 16, 2), dim3(1024), 0, stream,
                     nullptr, 0, (int)p.head_dim, dq, dk);
  return hipGetLastError();
}

int64_t norm_rotary_workspace_bytes(int64_t head_dim) {
  return 2 * (int64_t)kBackGroups * head_dim * 4;
}

hipError_t launch_norm_rotary(const fl_rotary_params& p, const fl_norm_params& nm,
                              const fl_cache_store* c, const fl_norm_grads* d, void* ws,
                              hipStream_t stream) {
  NormGeom g = {};
  NormRows &q = g.rows[0], &k = g.rows[1], &v = g.rows[2];
  q.in = p.q;
  q.out = p.q_out;
  q.weight = nm.q_weight;
  q.heads = (int)p.heads;
  strides(q.in_st, p.q_stride);
  strides(q.out_st, p.q_out_stride);
  k.in = p.k;
  k.out = p.k_out;
  k.weight = nm.k_weight;
  k.heads = p.k ? (int)p.kv_heads : 0;
  strides(k.in_st, p.k_stride);
  strides(k.out_st, p.k_out_stride);
  g.positions = p.positions;
  g.pos_sa = nm.axis_stride;
  g.pos_sb = p.position_stride[0];
  g.pos_sr = p.position_stride[1];
  g.pos64 = p.position_bits == 64;
  g.axes = nm.axes;
  g.num_axes = (int)nm.num_axes;
  g.freqs = p.freqs;
  g.pairs = (int)p.pairs;
  g.weight32 = nm.weight_dtype == FL_DTYPE_F32;
  g.tokens = (uint32_t)(p.batch * p.rows);
  g.by_rows = fast_div((int)p.rows);
  g.by_pairs = fast_div(std::max(1, (int)p.pairs));
  g.scale = (float)p.scale;
  g.scale64 = p.scale;
  g.sign = d ? -1.0f : 1.0f;
  g.eps = (float)nm.eps;
  g.offset = (float)nm.weight_offset;
  const bool inter = p.interleaved != 0;
  const int dim = (int)p.head_dim;
  if (c != nullptr) {
    k.out = c->k_cache;
    strides(k.out_st, c->k_cache_stride);
    v.in = c->v;
    v.out = c->v_cache;
    v.heads = k.heads;
    strides(v.in_st, c->v_stride);
    strides(v.out_st, c->v_cache_stride);
    g.slots = c->slots;
    g.slot_sb = c->slot_stride[0];
    g.slot_sr = c->slot_stride[1];
    g.num_slots = c->num_blocks * c->block_size;
    g.block = fast_div((int)c->block_size);
    if (p.dtype == FL_DTYPE_BF16)
      launch_any<__bf16, kStore>(g, 3, dim, inter, nullptr, nullptr, stream);
    else
      launch_any<_Float16, kStore>(g, 3, dim, inter, nullptr, nullptr, stream);
    return hipGetLastError();
  }
  const int tensors = 2;
  if (d != nullptr) {
    q.x = d->q;
    strides(q.x_st, d->q_stride);
    k.x = d->k;
    strides(k.x_st, d->k_stride);
    float *dq = q.weight ? d->dq_weight : nullptr, *dk = k.weight ? d->dk_weight : nullptr;
    g.part = dq || dk ? static_cast<float*>(ws) : nullptr;
    if (p.dtype == FL_DTYPE_F32)
      launch_any<float, kBackward>(g, tensors, dim, inter, dq, dk, stream);
    else if (p.dtype == FL_DTYPE_BF16)
      launch_any<__bf16, kBackward>(g, tensors, dim, inter, dq, dk, stream);
    else
      launch_any<_Float16, kBackward>(g, tensors, dim, inter, dq, dk, stream);
    return hipGetLastError();
  }
  if (p.dtype == FL_DTYPE_F32)
    launch_any<float, kForward>(g, tensors, dim, inter, nullptr, nullptr, stream);
  else if (p.dtype == FL_DTYPE_BF16)
    launch_any<__bf16, kForward>(g, tensors, dim, inter, nullptr, nullptr, stream);
  else
    launch_any<_Float16, kForward>(g, tensors, dim, inter, nullptr, nullptr, stream);
  return hipGetLastError();
}

}  // namespace fl
