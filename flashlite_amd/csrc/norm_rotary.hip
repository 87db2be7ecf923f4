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
// row and dy).  As in rotary.hip a thread owns V pairs of one token and walks a
// few heads with their sines and cosines in registers; the D / 2V threads of a
// row, neighbours in a wave, add up its sums across lanes in 32 bits, and each
// value is rounded once, at the end.  dw is summed in a work-group's registers
// and LDS, then over the work-groups by a second kernel in a fixed order: no
// atomics, the same bits every time.

#include <algorithm>
#include <type_traits>

#include "fl_serve.h"

namespace fl {

namespace {

constexpr int kLeastBlocks = 256;  // work-groups that a launch should have (rotary.hip)
constexpr int kAcross = 4, kAcrossLanes = 32;

enum { kForward, kStore, kBackward };

struct NormRows {
  const void* in;   // x; backward: dy
  const void* x;    // backward: x
  void* out;        // y, a cache, or dx
  const void* weight;  // null: neither normed nor scaled
  long long in_st[3], x_st[3];
  long long out_st[3];  // {batch, head, row}, or {block, head, row} of a cache
  int heads, per, across_log2, head_blocks, items;  // items: work-groups' worth
  int copy, paged;
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
  float* part;  // backward: [q, k][gridDim.x][D]
  int pos64, pairs, weight32;
  uint32_t tokens;  // batch * rows
  float scale, sign, eps, offset;
  double scale64;
  FastDiv by_rows, block;
};

template <class T, int N>
__device__ __forceinline__ void load(const T* p, T (&x)[N]) {
  __builtin_memcpy(x, __builtin_assume_aligned(p, sizeof(T) * N), sizeof(T) * N);
}
template <class T, int N>
__device__ __forceinline__ void store(T* p, const T (&x)[N]) {
  __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T) * N), x, sizeof(T) * N);
}

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

// A thread's columns: V at c0 and V at c1 (as in rotary_kernel).  blockIdx.y:
// q, k (or v).  UNROLL heads' loads in flight.
template <class T, int D, bool INTER, int V, int MODE, int UNROLL>
__global__ void __launch_bounds__(256) norm_rotary_kernel(const NormGeom g) {
  constexpr uint32_t kThreads = D / (2 * V);  // a row
  constexpr bool kBack = MODE == kBackward;
  const NormRows& n = g.rows[blockIdx.y];
  const int j = (int)(threadIdx.x % kThreads);
  const bool turns = j * V < g.pairs && !(MODE == kStore && n.copy);
  constexpr bool kHalves = !INTER || V > 1;
  const bool paired = j * V < g.pairs;
  const int rest = D - 2 * g.pairs;
  const int c0 = paired ? (kHalves ? j * V : 2 * j) : g.pairs + j * V;
  const int c1 = paired ? (kHalves ? g.pairs + j * V : 2 * j + 1) : c0 + rest / 2;
  const bool norm = n.weight != nullptr;
  float w0[V], w1[V];
#pragma unroll
  for (int e = 0; e < V; ++e) w0[e] = w1[e] = 1.0f;
  if (norm) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (g.weight32) {
        w0[e] = static_cast<const float*>(n.weight)[c0 + e] + g.offset;
        w1[e] = static_cast<const float*>(n.weight)[c1 + e] + g.offset;
      } else {
        w0[e] = (float)static_cast<const T*>(n.weight)[c0 + e] + g.offset;
        w1[e] = (float)static_cast<const T*>(n.weight)[c1 + e] + g.offset;
      }
    }
  }
  float s0[V], s1[V];  // dw
#pragma unroll
  for (int e = 0; e < V; ++e) s0[e] = s1[e] = 0.0f;

  const int across = 1 << n.across_log2;
  auto walk = [&](int item) __attribute__((always_inline)) {
    const int tx = item / n.head_blocks, hb = item - tx * n.head_blocks;
    const uint32_t x = (uint32_t)tx * 256 + threadIdx.x;
    const uint32_t token = x / kThreads >> n.across_log2;
    if (token >= g.tokens) return;
    const int b = divide((int)token, g.by_rows);
    const int i = (int)token - b * g.by_rows.d;
    long long blk = b, row = i;  // where the rows go
    if constexpr (MODE == kStore) {
      const long long slot = g.slots[b * g.slot_sb + i * g.slot_sr];
      if (slot < 0 || slot >= g.num_slots) return;
      if (n.paged) {
        blk = ((uint64_t)slot >> 31) == 0 ? divide((int)slot, g.block) : slot / g.block.d;
        row = slot - blk * g.block.d;
      }
    }
    const long long in = b * n.in_st[0] + i * n.in_st[2];
    const long long xin = kBack ? b * n.x_st[0] + i * n.x_st[2] : 0;
    const long long to = blk * n.out_st[0] + row * n.out_st[2];
    const int span = n.per << n.across_log2;
    int h = hb * span + (int)(x / kThreads & (uint32_t)(across - 1));
    const int h1 = min((hb + 1) * span, n.heads);
    if (h >= h1) return;
    T y0[UNROLL][V], y1[UNROLL][V], x0[UNROLL][V], x1[UNROLL][V];  // (x: backward)
    auto fetch = [&]() __attribute__((always_inline)) {  // (past h1: the first again)
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int hu = h + u * across, hh = hu < h1 ? hu : h;
        const T* const from = static_cast<const T*>(n.in) + (in + hh * n.in_st[1]);
        load<T, V>(from + c0, y0[u]);
        load<T, V>(from + c1, y1[u]);
        if constexpr (kBack) {
          if (norm) {
            const T* const rows = static_cast<const T*>(n.x) + (xin + hh * n.x_st[1]);
            load<T, V>(rows + c0, x0[u]);
            load<T, V>(rows + c1, x1[u]);
          }
        }
      }
    };
    fetch();
    float cs[V], sn[V];
    if (turns) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int pair = !INTER ? j * V + e
                         : V == 1 ? j
                                  : (e < V / 2 ? c0 / 2 + e : c1 / 2 + e - V / 2);
        long long at = b * g.pos_sb + i * g.pos_sr;
        if (g.axes != nullptr) at += min(max(g.axes[pair], 0), g.num_axes - 1) * g.pos_sa;
        const double position = g.pos64 ? (double)static_cast<const int64_t*>(g.positions)[at]
                                        : (double)static_cast<const int32_t*>(g.positions)[at];
        // Turns in 64 bits, reduced to [-1/2, 1/2]; 16-bit rows take the
        // hardware's sine and cosine of them in 32 bits, 32-bit rows round the
        // scaled ones once from 64 bits (rotary.hip).
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
    auto turn = [&](float (&a)[V], float (&c)[V]) __attribute__((always_inline)) {
      if (!turns) return;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float* const p = INTER && V > 1 ? (e < V / 2 ? &a[2 * e] : &c[2 * e - V]) : &a[e];
        float* const q = INTER && V > 1 ? p + 1 : &c[e];
        const float u = *p, v = *q;
        *p = u * cs[e] - v * sn[e];
        *q = u * sn[e] + v * cs[e];
      }
    };
    for (;;) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int hu = h + u * across;
        float a[V], c[V];
        if (MODE != kStore || !n.copy) {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            a[e] = (float)y0[u][e];
            c[e] = (float)y1[u][e];
          }
          if constexpr (!kBack) {
            if (norm) {
              float ss = 0.0f;
#pragma unroll
              for (int e = 0; e < V; ++e) ss += a[e] * a[e] + c[e] * c[e];
              ss = group_sum<kThreads>(ss);
              const float r = __builtin_amdgcn_rsqf(ss * (1.0f / D) + g.eps);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                a[e] *= r * w0[e];
                c[e] *= r * w1[e];
              }
            }
            turn(a, c);
          } else {
            turn(a, c);  // g
            if (norm) {
              float p[V], q[V], ss = 0.0f, dot = 0.0f;
#pragma unroll
              for (int e = 0; e < V; ++e) {
                p[e] = (float)x0[u][e];
                q[e] = (float)x1[u][e];
                ss += p[e] * p[e] + q[e] * q[e];
                dot += a[e] * w0[e] * p[e] + c[e] * w1[e] * q[e];
              }
              ss = group_sum<kThreads>(ss);
              dot = group_sum<kThreads>(dot);
              const float r = __builtin_amdgcn_rsqf(ss * (1.0f / D) + g.eps);
              const float along = dot * (1.0f / D) * r * r;
#pragma unroll
              for (int e = 0; e < V; ++e) {
                if (hu < h1) {
                  s0[e] += a[e] * (p[e] * r);
                  s1[e] += c[e] * (q[e] * r);
                }
                a[e] = r * (a[e] * w0[e] - p[e] * along);
                c[e] = r * (c[e] * w1[e] - q[e] * along);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < V; ++e) {
            y0[u][e] = (T)a[e];
            y1[u][e] = (T)c[e];
          }
        }
        if (hu < h1) {
          T* const out = static_cast<T*>(n.out) + (to + hu * n.out_st[1]);
          store<T, V>(out + c0, y0[u]);
          store<T, V>(out + c1, y1[u]);
        }
      }
      h += UNROLL * across;
      if (h >= h1) return;
      fetch();
    }
  };
  for (int item = blockIdx.x; item < n.items; item += gridDim.x) walk(item);
  if constexpr (kBack) {
    if (!norm || (int)blockIdx.x >= n.items) return;
    __shared__ float sums[4][D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = stride_sum<kThreads>(s0[e]), c = stride_sum<kThreads>(s1[e]);
      if (lane < (int)kThreads) {
        sums[wave][c0 + e] = a;
        sums[wave][c1 + e] = c;
      }
    }
    __syncthreads();
    if (threadIdx.x < D) {
      const float x = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) +
                      (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
      g.part[((long long)blockIdx.y * gridDim.x + blockIdx.x) * D + threadIdx.x] = x;
    }
  }
}

// Sums `count` rows of D partial sums: a work-group 16 columns of q's or k's
// (blockIdx.y), 64 threads a column.
__global__ void __launch_bounds__(1024) norm_weight_kernel(const float* part, int rows, int count_q,
                                                           int count_k, int D, float* q, float* k) {
  __shared__ float sums[64][16];
  float* const out = blockIdx.y == 0 ? q : k;
  if (out == nullptr) return;
  const int count = blockIdx.y == 0 ? count_q : count_k;
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
  const float* const from = part + (long long)blockIdx.y * rows * D + c;
  float x = 0.0f;
#pragma unroll 8
  for (int i = r; i < count; i += 64) x += from[(long long)i * D];
  sums[r][threadIdx.x & 15] = x;
  __syncthreads();
  for (int d = 32; d > 0; d >>= 1) {
    if (r < d) sums[r][threadIdx.x & 15] += sums[r + d][threadIdx.x & 15];
    __syncthreads();
  }
  if (r == 0) out[c] = sums[0][threadIdx.x];
}

// How a tensor's heads are dealt (as rotary.hip's launch): neighbouring threads
// first to the next of up to kAcross heads where heads lie closer together than
// rows, and as many heads a thread as leave kLeastBlocks work-groups, at most
// `most`.
void deal(NormRows& n, const long long* st, int threads, uint32_t tokens, int most) {
  n.across_log2 = 0;
  if (st[1] < st[2])
    while (1 << n.across_log2 < kAcross && 2 << n.across_log2 <= n.heads &&
           threads << (n.across_log2 + 1) <= kAcrossLanes &&
           ((int64_t)tokens * threads << (n.across_log2 + 1)) < (INT64_C(1) << 32) - 256)
      ++n.across_log2;  // (threads are counted in 32 bits)
  const int64_t blocks = (((int64_t)tokens << n.across_log2) * threads + 255) / 256;
  const int each = (n.heads + (1 << n.across_log2) - 1) >> n.across_log2;
  n.per = most;
  while (n.per > 1 && blocks * ((each + n.per - 1) / n.per) < kLeastBlocks) n.per /= 2;
  n.head_blocks = std::max(1, (each + n.per - 1) / n.per);
  n.items = n.heads > 0 ? (int)(blocks * n.head_blocks) : 0;
}

constexpr int kBackGroups = 1024;  // work-groups of a gradient's launch, a tensor

template <class T, int D, int V, int MODE, int UNROLL>
void launch_unroll(const NormGeom& g, bool inter, dim3 grid, hipStream_t st) {
  if (inter)
    hipLaunchKernelGGL((norm_rotary_kernel<T, D, true, V, MODE, UNROLL>), grid, dim3(256), 0, st, g);
  else
    hipLaunchKernelGGL((norm_rotary_kernel<T, D, false, V, MODE, UNROLL>), grid, dim3(256), 0, st,
                       g);
}

template <class T, int D, int V, int MODE>
void launch(NormGeom& g, int tensors, bool inter, float* dq, float* dk, hipStream_t st) {
  int most = 1, per = 1;
  for (int i = 0; i < tensors; ++i) {
    NormRows& n = g.rows[i];
    deal(n, n.in_st, D / (2 * V), g.tokens, MODE == kBackward ? 4 : 8);
    most = std::max(most, n.items);
    per = std::max(per, n.per);
  }
  if (MODE == kBackward) most = std::min(most, kBackGroups);
  const dim3 grid((unsigned)most, (unsigned)tensors);
  constexpr int kUnroll = MODE == kBackward ? 2 : 4;
  if (per >= kUnroll)
    launch_unroll<T, D, V, MODE, kUnroll>(g, inter, grid, st);
  else
    launch_unroll<T, D, V, MODE, 1>(g, inter, grid, st);
  if (MODE == kBackward && (dq || dk))
    hipLaunchKernelGGL(norm_weight_kernel, dim3(D / 16, 2), dim3(1024), 0, st, g.part, most,
                       std::min(most, g.rows[0].items), std::min(most, g.rows[1].items), D, dq, dk);
}

template <class T, int D, int MODE>
void launch_dim(NormGeom& g, int tensors, bool inter, float* dq, float* dk, hipStream_t st) {
  constexpr int kMost = 16 / (int)sizeof(T);
  int v = kMost;  // columns a load: 16 bytes where the pairs divide
  while (g.pairs % v != 0) v /= 2;
  if (v == 8) {
    if constexpr (kMost == 8) launch<T, D, 8, MODE>(g, tensors, inter, dq, dk, st);
  } else if (v == 4) {
    launch<T, D, 4, MODE>(g, tensors, inter, dq, dk, st);
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
                     nullptr, 0, 0, 0, (int)p.head_dim, dq, dk);
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
    v.copy = 1;
    strides(v.in_st, c->v_stride);
    strides(v.out_st, c->v_cache_stride);
    k.paged = v.paged = 1;
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
  const int tensors = k.heads > 0 ? 2 : 1;
  if (d != nullptr) {
    q.x = d->q;
    strides(q.x_st, d->q_stride);
    k.x = d->k;
    strides(k.x_st, d->k_stride);
    g.part = static_cast<float*>(ws);
    float *dq = q.weight ? d->dq_weight : nullptr, *dk = k.weight ? d->dk_weight : nullptr;
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
