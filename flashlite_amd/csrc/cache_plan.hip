// The bookkeeping of a paged cache on the GPU: blocks, slots and positions of
// a step's tokens (fl_attn_cache_plan), ancestors and positions of drafted
// tokens (fl_attn_tree_plan).
//
// Both are bound by launches and latency, not by traffic: a decode step of 32
// requests moves a few KiB (kernels of 3 and 2 us; 64 prompts of up to 4096
// tokens 6.4 us).

#include <algorithm>
#include <type_traits>

#include "fl_serve.h"

namespace fl {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// Exclusive sums of two values over the work-group, and their totals.
struct Sums {
  int before[2], total[2];
};

__device__ __forceinline__ Sums group_scan(int x, int y, int2 (&part)[kWaves]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int sx = wave_scan(x), sy = wave_scan(y);
  if (lane == 63) part[w] = make_int2(sx, sy);
  __syncthreads();
  Sums s = {{sx - x, sy - y}, {0, 0}};
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const int2 p = part[i];
    if (i < w) {
      s.before[0] += p.x;
      s.before[1] += p.y;
    }
    s.total[0] += p.x;
    s.total[1] += p.y;
  }
  return s;
}

struct PlanGeom {
  const int32_t* lengths;
  const int32_t* counts;
  int32_t* tables;
  const int32_t* held;
  int32_t* held_out;
  int32_t* ring;
  const int32_t* state;
  int32_t* state_out;
  int32_t* positions;
  int64_t* slots;
  int32_t* info;
  long long table_stride;
  int batch, width, max_blocks, pool;
  FastDiv block, by_width;
};

// Request b's blocks: what it holds, and what its length with its new tokens
// needs.
struct Want {
  int length, fresh, held;
  bool ended, wide;
  int need;
};

__device__ __forceinline__ Want want(const PlanGeom& g, int b) {
  Want r;
  r.length = max(g.lengths[b], 0);
  const int c = g.counts[b];
  r.ended = c < 0;
  r.fresh = min(max(c, 0), g.width);
  r.held = min(max(g.held[b], 0), g.max_blocks);
  // The last new token's block (past 2^31 tokens it is past the table's row).
  const uint32_t last = (uint32_t)r.length + (uint32_t)r.fresh - 1;
  const int blocks = last >> 31 ? g.max_blocks + 1 : divide((int)last, g.block) + 1;
  r.wide = r.fresh > 0 && blocks > g.max_blocks;
  r.need = r.fresh > 0 && !r.wide ? max(blocks - r.held, 0) : 0;
  return r;
}

// What a call does with one request (fl_attn_cache_plan's info), its length and
// the tokens that get slots.
struct Move {
  int status, held, moved, first, length, fresh;
};

// Index i of the ring, i < 2 pool.
__device__ __forceinline__ int wrap(const PlanGeom& g, uint32_t i) {
  return (int)(i >= (uint32_t)g.pool ? i - (uint32_t)g.pool : i);
}

// The moves of all requests, 256 at a time: put(b, move) is called for each by
// one thread; returns the ring's new head and count.  Every thread of the
// work-group takes part, and has read the state and every held count when it
// returns.
template <class F>
__device__ __forceinline__ int2 plan(const PlanGeom& g, F&& put) {
  __shared__ int2 part[2][kWaves];
  __shared__ int most;
  const uint32_t pool = (uint32_t)g.pool;
  const int count = min(max(g.state[1], 0), g.pool);
  const uint32_t head = (uint32_t)max(g.state[0], 0) % pool;
  const int tail = wrap(g, head + (uint32_t)count), room = g.pool - count;
  int needed = 0, backs = 0;
  if (threadIdx.x == 0) most = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < g.batch; b0 += kThreads) {
    const int b = b0 + threadIdx.x;
    Want r = {};
    if (b < g.batch) r = want(g, b);
    const int back = r.ended ? r.held : 0;
    // (two sets of parts: the last call's may still be read)
    const Sums s = group_scan(r.need, back, part[(b0 / kThreads) & 1]);
    const int off = needed + s.before[0], behind = backs + s.before[1];
    const bool served = !r.wide && (r.need == 0 || (long long)off + r.need <= count);
    Move m;
    m.status = r.wide ? 2 : served ? 0 : 1;
    m.held = r.held;
    m.length = r.length;
    m.fresh = served ? r.fresh : 0;
    m.moved = r.ended ? -min(back, max(room - behind, 0)) : served ? r.need : 0;
    m.first = (int)((r.ended ? (uint32_t)tail + (uint32_t)behind : head + (uint32_t)off) % pool);
    // Who takes blocks is a prefix of those in need of them.
    if (m.moved > 0) atomicMax(&most, off + m.moved);
    if (b < g.batch) put(b, m);
    needed += s.total[0];
    backs += s.total[1];
  }
  __syncthreads();
  const int taken = most;
  return make_int2(wrap(g, head + (uint32_t)taken), count - taken + min(backs, room));
}

// The held count and info of request b.
__device__ __forceinline__ void note(const PlanGeom& g, int b, const Move& m, bool ended) {
  g.held_out[b] = ended ? 0 : m.held + max(m.moved, 0);
  *reinterpret_cast<int4*>(g.info + 4LL * b) = make_int4(m.status, m.held, m.moved, m.first);
}

// Block k of request b: its table entry, or back to the ring.
__device__ __forceinline__ void move_block(const PlanGeom& g, int b, const Move& m, int k) {
  int32_t* const table = g.tables + b * g.table_stride;
  int32_t* const ring = g.ring + wrap(g, (uint32_t)m.first + (uint32_t)k);
  if (m.moved > 0)
    table[m.held + k] = *ring;
  else
    *ring = table[k];
}

// The blocks of the requests first, first + step, ..: a few by the thread that
// has the request, many by its wave.
template <class F>
__device__ __forceinline__ void move_blocks(const PlanGeom& g, int first, int step, F&& move_of) {
  constexpr int kFew = 4;
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int b0 = first; b0 < g.batch; b0 += kThreads * step) {
    const int b = b0 + threadIdx.x * step;
    Move m = {};
    if (b < g.batch) m = move_of(b);
    const int n = max(m.moved, -m.moved);
#pragma unroll 1
    for (int k = 0; k < min(n, kFew); ++k) move_block(g, b, m, k);
    uint64_t many = __builtin_amdgcn_ballot_w64(n > kFew);
#pragma unroll 1
    for (; many != 0; many &= many - 1) {
      const int l = __builtin_ctzll(many);
      const int of = __builtin_amdgcn_readlane(b, l), all = __builtin_amdgcn_readlane(n, l);
      const Move o = move_of(of);
      for (int k = kFew + lane; k < all; k += 64) move_block(g, of, o, k);
    }
  }
}

// Position and slot of new token i of request b.  (Blocks that this call takes
// are read from the ring, which it writes nowhere else.)
__device__ __forceinline__ void place(const PlanGeom& g, int b, int i, const Move& m) {
  int position = -1;
  long long slot = -1;
  if (i < m.fresh) {
    const int at = m.length + i;
    const int k = divide(at, g.block);
    const int id = k < m.held ? g.tables[b * g.table_stride + k]
                              : g.ring[wrap(g, (uint32_t)m.first + (uint32_t)(k - m.held))];
    if (id >= 0) {
      position = at;
      slot = (long long)id * g.block.d + (at - k * g.block.d);
    }
  }
  const long long o = (long long)b * g.width + i;
  g.positions[o] = position;
  g.slots[o] = slot;
}

// Up to kKept requests in one launch: every work-group finds all moves and
// keeps them in LDS, the first notes them, and the requests' blocks and the
// tokens are dealt to all.  With several work-groups the new held counts and
// ring state must not be the old ones' memory, which another may still read.
constexpr int kKept = 2048;
__global__ void __launch_bounds__(kThreads) cache_plan_kernel(const PlanGeom g) {
  __shared__ Move moves[kKept];
  const int2 state = plan(g, [&](int b, const Move& m) __attribute__((always_inline)) {
    moves[b] = m;
  });
  if (blockIdx.x == 0) {
    for (int b = threadIdx.x; b < g.batch; b += kThreads) note(g, b, moves[b], g.counts[b] < 0);
    if (threadIdx.x == 0) {
      g.state_out[0] = state.x;
      g.state_out[1] = state.y;
    }
  }
  move_blocks(g, blockIdx.x, gridDim.x,
              [&](int b) __attribute__((always_inline)) { return moves[b]; });
  const uint32_t all = (uint32_t)g.batch * (uint32_t)g.width, step = gridDim.x * kThreads;
  for (uint32_t e = blockIdx.x * kThreads + threadIdx.x; e < all; e += step) {
    const int b = divide((int)e, g.by_width);
    place(g, b, (int)e - b * g.width, moves[b]);
  }
}

// Otherwise in two: the moves by one work-group, then a work-group's threads
// each token of request blockIdx.y (the first also its blocks).  64 prompts of
// 4096 tokens 7.6 us, 5.0 in one launch; 1024 requests of 4 tokens 8.5 and 5.5.
__global__ void __launch_bounds__(kThreads) cache_plan_scan_kernel(const PlanGeom g) {
  const int2 state = plan(g, [&](int b, const Move& m) __attribute__((always_inline)) {
    note(g, b, m, g.counts[b] < 0);
  });
  if (threadIdx.x == 0) {
    g.state_out[0] = state.x;
    g.state_out[1] = state.y;
  }
}

__global__ void __launch_bounds__(kThreads) cache_plan_fill_kernel(const PlanGeom g) {
  const int b = blockIdx.y;
  const int4 info = *reinterpret_cast<const int4*>(g.info + 4LL * b);
  Move m = {info.x, info.y, info.z, info.w, max(g.lengths[b], 0), 0};
  if (m.status == 0) m.fresh = min(max(g.counts[b], 0), g.width);
  if (blockIdx.x == 0) {
    const int n = max(m.moved, -m.moved);
    for (int k = threadIdx.x; k < n; k += kThreads) move_block(g, b, m, k);
  }
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i < g.width) place(g, b, i, m);
}

// One work-group a request, a thread a draft.  seen[w][i] starts as draft i's
// own bit and up[i] as its parent; each round seen[.][i] |= seen[.][up[i]],
// up[i] = up[up[i]], after which it holds i's 2^round nearest ancestors, until
// no draft has further ones: about log2 of the tree's depth rounds.  (A round
// may already read a neighbour's new words: they only hold more of the same
// ancestors.)  Word w has bits of drafts from 64 w on only.
template <int THREADS>
__global__ void __launch_bounds__(THREADS)
tree_plan_kernel(const int32_t* parents, long long parent_stride, const int32_t* lengths,
                 const int32_t* counts, int64_t* mask, int32_t* positions, int n) {
  constexpr int kWords = THREADS / 64;
  __shared__ uint64_t seen[kWords][THREADS];
  __shared__ int up[2][THREADS];
  const int words = (n + 63) / 64;
  const int b = blockIdx.x, i = threadIdx.x;
  const int count = counts ? min(max(counts[b], 0), n) : n;
  const int length = max(lengths[b], 0);
  int u = i < n ? parents[b * parent_stride + i] : -1;
  u = u >= 0 && u < i ? u : -1;
  up[0][i] = u;
  uint64_t own[kWords];
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    own[w] = w == i >> 6 ? (uint64_t)1 << (i & 63) : 0;
    seen[w][i] = own[w];
  }
  int cur = 0;
#pragma unroll 1
  while (__syncthreads_or(u >= 0)) {
    int next = -1;
    if (u >= 0) {
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        own[w] |= seen[w][u];
        seen[w][i] = own[w];
      }
      next = up[cur][u];
    }
    cur ^= 1;
    u = next;
    up[cur][i] = u;
  }
  if (i >= n) return;
  int above = -1;
#pragma unroll
  for (int w = 0; w < kWords; ++w) above += __popcll(own[w]);
  const bool there = i < count;
  positions[(long long)b * n + i] = there ? length + above : -1;
  int64_t* const out = mask + ((long long)b * n + i) * words;
#pragma unroll
  for (int w = 0; w < kWords; ++w)
    if (w < words) out[w] = there ? (int64_t)own[w] : 0;
}

// Tokens a work-group of the one-launch form.
constexpr int kEach = 512;

}  // namespace

hipError_t launch_cache_plan(const fl_cache_plan_params& p, hipStream_t stream) {
  PlanGeom g;
  g.lengths = p.lengths;
  g.counts = p.counts;
  g.tables = p.block_tables;
  g.held = p.held;
  g.held_out = p.held_out;
  g.ring = p.free_blocks;
  g.state = p.free_state;
  g.state_out = p.free_state_out;
  g.positions = p.positions;
  g.slots = p.slots;
  g.info = p.info;
  g.table_stride = p.table_stride;
  g.batch = (int)p.batch;
  g.width = (int)p.width;
  g.max_blocks = (int)p.max_blocks;
  g.pool = (int)p.pool;
  g.block = fast_div((int)p.block_size);
  g.by_width = fast_div((int)std::max<int64_t>(1, p.width));
  const int64_t all = p.batch * p.width;
  const int64_t groups = std::max<int64_t>(1, std::min<int64_t>((all + kEach - 1) / kEach, 1024));
  const bool in_place = p.held == p.held_out || p.free_state == p.free_state_out;
  if (p.batch <= kKept && all <= INT32_MAX && (groups == 1 || !in_place)) {
    hipLaunchKernelGGL(cache_plan_kernel, dim3((unsigned)groups), dim3(kThreads), 0, stream, g);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(cache_plan_scan_kernel, dim3(1), dim3(kThreads), 0, stream, g);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const unsigned across = (unsigned)std::max<int64_t>(1, (p.width + kThreads - 1) / kThreads);
  hipLaunchKernelGGL(cache_plan_fill_kernel, dim3(across, (unsigned)p.batch), dim3(kThreads), 0,
                     stream, g);
  return hipGetLastError();
}

hipError_t launch_tree_plan(const fl_tree_plan_params& p, hipStream_t stream) {
  const int n = (int)p.drafts;
  auto go = [&](auto threads) {
    constexpr int kThreads = decltype(threads)::value;
    hipLaunchKernelGGL(tree_plan_kernel<kThreads>, dim3((unsigned)p.batch), dim3(kThreads), 0,
                       stream, p.parents, (long long)p.parent_stride, p.lengths, p.counts, p.mask,
                       p.positions, n);
  };
  if (n <= 64)
    go(std::integral_constant<int, 64>{});
  else if (n <= 256)
    go(std::integral_constant<int, 256>{});
  else
    go(std::integral_constant<int, FL_ATTN_MAX_DRAFTS>{});
  return hipGetLastError();
}

}  // namespace fl
