// The bookkeeping of a paged cache on the GPU: blocks, slots and positions of
// a step's tokens (fl_attn_cache_plan), ancestors and positions of drafted
// tokens (fl_attn_tree_plan).
//
// Both are bound by launches and latency, not by traffic: a decode step of 32
// requests moves a few KiB.

#include <algorithm>

#include "fl_serve.h"

namespace fl {

namespace {

// Sum over the lanes below (exclusive) within the work-group; `total` gets the
// whole sum.  `part` holds a value per wave.
template <int kWaves>
__device__ __forceinline__ long long group_scan(long long x, long long* part, long long& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  long long s = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const long long y = __shfl_up(s, d);
    if (lane >= d) s += y;
  }
  if (lane == 63) part[w] = s;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const long long y = part[i];
    if (i < w) before += y;
    total += y;
  }
  __syncthreads();
  return before + s - x;
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
  FastDiv block;
};

__device__ __forceinline__ int divide(int n, const FastDiv& f) {
  return (int)((__umulhi(f.mul, (uint32_t)n) + (uint32_t)n) >> f.shift);
}

// Request b's blocks: what it holds, and what its length with its new tokens
// needs (64-bit: a length near 2^31 with `width` more).
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
  const long long blocks =
      ((long long)r.length + r.fresh + g.block.d - 1) / (long long)g.block.d;
  r.wide = r.fresh > 0 && blocks > g.max_blocks;
  r.need = r.fresh > 0 && !r.wide ? max((int)(blocks - r.held), 0) : 0;
  return r;
}

constexpr int kScanThreads = 1024;

// One work-group: prefix sums of the blocks needed and given back over the
// requests, 1024 at a time.
__global__ void __launch_bounds__(kScanThreads) cache_plan_scan_kernel(const PlanGeom g) {
  constexpr int kWaves = kScanThreads / 64;
  __shared__ long long part[kWaves];
  const int count = min(max(g.state[1], 0), g.pool);
  const int head = (int)((unsigned)max(g.state[0], 0) % (unsigned)g.pool);
  long long before = 0, back_before = 0, taken_sum = 0, given_sum = 0;
  for (int b0 = 0; b0 < g.batch; b0 += kScanThreads) {
    const int b = b0 + threadIdx.x;
    Want r = {};
    if (b < g.batch) r = want(g, b);
    const int back = r.ended ? r.held : 0;
    long long sum_need, sum_back, sum_taken, sum_given;
    const long long off = before + group_scan<kWaves>(r.need, part, sum_need);
    const long long roff = back_before + group_scan<kWaves>(back, part, sum_back);
    const bool served = !r.wide && (r.need == 0 || off + r.need <= count);
    const int taken = served ? r.need : 0;
    const long long room = (long long)g.pool - count - roff;
    const int given = (int)min((long long)back, max(room, 0LL));
    group_scan<kWaves>(taken, part, sum_taken);
    group_scan<kWaves>(given, part, sum_given);
    if (b < g.batch) {
      g.held_out[b] = r.ended ? 0 : r.held + taken;
      int32_t* const info = g.info + 4LL * b;
      info[0] = r.wide ? 2 : served ? 0 : 1;
      info[1] = r.held;
      info[2] = taken - given;
      info[3] = (int)((head + (r.ended ? count + roff : off)) % g.pool);
    }
    before += sum_need;
    back_before += sum_back;
    taken_sum += sum_taken;
    given_sum += sum_given;
  }
  __syncthreads();  // every thread has read the state
  if (threadIdx.x == 0) {
    g.state_out[0] = (int)((head + taken_sum) % g.pool);
    g.state_out[1] = (int)(count - taken_sum + given_sum);
  }
}

// Request blockIdx.y: its taken blocks' table entries, or its blocks put back
// on the ring (the first work-group), and its share of positions and slots.
__global__ void __launch_bounds__(256) cache_plan_fill_kernel(const PlanGeom g) {
  const int b = blockIdx.y;
  const int32_t* const info = g.info + 4LL * b;
  const int status = info[0], held = info[1], moved = info[2], first = info[3];
  int32_t* const table = g.tables + b * g.table_stride;
  if (blockIdx.x == 0) {
    for (int k = threadIdx.x; k < moved; k += 256)
      table[held + k] = g.ring[((long long)first + k) % g.pool];
    for (int k = threadIdx.x; k < -moved; k += 256)
      g.ring[((long long)first + k) % g.pool] = table[k];
  }
  const int length = max(g.lengths[b], 0);
  const int fresh = status == 0 ? min(max(g.counts[b], 0), g.width) : 0;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= g.width) return;
  int position = -1;
  long long slot = -1;
  if (i < fresh) {
    const int at = length + i;
    const int k = divide(at, g.block);
    const int id = k < held ? table[k] : g.ring[((long long)first + (k - held)) % g.pool];
    if (id >= 0) {
      position = at;
      slot = (long long)id * g.block.d + (at - k * g.block.d);
    }
  }
  const long long o = (long long)b * g.width + i;
  g.positions[o] = position;
  g.slots[o] = slot;
}

// One work-group a request.  seen[i] starts as draft i's own bit and up[i] as
// its parent; each round seen[i] |= seen[up[i]], up[i] = up[up[i]], after
// which seen[i] holds i's 2^round nearest ancestors.  (A round may already
// read a neighbour's new words: they only hold more of the same ancestors.)
__global__ void __launch_bounds__(256)
tree_plan_kernel(const int32_t* parents, long long parent_stride, const int32_t* lengths,
                 const int32_t* counts, int64_t* mask, int32_t* positions, int n) {
  extern __shared__ uint64_t seen[];  // [n][words], then up[2][n]
  const int words = (n + 63) / 64;
  int* const up0 = reinterpret_cast<int*>(seen + n * words);
  const int b = blockIdx.x;
  const int count = counts ? min(max(counts[b], 0), n) : n;
  for (int i = threadIdx.x; i < n; i += 256) {
    const int p = parents[b * parent_stride + i];
    up0[i] = p >= 0 && p < i ? p : -1;
  }
  for (int x = threadIdx.x; x < n * words; x += 256) {
    const int i = x / words, w = x - i * words;
    seen[x] = i >> 6 == w ? (uint64_t)1 << (i & 63) : 0;
  }
  __syncthreads();
  int cur = 0;
  for (int reach = 1; reach < n; reach <<= 1) {
    const int* const up = up0 + cur * n;
    int* const next = up0 + (cur ^ 1) * n;
    for (int x = threadIdx.x; x < n * words; x += 256) {
      const int i = x / words;
      const int u = up[i];
      if (u >= 0) seen[x] |= seen[u * words + (x - i * words)];
    }
    for (int i = threadIdx.x; i < n; i += 256) next[i] = up[i] >= 0 ? up[up[i]] : -1;
    cur ^= 1;
    __syncthreads();
  }
  const int length = max(lengths[b], 0);
  for (int i = threadIdx.x; i < n; i += 256) {
    int above = -1;
    for (int w = 0; w < words; ++w) above += __popcll(seen[i * words + w]);
    positions[(long long)b * n + i] = i < count ? length + above : -1;
  }
  for (int x = threadIdx.x; x < n * words; x += 256)
    mask[(long long)b * n * words + x] = x / words < count ? (int64_t)seen[x] : 0;
}

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
  hipLaunchKernelGGL(cache_plan_scan_kernel, dim3(1), dim3(kScanThreads), 0, stream, g);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.batch == 0) return e;
  const unsigned across = (unsigned)std::max<int64_t>(1, (p.width + 255) / 256);
  hipLaunchKernelGGL(cache_plan_fill_kernel, dim3(across, (unsigned)p.batch), dim3(256), 0, stream,
                     g);
  return hipGetLastError();
}

hipError_t launch_tree_plan(const fl_tree_plan_params& p, hipStream_t stream) {
  const int n = (int)p.drafts, words = (n + 63) / 64;
  const size_t lds = (size_t)n * words * 8 + 2 * (size_t)n * 4;
  hipLaunchKernelGGL(tree_plan_kernel, dim3((unsigned)p.batch), dim3(256), lds, stream, p.parents,
                     (long long)p.parent_stride, p.lengths, p.counts, p.mask, p.positions, n);
  return hipGetLastError();
}

}  // namespace fl
