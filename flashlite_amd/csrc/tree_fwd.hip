// Attention of drafted tokens over a paged cache (fl_attn_tree_fwd), fp16 and
// bf16, head dim 64 and 128.  Shared building blocks: fa2_common.h, fa2_d128.h.
//
// The rows of one key/value head are its group of query heads times the drafts
// (row r: draft r / group, head r % group), so a cached key is read once for
// all of them.  A unit is 32 such rows of one (request, key/value head).

#include <cmath>

#include "fa2_d128.h"
#include "fl_serve.h"

namespace fl {

namespace {

struct TreeGeom {
  long long q_sb, q_sh, q_sr, o_sb, o_sh, o_sr;  // elements
  long long k_blk, k_head, k_row, v_blk, v_head, v_row;  // bytes
  const int32_t* tables;
  long long table_stride;
  const int32_t* lengths;
  const int32_t* counts;
  const int64_t* mask;
  long long mask_stride;
  float* lse;
  int batch, heads, kv_heads, group, drafts, rows, words, blocks_of_rows;
  int num_blocks, max_blocks;
  FastDiv block;
};

__device__ __forceinline__ int divide(int n, const FastDiv& f) {
  return (int)((__umulhi(f.mul, (uint32_t)n) + (uint32_t)n) >> f.shift);
}

// The first n of 64 bits.
__device__ __forceinline__ uint64_t first_bits(int n) {
  return n <= 0 ? 0 : n >= 64 ? ~(uint64_t)0 : ((uint64_t)1 << n) - 1;
}

// NaN and infinities of a V operand become 0.
template <class T>
__device__ __forceinline__ typename Elem<T>::v8 finite_only(const typename Elem<T>::v8& v) {
  constexpr uint32_t kExp = sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7C00u : 0x7F80u;
  u32x4_t x = __builtin_bit_cast(u32x4_t, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((x[i] & kExp) == kExp) x[i] &= 0xFFFF0000u;
    if ((x[i] & (kExp << 16)) == (kExp << 16)) x[i] &= 0x0000FFFFu;
  }
  return __builtin_bit_cast(typename Elem<T>::v8, x);
}

// One wave's 32 rows: Rows / Rows128 (non-causal) with scores masked by bits,
// a stabiliser that waits for a row's first visible key, and a product with V
// that hidden rows of V do not reach.
template <int D, class T>
struct TreeRows;

template <class T>
struct TreeRows<64, T> : Rows<false, true, T> {
  using Base = Rows<false, true, T>;
  using V8 = typename Base::V8;
  static constexpr int kKeys = kBc, kSteps = 4, kOps = 8;
  struct Scores {
    float16_t s[2];
  };
  struct Probs {
    V8 p[2][2];
  };
  __device__ __forceinline__ void place(int lane, float cr) {
    Base::place(lane, 0, 0, 0, 0, cr);
    this->reset();
  }
  __device__ __forceinline__ void scores(const uint8_t* kt, Scores& s) const {
    V8 ka[2][4];
    this->read_k(kt, ka);
    this->gemm1(ka, s.s);
  }
  __device__ __forceinline__ void hide(uint64_t seen, Scores& s) const {
    const uint64_t x = seen >> (4 * this->g);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint32_t word = kb ? (uint32_t)(x >> 32) : (uint32_t)x;
        s.s[kb][r] = (word >> (8 * (r >> 2) + (r & 3))) & 1 ? s.s[kb][r] : ninf();
      }
  }
  // Rows without a stabiliser take the tile's row max, if they see a key.
  __device__ __forceinline__ bool settle(bool unset, Scores& s) {
    const float mx = this->tile_max(s.s);
    const bool now = unset && mx != ninf();
    const float d = now ? mx : 0.0f;
    this->sub(s.s, d);
    this->set_m(this->m + d);
    return unset && !now;
  }
  __device__ __forceinline__ void softmax(Scores& s, Probs& p) { this->softmax_checked(s.s, p.p); }
  __device__ __forceinline__ void read_ops(const uint8_t* vt, V8 (&va)[8]) const {
#pragma unroll
    for (int u = 0; u < 8; ++u) va[u] = this->read_v_op(vt, u & 1, u >> 1);
  }
  __device__ __forceinline__ void output(const V8 (&va)[8], const Probs& p) {
#pragma unroll
    for (int u = 0; u < 8; ++u)
      this->o[u & 1] = Base::E::mfma(va[u], p.p[u >> 2][(u >> 1) & 1], this->o[u & 1]);
  }
  __device__ __forceinline__ float stabiliser() const { return this->m * this->cr; }
  __device__ __forceinline__ static int v_phys(int row, int chunk) { return chunk ^ v_swz(row); }
};

template <class T>
struct TreeRows<128, T> : Rows128<false, T> {
  using Base = Rows128<false, T>;
  using V8 = typename Base::V8;
  static constexpr int kKeys = kBc2, kSteps = 8, kOps = 8;
  struct Scores {
    float16_t s;
  };
  struct Probs {
    V8 p[2];
  };
  __device__ __forceinline__ void place(int lane, float cr) {
    Base::place(lane, 0, 0, 0, 0, cr);
  }
  __device__ __forceinline__ void scores(const uint8_t* kt, Scores& s) const {
    this->gemm1(kt, s.s);
  }
  __device__ __forceinline__ void hide(uint64_t seen, Scores& s) const {
    const uint32_t x = (uint32_t)seen >> (4 * this->g);
#pragma unroll
    for (int r = 0; r < 16; ++r)
      s.s[r] = (x >> (8 * (r >> 2) + (r & 3))) & 1 ? s.s[r] : ninf();
  }
  __device__ __forceinline__ bool settle(bool unset, Scores& s) {
    const float mx = this->tile_max(s.s);
    const bool now = unset && mx != ninf();
    if (now) this->mc = mx;
    return unset && !now;
  }
  __device__ __forceinline__ void softmax(Scores& s, Probs& p) { this->softmax_checked(s.s, p.p); }
  __device__ __forceinline__ void read_ops(const uint8_t* vt, V8 (&va)[8]) const {
#pragma unroll
    for (int u = 0; u < 8; ++u) va[u] = this->read_v_op(vt, u & 3, u >> 2);
  }
  __device__ __forceinline__ void output(const V8 (&va)[8], const Probs& p) {
#pragma unroll
    for (int u = 0; u < 8; ++u) this->o[u & 3] = Base::E::mfma(va[u], p.p[u >> 2], this->o[u & 3]);
  }
  __device__ __forceinline__ float stabiliser() const { return this->mc; }
  __device__ __forceinline__ static int v_phys(int row, int chunk) { return chunk ^ v_swz128(row); }
};

// 16 (or 4) bytes a lane from a 64-bit address of its own into LDS at
// base + 16 (4) * lane, asynchronously (vmcnt).  Inline assembly, so that the
// compiler does not guard reads of other slots with waits on it.
__device__ __forceinline__ void fetch16(uint64_t address, const void* lds) {
  const uint32_t base = (uint32_t)(uintptr_t)lds;
  asm volatile("global_load_lds_dwordx4 %0, off" : : "v"(address), "{m0}"(base) : "memory");
}
__device__ __forceinline__ void fetch4(uint64_t address, const void* lds) {
  const uint32_t base = (uint32_t)(uintptr_t)lds;
  asm volatile("global_load_lds_dword %0, off" : : "v"(address), "{m0}"(base) : "memory");
}

constexpr int kWaves = 4;

// Four waves own one unit's 32 rows; wave w walks key tiles w, w + 4, ...,
// each through a K and a V slot of its own, and the partial results meet in
// LDS.  Keys are found through the block table: lane l looks up key l of a
// tile (its table entry fetched by DMA two tiles ahead), writes the key's row
// addresses to a small table in LDS, and each 1 KiB fetch reads its lanes'
// addresses there, so pages may end anywhere in a tile.
template <int D, class T>
__global__ void __launch_bounds__(64 * kWaves, 2)
tree_fwd_kernel(const T* Q, const uint8_t* K, const uint8_t* V, T* O, const TreeGeom g, float cq,
                float cr) {
  using RowsT = TreeRows<D, T>;
  using V8 = typename RowsT::V8;
  constexpr int kKeys = RowsT::kKeys, kRowB = 2 * D;
  constexpr int kLanes = kRowB / 16;      // lanes a row of a fetch
  constexpr int kSegRows = 64 / kLanes;   // rows a fetch
  constexpr int kAcc = D / 2;
  static_assert(kKeys * kRowB == kTileBytes, "tile size");
  __shared__ __attribute__((aligned(16))) uint8_t buf[kWaves][2][kTileBytes];
  __shared__ __attribute__((aligned(16))) uint64_t where[kWaves][2][64];  // K, V row addresses
  __shared__ __attribute__((aligned(16))) int32_t ids[kWaves][2][64];
  __shared__ float2 mlbuf[kWaves][64];

  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The unit.
  const int per = g.kv_heads * g.blocks_of_rows;
  const int b = blockIdx.x / per;
  const int rest = blockIdx.x - b * per;
  const int kvh = rest / g.blocks_of_rows, rb = rest - kvh * g.blocks_of_rows;
  const int capacity = g.max_blocks * g.block.d;
  const int count = g.counts ? min(max(g.counts[b], 0), g.drafts) : g.drafts;
  const int length = min(max(g.lengths[b], 0), capacity);
  const int row0 = 32 * rb;
  if (row0 / g.group >= count) return;  // no draft of these rows is there
  int drafts = min(count, capacity - length);  // with keys
  if (g.mask == nullptr)  // a chain: the rows' last draft sees no later one
    drafts = min(drafts, (min(row0 + 32, g.rows) - 1) / g.group + 1);
  const int keys = length + drafts;
  const int tiles = (keys + kKeys - 1) / kKeys;
  const int n = tiles > w ? (tiles - w + kWaves - 1) / kWaves : 0;  // this wave's

  RowsT rows;
  rows.place(lane, cr);
  const int row = row0 + rows.col;
  const int my_row = min(row, g.rows - 1);
  const int draft = my_row / g.group;
  const int head = kvh * g.group + (my_row - draft * g.group);
  const bool mine = row < g.rows && draft < count;
  {
    const T* q = Q + (b * g.q_sb + head * g.q_sh + draft * g.q_sr) + 8 * rows.g;
    const uint32_t sign = cq < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int st = 0; st < RowsT::kSteps; ++st) {
      const u32x4_t raw = *reinterpret_cast<const u32x4_t*>(q + 16 * st);
      rows.qf[st] = __builtin_bit_cast(V8, raw ^ (u32x4_t){sign, sign, sign, sign});
    }
#pragma unroll
    for (int st = 0; st < RowsT::kSteps; ++st) asm volatile("" : "+v"(rows.qf[st]));
  }
  const int64_t* const mask =
      g.mask ? g.mask + b * g.mask_stride + (long long)draft * g.words : nullptr;
  // This lane's row's visible keys of tile [k0, k0 + 64) behind the prefix.
  auto seen_bits = [&](int k0) __attribute__((always_inline)) {
    const int d0 = k0 - length;  // the tile's first draft
    const int from = max(d0, 0);
    uint64_t x = first_bits(drafts - from);
    if (mask == nullptr) {
      x &= first_bits(draft + 1 - from);
    } else {
      const int w0 = from >> 6, sh = from & 63;
      uint64_t m = w0 < g.words ? (uint64_t)mask[w0] >> sh : 0;
      if (sh != 0 && w0 + 1 < g.words) m |= (uint64_t)mask[w0 + 1] << (64 - sh);
      x &= m;
    }
    return d0 >= 0 ? x : (d0 > -64 ? x << -d0 : 0) | first_bits(-d0);
  };

  const uint64_t table = (uint64_t)(uintptr_t)(g.tables + b * g.table_stride);
  const uint64_t kbase = (uint64_t)(uintptr_t)(K + kvh * g.k_head);
  const uint64_t vbase = (uint64_t)(uintptr_t)(V + kvh * g.v_head);
  // Key l of this wave's tile i (past the last: the last again).
  auto key_of = [&](int i) __attribute__((always_inline)) {
    return min((w + kWaves * i) * kKeys + (lane & (kKeys - 1)), keys - 1);
  };
  auto fetch_ids = [&](int i) __attribute__((always_inline)) {
    fetch4(table + 4 * (uint64_t)divide(key_of(i), g.block), ids[w][i & 1]);
  };
  // Row addresses of tile i; the result has a bit per key with a block.
  auto locate = [&](int i) __attribute__((always_inline)) {
    const int key = key_of(i);
    const int in = key - divide(key, g.block) * g.block.d;
    int id = ids[w][i & 1][lane];
    const bool ok = (uint32_t)id < (uint32_t)g.num_blocks;
    id = ok ? id : 0;
    where[w][0][lane] = kbase + (id * g.k_blk + in * g.k_row);
    where[w][1][lane] = vbase + (id * g.v_blk + in * g.v_row);
    return __builtin_amdgcn_ballot_w64(ok);
  };
  auto fetch = [&](int t) __attribute__((always_inline)) {  // 0: K, 1: V
#pragma unroll
    for (int seg = 0; seg < 8; ++seg) {
      const int r = kSegRows * seg + lane / kLanes;
      const int phys = lane & (kLanes - 1);
      const int chunk = phys ^ (D == 64 ? (t ? v_swz(r) : k_swz(r))
                                        : (t ? v_swz128(r) : k_swz128(r)));
      fetch16(where[w][t][r] + 16 * chunk, buf[w][t] + 1024 * seg);
    }
  };

  uint64_t ok = 0;
  if (n > 0) {
    fetch_ids(0);
    fetch_ids(1);
    asm volatile("s_waitcnt vmcnt(1)" : : : "memory");
    ok = locate(0);
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    fetch(0);
    fetch(1);
  }
  bool unset = true;
  for (int i = 0; i < n; ++i) {
    typename RowsT::Scores s;
    typename RowsT::Probs p;
    asm volatile("s_waitcnt vmcnt(8)" : : : "memory");  // K(i), and the ids of i + 1
    rows.scores(buf[w][0], s);
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // its operands are in registers
    const bool more = i + 1 < n;
    uint64_t ok_next = 0;
    if (more) {
      ok_next = locate(i + 1);
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      fetch_ids(i + 2);
      fetch(0);
    }
    const int k0 = (w + kWaves * i) * kKeys;
    const bool checked = k0 + kKeys > length || ~ok != 0;
    uint64_t seen = ~(uint64_t)0;
    if (checked) {
      seen = seen_bits(k0) & ok;
      rows.hide(seen, s);
    }
    if (__builtin_amdgcn_ballot_w64(unset) != 0) unset = rows.settle(unset, s);
    rows.softmax(s, p);
    if (more)
      asm volatile("s_waitcnt vmcnt(9)" : : : "memory");  // V(i)
    else
      asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    V8 va[8];
    rows.read_ops(buf[w][1], va);
    if (checked) {
      // What p = 0 meets must be finite; a visible NaN or infinity is added
      // to the rows that see it.
      bool odd = false;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const V8 f = finite_only<T>(va[u]);
        const u32x4_t x = __builtin_bit_cast(u32x4_t, f) ^ __builtin_bit_cast(u32x4_t, va[u]);
        odd |= (x[0] | x[1] | x[2] | x[3]) != 0;
        va[u] = f;
      }
      if (__builtin_amdgcn_ballot_w64(odd) != 0) {
#pragma unroll 1
        for (int j = 0; j < kKeys; ++j) {
          const bool sees = (seen >> j) & 1;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const int chunk = RowsT::v_phys(j, 2 * c + rows.g);
            const V8 x = *reinterpret_cast<const V8*>(buf[w][1] + j * kRowB + 16 * chunk);
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
    rows.output(va, p);
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    if (more) fetch(1);
    ok = ok_next;
  }
  // Nothing may still write this wave's slots: its O goes there.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
  float4* const mine4 = reinterpret_cast<float4*>(buf[w][0]);
#pragma unroll
  for (int c = 0; c < kAcc / 4; ++c) {
    const float16_t& x = rows.o[c >> 2];
    const int r = 4 * (c & 3);
    mine4[c * 64 + lane] = make_float4(x[r], x[r + 1], x[r + 2], x[r + 3]);
  }
  mlbuf[w][lane] = make_float2(rows.stabiliser(), rows.l);
  __syncthreads();
  // Partial results meet at their largest stabiliser; one without a visible
  // key (l = 0 across the lane pair) is passed over.
  float mm = ninf(), lt = 0.0f, a[kWaves];
  float2 ml[kWaves];
  bool has[kWaves];
#pragma unroll
  for (int j = 0; j < kWaves; ++j) {
    ml[j] = mlbuf[j][lane];
    has[j] = pair_sum(ml[j].y) != 0.0f;
    if (has[j]) mm = fmaxf(mm, ml[j].x);
  }
#pragma unroll
  for (int j = 0; j < kWaves; ++j) {
    a[j] = has[j] ? __builtin_amdgcn_exp2f(ml[j].x - mm) : 0.0f;
    lt += a[j] * ml[j].y;
  }
  const float l_tot = pair_sum(lt);
  const float inv = l_tot == 0.0f ? 0.0f : 1.0f / l_tot;
  T* const orow = O + (b * g.o_sb + head * g.o_sh + draft * g.o_sr);
  for (int c = w; c < D / 16; c += kWaves) {
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < kWaves; ++j) {
      const float4* const pj = reinterpret_cast<const float4*>(buf[j][0]);
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
    if (!mine) continue;
    V8 out;
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = (T)(acc[e] * inv);
    *reinterpret_cast<V8*>(orow + 32 * (c >> 1) + 16 * (c & 1) + 8 * rows.g) = out;
  }
  if (w == 0 && rows.g == 0 && mine && g.lse != nullptr)
    g.lse[((long long)b * g.heads + head) * g.drafts + draft] =
        l_tot == 0.0f ? ninf() : 0.693147180559945309f * (mm + __builtin_amdgcn_logf(l_tot));
}

template <int D, class T>
hipError_t launch_t(const fl_tree_params& p, const TreeGeom& g, float cq, float cr, hipStream_t st) {
  const unsigned units = (unsigned)(g.batch * g.kv_heads * g.blocks_of_rows);
  hipLaunchKernelGGL((tree_fwd_kernel<D, T>), dim3(units), dim3(64 * kWaves), 0, st,
                     static_cast<const T*>(p.q), static_cast<const uint8_t*>(p.k_cache),
                     static_cast<const uint8_t*>(p.v_cache), static_cast<T*>(p.o), g, cq, cr);
  return hipGetLastError();
}

}  // namespace

int64_t tree_workspace_bytes(const fl_tree_params&) { return 0; }

hipError_t launch_tree_fwd(const fl_tree_params& p, void*, hipStream_t st) {
  TreeGeom g = {};
  g.q_sb = p.q_stride[0];
  g.q_sh = p.q_stride[1];
  g.q_sr = p.q_stride[2];
  g.o_sb = p.o_stride[0];
  g.o_sh = p.o_stride[1];
  g.o_sr = p.o_stride[2];
  g.k_blk = 2 * p.k_stride[0];
  g.k_head = 2 * p.k_stride[1];
  g.k_row = 2 * p.k_stride[2];
  g.v_blk = 2 * p.v_stride[0];
  g.v_head = 2 * p.v_stride[1];
  g.v_row = 2 * p.v_stride[2];
  g.tables = p.block_tables;
  g.table_stride = p.table_stride;
  g.lengths = p.lengths;
  g.counts = p.counts;
  g.mask = p.mask;
  g.mask_stride = p.mask_stride;
  g.lse = p.lse;
  g.batch = (int)p.batch;
  g.heads = (int)p.heads;
  g.kv_heads = (int)p.kv_heads;
  g.group = (int)(p.heads / p.kv_heads);
  g.drafts = (int)p.drafts;
  g.rows = g.group * g.drafts;
  g.words = (g.drafts + 63) / 64;
  g.blocks_of_rows = (g.rows + 31) / 32;
  g.num_blocks = (int)p.num_blocks;
  g.max_blocks = (int)p.max_blocks;
  g.block = fast_div((int)p.block_size);
  const double s = p.sm_scale == 0.0 ? (double)(1.0f / std::sqrt((float)p.head_dim)) : p.sm_scale;
  const float cr = (float)(std::fabs(s) * 1.44269504088896340736), cq = s < 0.0 ? -1.0f : 1.0f;
  const bool bf = p.dtype == FL_DTYPE_BF16;
  if (p.head_dim == 128)
    return bf ? launch_t<128, __bf16>(p, g, cq, cr, st) : launch_t<128, _Float16>(p, g, cq, cr, st);
  return bf ? launch_t<64, __bf16>(p, g, cq, cr, st) : launch_t<64, _Float16>(p, g, cq, cr, st);
}

}  // namespace fl
