// C-ABI entry points of the paged-cache operators: argument checks and the
// launch.  No counterpart in the reference.

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <utility>

#include "fl_serve.h"

namespace {

using fl::set_error;

int launched(hipError_t e, const char* who) {
  if (e == hipSuccess) return FL_OK;
  return set_error(FL_ERR_LAUNCH, "%s: launch failed: %s", who, hipGetErrorString(e));
}

int null_params(const char* who) {
  return set_error(FL_ERR_INVALID_ARGUMENT, "%s: params is NULL", who);
}

bool fits32(int64_t x) { return x >= 0 && x <= INT32_MAX; }

bool aligned(const void* p, uintptr_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// Strides of an [n0, n1, n2, head_dim] view: non-negative, and rows of whole
// 16-byte pieces.  (Those of one entry step nowhere.)
int check_view(const int64_t st[3], int64_t n0, int64_t n1, int64_t n2, int64_t unit,
               const char* name, const char* who) {
  const int64_t n[3] = {n0, n1, n2};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (st[i] < 0 || st[i] % unit != 0))
      return set_error(FL_ERR_UNSUPPORTED,
                       "%s: %s strides must be non-negative multiples of %lld elements (got %lld, "
                       "%lld, %lld)", who, name, (long long)unit, (long long)st[0],
                       (long long)st[1], (long long)st[2]);
  return FL_OK;
}

// Rows of head_dim columns that are written: no two may share a place.  The
// dimensions must nest: each stride reaches past everything that the smaller
// ones span.
int check_apart(const int64_t st[3], int64_t n0, int64_t n1, int64_t n2, int64_t head_dim,
                const char* name, const char* who) {
  if (n0 == 0 || n1 == 0 || n2 == 0) return FL_OK;
  std::pair<int64_t, int64_t> dim[3] = {{st[0], n0}, {st[1], n1}, {st[2], n2}};
  std::sort(dim, dim + 3);
  __int128 span = head_dim;
  for (const auto& [stride, n] : dim) {
    if (n <= 1) continue;
    if (stride < span)
      return set_error(FL_ERR_INVALID_ARGUMENT, "%s: %s is written, its rows must not overlap", who,
                       name);
    span += (__int128)stride * (n - 1);
  }
  return FL_OK;
}

int check_pages(int64_t num_blocks, int64_t block_size, const char* who) {
  if (num_blocks < 1 || block_size < 1)
    return set_error(FL_ERR_INVALID_ARGUMENT,
                     "%s: the cache needs blocks and rows (got %lld blocks of %lld)", who,
                     (long long)num_blocks, (long long)block_size);
  if (num_blocks > INT32_MAX || block_size > INT32_MAX)
    return set_error(FL_ERR_UNSUPPORTED, "%s: num_blocks and block_size must fit in int32", who);
  return FL_OK;
}

int check_rotary(const fl_rotary_params* p, bool cache, const char* who) {
  if (p == nullptr) return null_params(who);
  if (p->dtype != FL_DTYPE_F16 && p->dtype != FL_DTYPE_BF16 &&
      (cache || p->dtype != FL_DTYPE_F32))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", who, (int)p->dtype);
  if (p->batch < 0 || p->heads < 0 || p->rows < 0 || p->kv_heads < 0 || p->pairs < 0)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: sizes must be non-negative", who);
  if (p->head_dim != 64 && p->head_dim != 128)
    return set_error(FL_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128 (got %lld)", who,
                     (long long)p->head_dim);
  if (2 * p->pairs > p->head_dim)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: %lld pairs do not fit head_dim %lld", who,
                     (long long)p->pairs, (long long)p->head_dim);
  if (p->position_bits != 32 && p->position_bits != 64)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: position_bits must be 32 or 64", who);
  if (!std::isfinite(p->scale) || !std::isfinite((float)p->scale))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: scale must be finite", who);
  if (!fits32(p->batch) || !fits32(p->rows) || p->heads > 16384 || p->kv_heads > 16384 ||
      (p->rows > 0 && p->batch > INT64_C(0x3ffffff) / p->rows))
    return set_error(FL_ERR_UNSUPPORTED, "%s: batch * rows must be below 2^26 and heads at most "
                     "16384", who);
  const int64_t unit = p->dtype == FL_DTYPE_F32 ? 4 : 8;
  auto view = [&](const int64_t st[3], int64_t heads, const char* name) {
    return check_view(st, p->batch, heads, p->rows, unit, name, who);
  };
  int rc = view(p->q_stride, p->heads, "q");
  if (rc == FL_OK) rc = view(p->q_out_stride, p->heads, "q_out");
  if (rc == FL_OK && p->k) rc = view(p->k_stride, p->kv_heads, "k");
  if (rc == FL_OK && p->k && !cache) rc = view(p->k_out_stride, p->kv_heads, "k_out");
  if (rc == FL_OK)
    rc = check_apart(p->q_out_stride, p->batch, p->heads, p->rows, p->head_dim, "q_out", who);
  if (rc == FL_OK && p->k && !cache)
    rc = check_apart(p->k_out_stride, p->batch, p->kv_heads, p->rows, p->head_dim, "k_out", who);
  return rc;
}

int check_rotary_pointers(const fl_rotary_params* p, bool cache, const char* who) {
  // (what has no heads has no memory)
  if ((p->heads > 0 && (!p->q || !p->q_out)) ||
      (!cache && p->k && p->kv_heads > 0 && !p->k_out) ||
      (p->pairs > 0 && (!p->positions || !p->freqs)))
    return set_error(FL_ERR_INVALID_ARGUMENT,
                     "%s: q, the outputs, positions and freqs must be non-NULL", who);
  if (!aligned(p->q, 16) || !aligned(p->q_out, 16) || !aligned(p->k, 16) ||
      (!cache && !aligned(p->k_out, 16)))
    return set_error(FL_ERR_MISALIGNED, "%s: q, k and the outputs must be 16-byte aligned", who);
  if (!aligned(p->freqs, 8) || !aligned(p->positions, p->position_bits / 8))
    return set_error(FL_ERR_MISALIGNED, "%s: freqs and positions must be aligned", who);
  return FL_OK;
}

int check_tree(const fl_tree_params* p, const char* who) {
  if (p == nullptr) return null_params(who);
  if (p->dtype != FL_DTYPE_F16 && p->dtype != FL_DTYPE_BF16)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", who, (int)p->dtype);
  if (p->batch < 0 || p->heads < 0 || p->kv_heads < 0 || p->drafts < 0)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: sizes must be non-negative", who);
  if (p->head_dim != 64 && p->head_dim != 128)
    return set_error(FL_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128 (got %lld)", who,
                     (long long)p->head_dim);
  if (p->heads > 0 && (p->kv_heads == 0 || p->heads % p->kv_heads != 0))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: %lld heads are not a multiple of %lld key/value "
                     "heads", who, (long long)p->heads, (long long)p->kv_heads);
  const double s = p->sm_scale == 0.0 ? 1.0 / std::sqrt((double)p->head_dim) : p->sm_scale;
  const float c = (float)(std::fabs(s) * 1.4426950408889634);
  if (!std::isfinite(s) || !std::isfinite(c) || c == 0.0f)
    return set_error(FL_ERR_INVALID_ARGUMENT,
                     "%s: sm_scale*log2(e) must be finite and non-zero (sm_scale=%g)", who, s);
  int rc = check_pages(p->num_blocks, p->block_size, who);
  if (rc != FL_OK) return rc;
  if (p->max_blocks < 1)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: the block tables need entries", who);
  // (keys are counted in 32 bits, those of lookups past the last one too)
  if (p->max_blocks > INT32_MAX / p->block_size ||
      p->max_blocks * p->block_size >= (INT64_C(1) << 31) - 65536)
    return set_error(FL_ERR_UNSUPPORTED, "%s: max_blocks * block_size must be below 2^31 - 65536",
                     who);
  if (!fits32(p->batch) || !fits32(p->heads) || !fits32(p->drafts) ||
      (p->drafts > 0 && p->heads > INT32_MAX / 2 / p->drafts))
    return set_error(FL_ERR_UNSUPPORTED, "%s: batch and heads * drafts must fit in int32", who);
  if (p->heads > 0 && p->drafts > 0) {
    const int64_t units = (p->heads / p->kv_heads * p->drafts + 31) / 32 * p->kv_heads;
    if (p->batch > (INT32_MAX / 256) / units)
      return set_error(FL_ERR_UNSUPPORTED, "%s: too many work-groups", who);
  }
  if ((p->table_stride < p->max_blocks && p->batch > 1) || p->table_stride < 0)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: table_stride %lld is below max_blocks %lld", who,
                     (long long)p->table_stride, (long long)p->max_blocks);
  if (p->mask_stride < 0)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: mask_stride must be non-negative", who);
  auto view = [&](const int64_t st[3], const char* name) {
    return check_view(st, p->batch, p->heads, p->drafts, 8, name, who);
  };
  auto cache = [&](const int64_t st[3], const char* name) {
    return check_view(st, p->num_blocks, p->kv_heads, p->block_size, 8, name, who);
  };
  rc = view(p->q_stride, "q");
  if (rc == FL_OK) rc = view(p->o_stride, "o");
  if (rc == FL_OK) rc = cache(p->k_stride, "k_cache");
  if (rc == FL_OK) rc = cache(p->v_stride, "v_cache");
  if (rc != FL_OK) return rc;
  // Rows are found by 32-bit block and row strides in bytes.
  for (int i = 0; i < 3; i += 2)
    if ((i == 0 ? p->num_blocks : p->block_size) > 1 &&
        (p->k_stride[i] > INT32_MAX || p->v_stride[i] > INT32_MAX))
      return set_error(FL_ERR_UNSUPPORTED,
                       "%s: block and row strides of the caches must be below 2^31 elements", who);
  return FL_OK;
}

bool empty_tree(const fl_tree_params* p) { return p->batch == 0 || p->heads == 0 || p->drafts == 0; }

}  // namespace

extern "C" {

int fl_attn_cache_plan(const fl_cache_plan_params* p, void* stream) {
  const char* who = "fl_attn_cache_plan";
  if (p == nullptr) return null_params(who);
  if (p->batch < 0 || p->width < 0 || p->block_size < 1 || p->max_blocks < 0 || p->pool < 1 ||
      p->table_stride < 0)
    return set_error(FL_ERR_INVALID_ARGUMENT,
                     "%s: sizes must be non-negative, block_size and pool at least 1", who);
  if (p->batch > 65535 || !fits32(p->width) || !fits32(p->pool) || !fits32(p->block_size) ||
      !fits32(p->max_blocks) || p->max_blocks > INT32_MAX / p->block_size)
    return set_error(FL_ERR_UNSUPPORTED, "%s: batch must be at most 65535, and width, pool and "
                     "max_blocks * block_size fit in int32", who);
  if (p->batch > 0 && p->max_blocks > INT32_MAX / p->batch)
    return set_error(FL_ERR_UNSUPPORTED, "%s: batch * max_blocks must fit in int32", who);
  if (p->batch > 1 && p->table_stride < p->max_blocks)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: table_stride %lld is below max_blocks %lld", who,
                     (long long)p->table_stride, (long long)p->max_blocks);
  if (!p->free_blocks || !p->free_state || !p->free_state_out)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: the free blocks' pointers must be non-NULL", who);
  if (p->batch > 0 && (!p->lengths || !p->counts || !p->held || !p->held_out || !p->info ||
                       (p->max_blocks > 0 && !p->block_tables) ||
                       (p->width > 0 && (!p->positions || !p->slots))))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: the requests' pointers must be non-NULL", who);
  // (work-groups read the old ones while others write the new)
  auto meet = [](const int32_t* x, const int32_t* y, int64_t n) {
    return x != y && (uintptr_t)x < (uintptr_t)y + 4 * n && (uintptr_t)y < (uintptr_t)x + 4 * n;
  };
  if (meet(p->held, p->held_out, p->batch) || meet(p->free_state, p->free_state_out, 2))
    return set_error(FL_ERR_INVALID_ARGUMENT,
                     "%s: held_out and free_state_out must be in place or apart", who);
  const void* const four[] = {p->lengths, p->counts, p->block_tables, p->held, p->held_out,
                              p->free_blocks, p->free_state, p->free_state_out, p->positions,
                              p->info};
  for (const void* x : four)
    if (!aligned(x, 4))
      return set_error(FL_ERR_MISALIGNED, "%s: int32 pointers must be 4-byte aligned", who);
  if (!aligned(p->slots, 8) || !aligned(p->info, 16))
    return set_error(FL_ERR_MISALIGNED, "%s: slots must be 8-byte aligned, info 16", who);
  return launched(fl::launch_cache_plan(*p, static_cast<hipStream_t>(stream)), who);
}

int fl_attn_tree_plan(const fl_tree_plan_params* p, void* stream) {
  const char* who = "fl_attn_tree_plan";
  if (p == nullptr) return null_params(who);
  if (p->batch < 0 || p->drafts < 0)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: sizes must be non-negative", who);
  if (p->drafts > FL_ATTN_MAX_DRAFTS || !fits32(p->batch) || p->batch > INT32_MAX / 256)
    return set_error(FL_ERR_UNSUPPORTED, "%s: at most %d drafts a request (got %lld)", who,
                     FL_ATTN_MAX_DRAFTS, (long long)p->drafts);
  if (p->parent_stride < 0 || (p->batch > 1 && p->parent_stride != 0 && p->parent_stride < p->drafts))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: parent_stride %lld is below drafts %lld", who,
                     (long long)p->parent_stride, (long long)p->drafts);
  if (p->batch == 0 || p->drafts == 0) return FL_OK;
  if (!p->parents || !p->lengths || !p->mask || !p->positions)
    return set_error(FL_ERR_INVALID_ARGUMENT,
                     "%s: parents, lengths, mask and positions must be non-NULL", who);
  if (!aligned(p->parents, 4) || !aligned(p->lengths, 4) || !aligned(p->counts, 4) ||
      !aligned(p->positions, 4) || !aligned(p->mask, 8))
    return set_error(FL_ERR_MISALIGNED, "%s: pointers must be aligned to their elements", who);
  return launched(fl::launch_tree_plan(*p, static_cast<hipStream_t>(stream)), who);
}

int fl_attn_rotary(const fl_rotary_params* p, void* stream) {
  const char* who = "fl_attn_rotary";
  int rc = check_rotary(p, false, who);
  if (rc != FL_OK) return rc;
  if (p->batch == 0 || p->rows == 0 || p->heads + (p->k ? p->kv_heads : 0) == 0) return FL_OK;
  rc = check_rotary_pointers(p, false, who);
  if (rc != FL_OK) return rc;
  return launched(fl::launch_rotary(*p, nullptr, static_cast<hipStream_t>(stream)), who);
}

int fl_attn_rotary_cache(const fl_rotary_params* p, const fl_cache_store* c, void* stream) {
  const char* who = "fl_attn_rotary_cache";
  int rc = check_rotary(p, true, who);
  if (rc != FL_OK) return rc;
  if (c == nullptr) return set_error(FL_ERR_INVALID_ARGUMENT, "%s: the cache is NULL", who);
  if (p->transpose)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: transpose is not for a cache", who);
  rc = check_pages(c->num_blocks, c->block_size, who);
  if (rc == FL_OK) rc = check_view(c->v_stride, p->batch, p->kv_heads, p->rows, 8, "v", who);
  auto cache = [&](const int64_t st[3], const char* name) {
    return check_view(st, c->num_blocks, p->kv_heads, c->block_size, 8, name, who);
  };
  if (rc == FL_OK) rc = cache(c->k_cache_stride, "k_cache");
  if (rc == FL_OK) rc = cache(c->v_cache_stride, "v_cache");
  if (rc == FL_OK)
    rc = check_apart(c->k_cache_stride, c->num_blocks, p->kv_heads, c->block_size, p->head_dim,
                     "k_cache", who);
  if (rc == FL_OK)
    rc = check_apart(c->v_cache_stride, c->num_blocks, p->kv_heads, c->block_size, p->head_dim,
                     "v_cache", who);
  if (rc != FL_OK) return rc;
  if (p->batch == 0 || p->rows == 0 || p->heads + p->kv_heads == 0) return FL_OK;
  if (!c->slots || (p->kv_heads > 0 && (!p->k || !c->v || !c->k_cache || !c->v_cache)))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: k, v, the caches and slots must be non-NULL", who);
  rc = check_rotary_pointers(p, true, who);
  if (rc != FL_OK) return rc;
  if (!aligned(c->v, 16) || !aligned(c->k_cache, 16) || !aligned(c->v_cache, 16) ||
      !aligned(c->slots, 8))
    return set_error(FL_ERR_MISALIGNED, "%s: v and the caches must be 16-byte aligned, slots 8", who);
  return launched(fl::launch_rotary(*p, c, static_cast<hipStream_t>(stream)), who);
}

int64_t fl_attn_tree_workspace_bytes(const fl_tree_params* p) {
  if (check_tree(p, "fl_attn_tree_workspace_bytes") != FL_OK) return -1;
  if (empty_tree(p)) return 0;
  return fl::tree_workspace_bytes(*p);
}

int fl_attn_tree_fwd(const fl_tree_params* p, void* workspace, int64_t workspace_bytes,
                     void* stream) {
  const char* who = "fl_attn_tree_fwd";
  const int rc = check_tree(p, who);
  if (rc != FL_OK) return rc;
  if (empty_tree(p)) return FL_OK;
  if (!p->q || !p->o || !p->k_cache || !p->v_cache || !p->block_tables || !p->lengths)
    return set_error(FL_ERR_INVALID_ARGUMENT,
                     "%s: q, o, the caches, block_tables and lengths must be non-NULL", who);
  if (!aligned(p->q, 16) || !aligned(p->o, 16) || !aligned(p->k_cache, 16) ||
      !aligned(p->v_cache, 16))
    return set_error(FL_ERR_MISALIGNED, "%s: q, o and the caches must be 16-byte aligned", who);
  if (!aligned(p->block_tables, 4) || !aligned(p->lengths, 4) || !aligned(p->counts, 4) ||
      !aligned(p->lse, 4) || !aligned(p->mask, 8))
    return set_error(FL_ERR_MISALIGNED,
                     "%s: block_tables, lengths, counts and lse must be 4-byte aligned, mask 8", who);
  const int apart =
      check_apart(p->o_stride, p->batch, p->heads, p->drafts, p->head_dim, "o", who);
  if (apart != FL_OK) return apart;
  const int64_t need = fl::tree_workspace_bytes(*p);
  void* const ws = need > 0 && workspace_bytes >= need ? workspace : nullptr;
  if (!aligned(ws, 16))
    return set_error(FL_ERR_MISALIGNED, "%s: workspace must be 16-byte aligned", who);
  return launched(fl::launch_tree_fwd(*p, ws, static_cast<hipStream_t>(stream)), who);
}

}  // extern "C"
