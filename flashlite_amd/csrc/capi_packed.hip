// C-ABI entry points of attention over packed sequences: argument checks and
// the launch.  No counterpart in the reference.

#include <cmath>

#include "capi_checks.h"

namespace {

constexpr int64_t kMostRows = INT64_C(1) << 30;
constexpr int64_t kMostStride = INT64_C(1) << 24;

// A [heads, rows, head_dim] view with rows at least `least` elements apart.
int check_rows(const int64_t st[2], int64_t heads, int64_t rows, int64_t least, const char* name,
               const char* who) {
  const int64_t all[3] = {0, st[0], st[1]};
  const int rc = check_view(all, 1, heads, rows, 8, name, who);
  if (rc != FL_OK) return rc;
  if (rows > 1 && (st[1] < least || st[1] >= kMostStride))
    return set_error(FL_ERR_UNSUPPORTED, "%s: the row stride of %s must be in [%lld, 2^24) (got "
                     "%lld)", who, name, (long long)least, (long long)st[1]);
  return FL_OK;
}

int check_written(const int64_t st[2], int64_t heads, int64_t rows, int64_t head_dim,
                  const char* name, const char* who) {
  const int64_t all[3] = {0, st[0], st[1]};
  return check_apart(all, 1, heads, rows, head_dim, name, who);
}

int check_packed(const fl_packed_params* p, const char* who) {
  if (p == nullptr) return null_params(who);
  if (p->dtype != FL_DTYPE_F16 && p->dtype != FL_DTYPE_BF16)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", who, (int)p->dtype);
  if (p->sequences < 0 || p->rows < 0 || p->key_rows < 0 || p->heads < 0 || p->kv_heads < 0)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: sizes must be non-negative", who);
  if (p->head_dim != 64 && p->head_dim != 128)
    return set_error(FL_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128 (got %lld)", who,
                     (long long)p->head_dim);
  if (p->heads > 0 ? p->kv_heads == 0 || p->heads % p->kv_heads != 0 : p->kv_heads > 0)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: %lld heads are not a multiple of %lld key/value "
                     "heads", who, (long long)p->heads, (long long)p->kv_heads);
  const double s = p->sm_scale == 0.0 ? 1.0 / std::sqrt((double)p->head_dim) : p->sm_scale;
  const float c = (float)(std::fabs(s) * 1.4426950408889634);
  if (!std::isfinite(s) || !std::isfinite(c) || c == 0.0f)
    return set_error(FL_ERR_INVALID_ARGUMENT,
                     "%s: sm_scale*log2(e) must be finite and non-zero (sm_scale=%g)", who, s);
  if (p->key_starts == nullptr && p->key_rows != p->rows)
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: without key_starts there are as many key rows as "
                     "rows (%lld, got %lld)", who, (long long)p->rows, (long long)p->key_rows);
  if (p->rows > kMostRows || p->key_rows > kMostRows || p->heads > 16384 ||
      p->sequences > (INT64_C(1) << 24))
    return set_error(FL_ERR_UNSUPPORTED, "%s: at most 2^30 rows, 16384 heads and 2^24 sequences",
                     who);
  if (!(std::fabs(s) >= 1e-30))
    return set_error(FL_ERR_UNSUPPORTED, "%s: sm_scale must be at least 1e-30 in size (got %g)", who,
                     s);
  if (p->heads > 0 && (std::max(p->rows, p->key_rows) / 32 + p->sequences) >
                          INT32_MAX / 16 / p->heads)
    return set_error(FL_ERR_UNSUPPORTED, "%s: too many work-groups", who);
  int rc = check_rows(p->q_stride, p->heads, p->rows, p->head_dim, "q", who);
  if (rc == FL_OK) rc = check_rows(p->k_stride, p->kv_heads, p->key_rows, p->head_dim, "k", who);
  if (rc == FL_OK) rc = check_rows(p->v_stride, p->kv_heads, p->key_rows, p->head_dim, "v", who);
  if (rc == FL_OK) rc = check_rows(p->o_stride, p->heads, p->rows, p->head_dim, "o", who);
  if (rc != FL_OK) return rc;
  if (p->key_rows > 1)
    for (const int64_t sr : {p->k_stride[1], p->v_stride[1]})
      // (tiles past the last key are fetched as zeros, by offsets that must not wrap)
      if ((p->key_rows + 128) * sr * 2 > INT32_MAX)
        return set_error(FL_ERR_UNSUPPORTED,
                         "%s: the rows of k and v, and 128 more, must lie within 2^31 bytes", who);
  return FL_OK;
}

// Dimensions of one entry step nowhere: strides that every kernel's arithmetic
// takes.
void normal(int64_t st[2], int64_t heads, int64_t rows, int64_t head_dim) {
  if (heads <= 1) st[0] = 0;
  if (rows <= 1) st[1] = head_dim;
}

fl_packed_params normal(const fl_packed_params& p) {
  fl_packed_params x = p;
  normal(x.q_stride, p.heads, p.rows, p.head_dim);
  normal(x.o_stride, p.heads, p.rows, p.head_dim);
  normal(x.k_stride, p.kv_heads, p.key_rows, p.head_dim);
  normal(x.v_stride, p.kv_heads, p.key_rows, p.head_dim);
  return x;
}

int check_packed_pointers(const fl_packed_params* p, const char* who) {
  if (!p->starts || (p->rows > 0 && (!p->q || !p->o)) ||
      (p->key_rows > 0 && (!p->k || !p->v)))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: q, k, v, o and starts must be non-NULL", who);
  if (!aligned(p->q, 16) || !aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->o, 16))
    return set_error(FL_ERR_MISALIGNED, "%s: q, k, v and o must be 16-byte aligned", who);
  if (!aligned(p->starts, 4) || !aligned(p->key_starts, 4) || !aligned(p->lse, 4))
    return set_error(FL_ERR_MISALIGNED, "%s: starts and lse must be 4-byte aligned", who);
  return FL_OK;
}

}  // namespace

namespace fl {

// Parts that a key block's queries are cut into, each a work-group with sums of
// its own (packed_bwd.h): at most as many as bring the work-groups that the chip
// holds at once, two a CU, or under a causal mask over long keys, where they
// differ most, twice that (us).  B2 H16/2 N7000-8192 D 128 causal 3169 with one
// a CU, 2117 with two, 1691 with four; B1 H8 N2048 D 64 causal 82.7, 74.5, 82.2;
// 8 sequences of 300-700, H16, not causal, with two 80, with four 101.  Fewer
// where the partial sums cost more than the shorter walks save: a tile of the
// walk takes about 1 us, the join's launch 5, a part 0.3 a MB written and read
// (with dq and dk, dv in two launches, 4 sequences of 300-700, H8 D 64: one part
// 36.4, two 41.8, four 45.7; 4 of 33-257, H8/2: one 39.7, two 31.5, four 27.1,
// eight 26.3; one of 300, H16/4 D 128: one 64.5, eight 37.9).
int packed_bwd_parts(const fl_packed_params& p) {
  const int64_t groups = (p.key_rows / 128 + p.sequences) * p.kv_heads;
  const int64_t a_cu = p.causal && p.key_rows / p.sequences >= 4096 ? 4 : 2;
  const int64_t want = a_cu * device_cus();
  const int64_t most = std::min<int64_t>(4 * a_cu, (want + groups / 2) / groups);
  const int64_t tile = p.head_dim == 128 ? 32 : 64;
  const double walk =
      (double)(p.heads / p.kv_heads) * ((p.rows / p.sequences + tile - 1) / tile);
  const double part = 0.3e-6 * p.kv_heads * p.key_rows * 2 * p.head_dim * 4;
  int best = 1;
  for (int n = 2; n <= most; ++n)
    if (walk / n + 5 + n * part < walk / best + (best > 1 ? 5 + best * part : 0)) best = n;
  return best;
}

}  // namespace fl

extern "C" {

int fl_attn_packed_fwd(const fl_packed_params* p, void* stream) {
  const char* who = "fl_attn_packed_fwd";
  int rc = check_packed(p, who);
  if (rc == FL_OK) rc = check_written(p->o_stride, p->heads, p->rows, p->head_dim, "o", who);
  if (rc != FL_OK) return rc;
  if (p->sequences == 0 || p->rows == 0 || p->heads == 0) return FL_OK;
  rc = check_packed_pointers(p, who);
  if (rc != FL_OK) return rc;
  const fl_packed_params x = normal(*p);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool bf16 = p->dtype == FL_DTYPE_BF16;
  return launched(p->head_dim == 128 ? (bf16 ? fl::launch_packed_fwd_d128_bf16(x, st)
                                             : fl::launch_packed_fwd_d128_f16(x, st))
                                     : (bf16 ? fl::launch_packed_fwd_d64_bf16(x, st)
                                             : fl::launch_packed_fwd_d64_f16(x, st)), who);
}

int64_t fl_attn_packed_bwd_workspace_bytes(const fl_packed_params* p) {
  if (check_packed(p, "fl_attn_packed_bwd_workspace_bytes") != FL_OK) return -1;
  if (p->sequences == 0 || p->heads == 0) return 0;
  // (whichever the mask)
  fl_packed_params x = *p;
  x.causal = 0;
  int64_t parts = fl::packed_bwd_parts(x);
  x.causal = 1;
  parts = std::max<int64_t>(parts, fl::packed_bwd_parts(x));
  return fl::packed_stat_bytes(*p) +
         (parts > 1 ? parts * p->kv_heads * p->key_rows * 2 * p->head_dim * 4 : 0);
}

int fl_attn_packed_bwd(const fl_packed_params* p, const fl_packed_grads* d, void* workspace,
                       int64_t workspace_bytes, void* stream) {
  const char* who = "fl_attn_packed_bwd";
  int rc = check_packed(p, who);
  if (rc != FL_OK) return rc;
  if (d == nullptr) return null_params(who);
  rc = check_rows(d->dout_stride, p->heads, p->rows, 0, "dout", who);
  if (rc == FL_OK) rc = check_rows(d->dq_stride, p->heads, p->rows, 0, "dq", who);
  if (rc == FL_OK) rc = check_rows(d->dk_stride, p->kv_heads, p->key_rows, 0, "dk", who);
  if (rc == FL_OK) rc = check_rows(d->dv_stride, p->kv_heads, p->key_rows, 0, "dv", who);
  if (rc == FL_OK) rc = check_written(d->dq_stride, p->heads, p->rows, p->head_dim, "dq", who);
  if (rc == FL_OK)
    rc = check_written(d->dk_stride, p->kv_heads, p->key_rows, p->head_dim, "dk", who);
  if (rc == FL_OK)
    rc = check_written(d->dv_stride, p->kv_heads, p->key_rows, p->head_dim, "dv", who);
  if (rc != FL_OK) return rc;
  if (p->sequences == 0 || p->heads == 0) return FL_OK;
  rc = check_packed_pointers(p, who);
  if (rc != FL_OK) return rc;
  if ((p->rows > 0 && (!p->lse || !d->dout || !d->dq)) || (p->key_rows > 0 && (!d->dk || !d->dv)))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: lse, dout, dq, dk and dv must be non-NULL", who);
  if (!aligned(d->dout, 16) || !aligned(d->dq, 16) || !aligned(d->dk, 16) || !aligned(d->dv, 16))
    return set_error(FL_ERR_MISALIGNED, "%s: dout, dq, dk and dv must be 16-byte aligned", who);
  const int64_t need = fl_attn_packed_bwd_workspace_bytes(p);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(FL_ERR_INVALID_ARGUMENT, "%s: a workspace of %lld bytes is needed (got %lld)",
                     who, (long long)need, (long long)(workspace ? workspace_bytes : 0));
  if (!aligned(workspace, 16))
    return set_error(FL_ERR_MISALIGNED, "%s: workspace must be 16-byte aligned", who);
  const fl_packed_params x = normal(*p);
  fl_packed_grads y = *d;
  normal(y.dout_stride, p->heads, p->rows, p->head_dim);
  normal(y.dq_stride, p->heads, p->rows, p->head_dim);
  normal(y.dk_stride, p->kv_heads, p->key_rows, p->head_dim);
  normal(y.dv_stride, p->kv_heads, p->key_rows, p->head_dim);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  return launched(p->dtype == FL_DTYPE_BF16 ? fl::launch_packed_bwd_bf16(x, y, workspace, st)
                                            : fl::launch_packed_bwd_f16(x, y, workspace, st), who);
}

}  // extern "C"
