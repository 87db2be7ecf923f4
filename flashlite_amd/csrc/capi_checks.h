// Argument checks that the C-ABI entry points of capi_serve.hip and
// capi_packed.hip share.
#pragma once

#include <algorithm>
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

[[maybe_unused]] bool fits32(int64_t x) { return x >= 0 && x <= INT32_MAX; }

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

}  // namespace
