// Checks of views that the entry points of the cache and of latent attention share.
#pragma once
#include "aotriton_amd/cache.h"
#include "fa_args.h"

namespace fa {
namespace checks {

constexpr int64_t kMaxRowStride = 1 << 21;      // elements, as in the other entry points
constexpr uint64_t kMaxCount = 0x7fffffff;
constexpr uint64_t kTreeColumns = 256;      // of the attention over K and V; what only moves rows takes those of a latent cache, too
constexpr uint64_t kRowColumns = 576;

inline bool empty(const fa_tensor4& t) { return t.sizes[0] == 0 || t.sizes[1] == 0 || t.sizes[2] == 0; }

// rows of up to `columns` columns made of aligned 16-byte pieces, no negative stride
inline int check_rows(const fa_tensor4& t, int dtype, uint64_t columns) {
  if (t.dtype != dtype || (t.ptr == nullptr && !empty(t))) return FA_ERROR_INVALID_VALUE;
  for (int i = 0; i < 4; ++i)
    if (t.sizes[i] > kMaxCount) return FA_ERROR_INVALID_VALUE;
  if (t.sizes[3] == 0 || t.sizes[3] > columns || t.sizes[3] % 8 != 0 || (t.strides[3] != 1 && t.sizes[3] > 1)) return FA_ERROR_NOT_SUPPORTED;
  if ((reinterpret_cast<uintptr_t>(t.ptr) & 15u) != 0) return FA_ERROR_NOT_SUPPORTED;
  for (int i = 0; i < 3; ++i)
    if (t.sizes[i] > 1 && ((int64_t)t.strides[i] < 0 || t.strides[i] % 8 != 0)) return FA_ERROR_NOT_SUPPORTED;
  if (t.sizes[2] > 1 && (int64_t)t.strides[2] > kMaxRowStride) return FA_ERROR_NOT_SUPPORTED;
  return FA_SUCCESS;
}

// int32 values next to each other, `n` of them
inline int check_ints(const fa_tensor1& t, uint64_t n) {
  if (t.dtype != FA_DTYPE_INT32 || t.sizes[0] != n || (t.ptr == nullptr && n > 0)) return FA_ERROR_INVALID_VALUE;
  if (n > 1 && t.strides[0] != 1) return FA_ERROR_NOT_SUPPORTED;
  return FA_SUCCESS;
}

// int32 rows with adjacent columns
inline int check_int_rows(const fa_tensor2& t, uint64_t rows) {
  if (t.dtype != FA_DTYPE_INT32 || t.sizes[0] != rows || t.sizes[1] > kMaxCount) return FA_ERROR_INVALID_VALUE;
  if (t.ptr == nullptr && t.sizes[0] * t.sizes[1] > 0) return FA_ERROR_INVALID_VALUE;
  if ((t.sizes[1] > 1 && t.strides[1] != 1) || (t.sizes[0] > 1 && (int64_t)t.strides[0] < 0)) return FA_ERROR_NOT_SUPPORTED;
  return FA_SUCCESS;
}

// Rows of a tensor that is written have to lie apart.
inline bool rows_apart(const fa_tensor2& t) { return t.sizes[0] <= 1 || t.strides[0] >= t.sizes[1]; }
// (an expanded cache has one row for many)
inline bool written_apart(const fa_tensor4& t) {
  for (int i = 0; i < 3; ++i)
    if (t.sizes[i] > 1 && t.strides[i] < t.sizes[3]) return false;
  return true;
}
inline bool written_apart(const fa_cache& c) { return written_apart(c.K) && written_apart(c.V); }

inline fa::Strides3 strides3(const fa_tensor4& t) {
  return fa::Strides3{(int64_t)t.strides[0], (int64_t)t.strides[1], (int64_t)t.strides[2]};
}

// a launch's workgroups have to fit 31 bits
inline bool fits(double workgroups) { return workgroups < 2147483648.0; }

}  // namespace checks
}  // namespace fa
