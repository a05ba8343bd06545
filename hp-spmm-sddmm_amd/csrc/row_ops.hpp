// Host side shared by the row operators (row_ops.hip, grouped_mm.hip): their plan, their argument checks, the
// dispatch on element types.
#pragma once

#include "host.hpp"
#include "row_types.hpp"

struct hpspmm_rows_plan {
  int device = 0;
  int64_t max_rows = 0, max_ids = 0, max_width = 0;
  char* arena = nullptr;
  uint32_t* d_keys[2] = {nullptr, nullptr};  // [max_rows] ids, sorted
  int32_t* d_vals[2] = {nullptr, nullptr};   // [max_rows] the rows they belong to
  uint32_t* d_hist = nullptr;                // [tiles * bins] counts per digit and tile of rows
  uint32_t* d_scan = nullptr;
  float* d_carry = nullptr;                  // sums that cross chunks of the sorted rows
  int64_t carry_floats = 0;
  float* d_split = nullptr;                  // sums of the parts of a gradient of the weights
};

namespace hpspmm_host {

inline bool known_dtype(int t) { return t == HPSPMM_F32 || t == HPSPMM_BF16 || t == HPSPMM_F16; }
inline int64_t dtype_size(int t) { return t == HPSPMM_F32 ? 4 : 2; }

// f(T{}) for the element type of an hpspmm_dtype.
template <class F>
int dispatch_dtype(int t, F&& f) {
  switch (t) {
    case HPSPMM_BF16: return f(hpspmm::bf16_t{});
    case HPSPMM_F16: return f(hpspmm::f16_t{});
    default: return f(float{});
  }
}
template <class F>
int dispatch_id(int t, F&& f) {
  return t == HPSPMM_I64 ? f(int64_t{}) : f(int32_t{});
}

// Elements of a row length or leading dimension: 1 ... 2^20 columns, rows at most 2^40 elements apart.
constexpr int64_t kMaxRowLength = (int64_t)1 << 20;
constexpr int64_t kMaxStride = (int64_t)1 << 40;

inline bool aligned_to(const void* p, int64_t bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

// A matrix operand: its address (may be null only where it has no rows) and its leading dimension.
int check_matrix(const char* name, const void* p, int64_t rows, int64_t width, int64_t ld, int dtype);

// The plan serves `rows` rows of ids below `ids` (and rows of `width` columns), on the current device.
int check_rows_plan(const hpspmm_rows_plan* plan, int64_t rows, int64_t ids, int64_t width);

}  // namespace hpspmm_host
