// Kernels of the embedding lookup, of its gradient and of the rows sorted by id.
#pragma once

#include "row_types.hpp"
#include "spmm_kernels.hpp"

namespace hpspmm {

// out[i, :] = scale * table[ids[i], :], rows of zeros for ids outside the table.  A thread owns 16 bytes of a row;
// 2^tpr_log2 adjacent threads share a row's column tile, a workgroup covers kRows rows one after the other, all of
// whose loads are in flight together.
template <class T, class Id, bool kAligned, int kRows>
__global__ __launch_bounds__(kBlock) void embedding_lookup_kernel(int64_t n, uint32_t vocab, int32_t width, int tpr_log2,
                                                                 const Id* __restrict__ ids, const T* __restrict__ table,
                                                                 int64_t ld_table, float scale, T* __restrict__ out,
                                                                 int64_t ld_out) {
  constexpr int V = kPer16<T>;
  const int tpr = 1 << tpr_log2;
  const int per_pass = kBlock >> tpr_log2;  // rows a pass of the workgroup covers
  const int col = ((int)blockIdx.y * tpr + ((int)threadIdx.x & (tpr - 1))) * V;
  const int64_t row0 = (int64_t)blockIdx.x * per_pass * kRows + ((int)threadIdx.x >> tpr_log2);
  if (col >= width) return;
  uint32_t key[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + (int64_t)r * per_pass;
    key[r] = row < n ? id_key(ids[row], vocab) : vocab;
  }
  if (col + V <= width) {
    float v[kRows][V];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (key[r] < vocab) {
        load16<kAligned>(table + (int64_t)key[r] * ld_table + col, v[r]);
#pragma unroll
        for (int i = 0; i < V; ++i) v[r][i] *= scale;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[r][i] = 0.f;
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = row0 + (int64_t)r * per_pass;
      if (row < n) store_n<kAligned, T, V>(out + row * ld_out + col, v[r]);
    }
  } else {
    for (int r = 0; r < kRows; ++r) {
      const int64_t row = row0 + (int64_t)r * per_pass;
      if (row >= n) break;
      for (int c = col; c < width; ++c)
        out[row * ld_out + c] =
            key[r] < vocab ? (T)(scale * (float)table[(int64_t)key[r] * ld_table + c]) : (T)0.f;
    }
  }
}

// keys[i] = id of row i (or `ids` when it is outside [0, ids)), vals[i] = i.
template <class Id>
__global__ __launch_bounds__(kBlock) void row_keys_kernel(int64_t n, uint32_t ids, const Id* __restrict__ id,
                                                         uint32_t* __restrict__ keys, int32_t* __restrict__ vals) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= n) return;
  keys[i] = id_key(id[i], ids);
  vals[i] = (int32_t)i;
}

// First position of the sorted keys that is not below `key`.
__device__ __forceinline__ int64_t lower_bound_u32(const uint32_t* __restrict__ keys, int64_t n, uint32_t key) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// offsets[g] = rows whose key is below g, g = 0 ... groups; order[i] = the sorted rows.
HPSPMM_KERNEL __launch_bounds__(kBlock) void row_offsets_kernel(int64_t n, int64_t groups,
                                                             const uint32_t* __restrict__ keys,
                                                             const int32_t* __restrict__ vals,
                                                             int32_t* __restrict__ order,
                                                             int32_t* __restrict__ offsets) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i <= groups) offsets[i] = (int32_t)lower_bound_u32(keys, n, (uint32_t)i);
  if (i < n) order[i] = vals[i];
}

// d_table[v, :] = (accumulate ? d_table[v, :] : 0) + scale * sum of the rows of `grad` whose key is v, in the order of
// their positions.  One workgroup per row of the table and column tile.
template <class T, class TO>
__global__ __launch_bounds__(kBlock) void embedding_grad_kernel(int64_t n, int32_t width, const uint32_t* __restrict__ keys,
                                                               const int32_t* __restrict__ pos,
                                                               const T* __restrict__ grad, int64_t ld_grad, float scale,
                                                               TO* __restrict__ d_table, int64_t ld_table,
                                                               int accumulate) {
  const uint32_t v = blockIdx.x;
  const int64_t first = lower_bound_u32(keys, n, v), last = lower_bound_u32(keys, n, v + 1);
  if (first == last && accumulate) return;
  for (int c = (int)blockIdx.y * kBlock + (int)threadIdx.x; c < width; c += (int)gridDim.y * kBlock) {
    float sum = 0.f;
    for (int64_t q = first; q < last; ++q) sum += (float)grad[(int64_t)pos[q] * ld_grad + c];
    TO* at = d_table + (int64_t)v * ld_table + c;
    const float old = accumulate ? (float)*at : 0.f;
    *at = (TO)(old + scale * sum);
  }
}

}  // namespace hpspmm
