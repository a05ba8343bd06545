// Kernels of the products grouped by expert.
//
//   kForward   y[i, :]  = x[i, :] * w[e]^T      rows i of group e, contraction over k
//   kGradX     dx[i, :] = dy[i, :] * w[e]       contraction over m
//   kGradW     dw[e]    = dy_e^T * x_e          contraction over the rows of group e
#pragma once

#include "row_types.hpp"
#include "spmm_kernels.hpp"

namespace hpspmm {

enum GroupedMode { kForward = 0, kGradX = 1, kGradW = 2 };

struct GroupedArgs {
  int64_t rows, groups;
  int32_t k, m;
  const int32_t* offsets;
  const void* a;  // x (forward), dy (gradients)
  int64_t lda;
  const void* b;  // w (forward, gradient of x), x (gradient of w)
  int64_t ldb, stride_b;
  void* c;  // y, dx, dw
  int64_t ldc, stride_c;
  int accumulate;
};

// Rows [begin, end) of a group; offsets that are no partition of the rows give other products, never an access
// outside the operands.
__device__ __forceinline__ void group_rows_of(const GroupedArgs& g, int64_t e, int64_t& begin, int64_t& end) {
  begin = min(max((int64_t)g.offsets[e], (int64_t)0), g.rows);
  end = min(max((int64_t)g.offsets[e + 1], begin), g.rows);
}

// The group and first row of row tile `tile` (tiles of `bm` rows, each group starts a tile of its own); false when
// there are fewer tiles.  Every wavefront looks for itself, 64 groups a step.
__device__ __forceinline__ bool find_row_tile(const GroupedArgs& g, int64_t tile, int bm, int64_t& e, int64_t& row0,
                                              int64_t& end) {
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int64_t base = 0; base < g.groups; base += 64) {
    int64_t b = 0, f = 0;
    if (base + lane < g.groups) group_rows_of(g, base + lane, b, f);
    const int tiles = (int)((f - b + bm - 1) / bm);
    int upto = tiles;  // tiles of the groups up to this lane's
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int other = __shfl_up(upto, d, 64);
      if (lane >= d) upto += other;
    }
    const uint64_t past = __ballot(before + upto > tile);
    if (past) {
      const int at = __ffsll((unsigned long long)past) - 1;
      e = base + at;
      const int64_t begin = __shfl(b, at, 64);
      end = __shfl(f, at, 64);
      const int first = __shfl(upto - tiles, at, 64);
      row0 = begin + (tile - before - first) * bm;
      return true;
    }
    before += __shfl(upto, 63, 64);
  }
  return false;
}

constexpr int kSimpleTile = 64, kSimpleDepth = 16;

// Any size and stride: tiles of 64 x 64 outputs, 16 terms of the contraction at a time in LDS as 32-bit values, each
// thread sums 4 x 4 of them.
template <class T, class TO, int kMode>
__global__ __launch_bounds__(kBlock) void grouped_simple_kernel(GroupedArgs g) {
  __shared__ float sa[kSimpleDepth][kSimpleTile + 1], sb[kSimpleDepth][kSimpleTile + 1];
  int64_t e, begin, end, row0 = 0;
  if constexpr (kMode == kGradW) {
    e = blockIdx.z;
    group_rows_of(g, e, begin, end);
  } else {
    if (!find_row_tile(g, blockIdx.x, kSimpleTile, e, row0, end)) return;
    begin = row0;
  }
  const T* a = (const T*)g.a;
  const T* b = (const T*)g.b + (kMode == kGradW ? 0 : e * g.stride_b);
  const int n_out = kMode == kForward ? g.m : g.k;  // columns of the output
  const int64_t m_out = kMode == kGradW ? (int64_t)g.m : end - row0;
  const int64_t depth = kMode == kForward ? (int64_t)g.k : kMode == kGradX ? (int64_t)g.m : end - begin;
  const int m0 = kMode == kGradW ? (int)blockIdx.x * kSimpleTile : 0;
  const int n0 = (int)blockIdx.y * kSimpleTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t d0 = 0; d0 < depth; d0 += kSimpleDepth) {
    for (int q = threadIdx.x; q < kSimpleTile * kSimpleDepth; q += kBlock) {
      // neighbouring threads read neighbouring elements
      const int ai = kMode == kGradW ? q & 63 : q >> 4, ad = kMode == kGradW ? q >> 6 : q & 15;
      float v = 0.f;
      if (m0 + ai < m_out && d0 + ad < depth)
        v = kMode == kGradW ? (float)a[(begin + d0 + ad) * g.lda + m0 + ai] : (float)a[(row0 + ai) * g.lda + d0 + ad];
      sa[ad][ai] = v;
      const int bi = kMode == kForward ? q >> 4 : q & 63, bd = kMode == kForward ? q & 15 : q >> 6;
      v = 0.f;
      if (n0 + bi < n_out && d0 + bd < depth) {
        if constexpr (kMode == kForward) v = (float)b[(int64_t)(n0 + bi) * g.ldb + d0 + bd];
        else if constexpr (kMode == kGradX) v = (float)b[(d0 + bd) * g.ldb + n0 + bi];
        else v = (float)b[(begin + d0 + bd) * g.ldb + n0 + bi];
      }
      sb[bd][bi] = v;
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < kSimpleDepth; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += sa[d][ty + 16 * i] * sb[d][tx + 16 * j];
    __syncthreads();
  }
  TO* c = (TO*)g.c + (kMode == kGradW ? e * g.stride_c : row0 * g.ldc);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int mi = m0 + ty + 16 * i, ni = n0 + tx + 16 * j;
      if (mi < m_out && ni < n_out) {
        TO* at = c + (int64_t)mi * g.ldc + ni;
        const float old = g.accumulate ? (float)*at : 0.f;
        *at = (TO)(old + acc[i][j]);
      }
    }
}

}  // namespace hpspmm
