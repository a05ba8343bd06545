// What the kernels of the products grouped by expert share: the operands, the row tiles of the groups.
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
  int splits;    // gradient of w: parts that the rows of a group are cut into
  float* parts;  // [splits * tiles][kSplitEdge * kSplitEdge] their sums
};

// Where the gradient of w has few tiles, the rows of each group are cut into parts: tiles of this edge, at most so many
// of them times parts (32 MB of sums).
constexpr int kSplitEdge = 128;
constexpr int64_t kSplitTiles = 512;

// Rows [begin, end) of a group; offsets that are no partition of the rows give other products, never an access
// outside the operands.
__device__ __forceinline__ void group_rows_of(const GroupedArgs& g, int64_t e, int64_t& begin, int64_t& end) {
  begin = min(max((int64_t)g.offsets[e], (int64_t)0), g.rows);
  end = min(max((int64_t)g.offsets[e + 1], begin), g.rows);
}

// A value that all lanes hold, in scalar registers.
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Row tiles of all groups together, each group starting a tile of its own.
__device__ __forceinline__ int64_t count_row_tiles(const GroupedArgs& g, int bm) {
  const int lane = threadIdx.x & 63;
  int tiles = 0;
#pragma unroll 4
  for (int64_t e = lane; e < g.groups; e += 64) {
    int64_t b, f;
    group_rows_of(g, e, b, f);
    tiles += (int)((f - b + bm - 1) / bm);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) tiles += __shfl_xor(tiles, d, 64);
  return __builtin_amdgcn_readfirstlane(tiles);
}

// The group of row tile `tile` (tiles of `bm` rows, each group starts a tile of its own), its rows [begin, end) and its
// first tile; false when there are fewer tiles.  Every wavefront looks for itself, 256 groups a step, four a lane (4096
// groups: 64 a step and 64 steps of two loads each made most of a product of 4096 x 64 x 64, 215 us).
__device__ __forceinline__ bool find_group(const GroupedArgs& g, int64_t tile, int bm, int64_t& e, int64_t& begin,
                                           int64_t& end, int64_t& first) {
  constexpr int kEach = 4;
  const int lane = threadIdx.x & 63;
  int64_t before = 0;
  for (int64_t base = 0; base < g.groups; base += 64 * kEach) {
    int64_t b[kEach] = {}, f[kEach] = {};
    int tiles[kEach], mine = 0;
#pragma unroll
    for (int q = 0; q < kEach; ++q) {
      const int64_t at = base + lane * kEach + q;
      if (at < g.groups) group_rows_of(g, at, b[q], f[q]);
      tiles[q] = (int)((f[q] - b[q] + bm - 1) / bm);
      mine += tiles[q];
    }
    int upto = mine;  // tiles of the groups up to this lane's
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int other = __shfl_up(upto, d, 64);
      if (lane >= d) upto += other;
    }
    const uint64_t past = __ballot(before + upto > tile);
    if (past) {
      // the lane that has the group, and which of its four
      const int at = __ffsll((unsigned long long)past) - 1;
      int64_t start = before + upto - mine, my_begin = b[0], my_end = f[0];
      int which = 0;
#pragma unroll
      for (int q = 0; q + 1 < kEach; ++q)
        if (which == q && start + tiles[q] <= tile) {
          start += tiles[q];
          which = q + 1;
          my_begin = b[q + 1];
          my_end = f[q + 1];
        }
      e = base + at * kEach + __builtin_amdgcn_readfirstlane(__shfl(which, at, 64));
      begin = uniform64(__shfl(my_begin, at, 64));
      end = uniform64(__shfl(my_end, at, 64));
      first = uniform64(__shfl(start, at, 64));
      return true;
    }
    before += __builtin_amdgcn_readfirstlane(__shfl(upto, 63, 64));
  }
  return false;
}

// Tile `t` of a matrix of row_tiles x col_tiles output tiles, walked in panels of kPanel columns, row by row within a
// panel: the tiles that are worked on at a time form a block, whose strips of the operands are shared.
constexpr int kPanel = 8;
__device__ __forceinline__ void panel_tile(int64_t t, int64_t row_tiles, int col_tiles, int64_t& row, int& col) {
  const int64_t panel = t / (row_tiles * kPanel);
  const int left = col_tiles - (int)panel * kPanel, wide = left < kPanel ? left : kPanel;
  const int64_t in = t - panel * row_tiles * kPanel;
  row = in / wide;
  col = (int)panel * kPanel + (int)(in - row * wide);
}

// dw = (accumulate ? dw : 0) + the parts' sums, added in their order and rounded once.  A workgroup sums 1024 elements of
// one tile; bound by the bytes of the parts, at most 32 MB (6 to 7 us).
template <class TO>
__global__ __launch_bounds__(kBlock) void grouped_join_kernel(GroupedArgs g, int col_tiles) {
  const int64_t t = blockIdx.x, tiles = gridDim.x;
  const int row_tiles = (g.m + kSplitEdge - 1) / kSplitEdge;
  const int64_t e = t / (row_tiles * col_tiles);
  int64_t mt;
  int nt;
  panel_tile(t - e * row_tiles * col_tiles, row_tiles, col_tiles, mt, nt);
  const int at = ((int)blockIdx.y * kBlock + (int)threadIdx.x) * 4;
  const int64_t row = mt * kSplitEdge + at / kSplitEdge;
  const int col = nt * kSplitEdge + at % kSplitEdge;
  if (row >= g.m || col >= g.k) return;
  float v[4] = {};
#pragma unroll 4
  for (int s = 0; s < g.splits; ++s) {
    float part[4];
    load16<true>(g.parts + (s * tiles + t) * (kSplitEdge * kSplitEdge) + at, part);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += part[i];
  }
  TO* out = (TO*)g.c + e * g.stride_c + row * g.ldc + col;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (col + i < g.k) out[i] = (TO)(v[i] + (g.accumulate ? (float)out[i] : 0.f));
}

}  // namespace hpspmm
