// Entry points of the products grouped by expert.
#include "row_ops.hpp"

#include "grouped_tile_kernel.hpp"

using namespace hpspmm_host;

namespace {

// Every workgroup of a product finds its tile's group by a walk over all offsets: 4096 groups of 64 x 64 (4096 rows) take 116
// us, 65535 of them (131072 rows) 34 ms, nearly all of it the search.  More groups than that are refused.
constexpr int64_t kMaxGroups = 65535;

int check_grouped(int64_t rows, int64_t groups, int64_t k, int64_t m, const int32_t* d_offsets, int dtype) {
  if (rows < 0 || groups < 0 || rows >= INT32_MAX || groups > kMaxGroups)
    return fail(HPSPMM_ERR_INVALID_ARG, "rows must be in [0, 2^31 - 1) and groups in [0, 65535], got %lld and %lld",
                (long long)rows, (long long)groups);
  if (k <= 0 || m <= 0 || k > kMaxRowLength || m > kMaxRowLength)
    return fail(HPSPMM_ERR_INVALID_ARG, "k and m must be in [1, 2^20], got %lld and %lld", (long long)k, (long long)m);
  if (!known_dtype(dtype)) return fail(HPSPMM_ERR_INVALID_ARG, "unknown element type %d", dtype);
  if (groups > 0 && !d_offsets) return fail(HPSPMM_ERR_INVALID_ARG, "d_offsets is NULL");
  if (!aligned_to(d_offsets, 4)) return fail(HPSPMM_ERR_INVALID_ARG, "d_offsets is not at a multiple of 4 bytes");
  return HPSPMM_OK;
}

// One matrix of m rows of k columns for every group, `stride` elements apart.
int check_weights(const char* name, const void* p, int64_t groups, int64_t k, int64_t m, int64_t ld, int64_t stride,
                  int dtype, bool written) {
  if (int rc = check_matrix(name, p, groups, k, ld, dtype)) return rc;
  if (stride < 0 || stride > kMaxStride || (written && groups > 1 && stride < (m - 1) * ld + k))
    return fail(HPSPMM_ERR_INVALID_ARG, "%s: stride %lld between matrices of %lld rows, leading dimension %lld", name,
                (long long)stride, (long long)m, (long long)ld);
  return HPSPMM_OK;
}

// Row tiles of bm rows that the groups can have together, whatever their sizes.
int64_t most_row_tiles(int64_t rows, int64_t groups, int64_t bm) { return std::min(rows, rows / bm + groups); }

// Rows of an operand that 16-byte chunks cover whole, at multiples of 16 bytes, near enough together for 32-bit offsets
// within a tile.
bool chunked(const void* p, int64_t ld, int64_t stride, int64_t width, int64_t size) {
  return aligned_to(p, 16) && ld * size % 16 == 0 && stride * size % 16 == 0 && width * size % 16 == 0 && ld < ((int64_t)1 << 21);
}

// Output tiles of edge `edge` that a product can be expected to have: every group ends half way through a tile.
int64_t expected_tiles(int mode, const hpspmm::GroupedArgs& g, int64_t edge) {
  const int64_t cols = ceil_div(mode == hpspmm::kForward ? g.m : g.k, edge);
  if (mode == hpspmm::kGradW) return cols * g.groups * ceil_div(g.m, edge);
  return cols * std::max<int64_t>(1, std::min(g.rows, g.rows / edge + g.groups / 2));
}

// Edge of the output tiles, 256 (16-bit operands at multiples of 16 bytes), 128 or 64: the one that is expected to take
// the least time, tiles per CU (one at least, and a part of a round that is not full) times the area of a tile over its
// rate.  bf16, rows x groups x k x m, product with tiles of 64 / 128 / 256, us a call among many on three sets of operands in
// turn: 32768 x 32 x 2048 x 4096 980 / 622 / 544, 8192 x 8 x 2048 x 2048 132 / 89 / 103, 8192 x 8 x 1024 x 1024 44 / 30 / 30,
// 2000 x 8 x 1024 x 1024 18 / 14 / 29, 32 x 64 x 2048 x 1024 22 / 31 / 49; gradient of x of 16384 x 16 x 2048 x 4096, 2.25
// rounds of 256, - / 322 / 304.  Only the ratios of the rates count: 128 to 256 is the first line's 0.875 raised to 0.893, from
// 0.888 on the second line gets its 128; 64 to 128 is set by the last two (the first line alone would have it 0.63).  32-bit
// products wait for the matrix cores whatever the tile, 64 / 128: 16384 x 16 x 2048 x 2048 1148 / 1102 us (the rate of 64),
// 8192 x 8 x 1024 x 1024 168 / 193, 20000 x 8 x 512 x 2048 390 / 335, gradient of x of 4096 x 8 x 1024 x 2048 185 / 253, of
// w 270 / 245, of 1777 x 10 x 1001 x 519 29 / 49.
int tile_edge(int mode, const hpspmm::GroupedArgs& g, bool wide, bool large) {
  const struct { int edge; double rate; } kinds[] = {{256, 1030}, {128, 920}, {64, wide ? 885.0 : 490.0}};
  int best = 64;
  double least = 0;
  for (const auto& q : kinds) {
    if (q.edge == 256 && !large) continue;
    const double per_cu = std::max(1.0, (double)expected_tiles(mode, g, q.edge) / 256 + 0.1);
    const double time = per_cu * q.edge * q.edge / q.rate;
    if (least == 0 || time < least) {
      least = time;
      best = q.edge;
    }
  }
  return best;
}

template <class T, class TO, int kMode, int kBM, int kBN, int kWM, int kWN, bool kDirect, int kStagesA, int kStagesB>
int launch_tiles(const hpspmm::GroupedArgs& g, hipStream_t st) {
  const int64_t n_out = kMode == hpspmm::kForward ? g.m : g.k;
  const int64_t col_tiles = ceil_div(n_out, kBN);
  const int64_t row_tiles = kMode == hpspmm::kGradW ? g.groups * ceil_div(g.m, kBM) : most_row_tiles(g.rows, g.groups, kBM);
  const int64_t tiles = ceil_div(row_tiles * col_tiles, hpspmm::kXcds) * hpspmm::kXcds;
  if (tiles == 0) return HPSPMM_OK;
  if (tiles > INT32_MAX / (64 * kWM * kWN)) return fail(HPSPMM_ERR_INVALID_ARG, "the product has too many output tiles");
  hipLaunchKernelGGL((hpspmm::grouped_tile_kernel<T, TO, kMode, kBM, kBN, kWM, kWN, kDirect, kStagesA, kStagesB>), dim3((unsigned)tiles),
                     dim3(64 * kWM * kWN), 0, st, g, (int)col_tiles);
  return HPSPMM_OK;
}

// Parts that the rows of every group are cut into for the gradient of the weights, 1 = none: where there are few output
// tiles and long groups, as many as give every slot of the chip a tile, each of at least 4 steps of the mean group.
// 18867 x 2 x 2304 x 89 bf16 116 -> 42 us, 32768 x 1 x 512 x 512 130 -> 31 us, 9000 x 2 x 200 x 89 51 -> 18 us.
int row_splits(const hpspmm::GroupedArgs& g, int64_t depth) {
  const int64_t tiles = expected_tiles(hpspmm::kGradW, g, hpspmm::kSplitEdge);
  const int64_t steps = g.rows / g.groups / depth;
  return (int)std::max<int64_t>(1, std::min(hpspmm::kSplitTiles / std::max<int64_t>(tiles, 1), steps / 4));
}

// How a product is cut: the edge of its output tiles, and the parts of the rows (1 = none) for the gradient of the weights.
struct Tiling {
  int edge, splits;
};
Tiling tiling_of(int mode, const hpspmm::GroupedArgs& g, int64_t size, bool direct) {
  if (mode == hpspmm::kGradW) {
    const int splits = row_splits(g, 128 / size);
    if (splits > 1) return {hpspmm::kSplitEdge, splits};
  }
  return {tile_edge(mode, g, size == 4, size == 2 && direct), 1};
}

// The gradient of the weights in parts: sums in 32 bits of every part and tile to the plan's workspace, then their sum.
template <class T, class TO>
int launch_split(hpspmm::GroupedArgs g, int splits, bool direct, hipStream_t st) {
  g.splits = splits;
  constexpr int E = hpspmm::kSplitEdge;
  const int64_t col_tiles = ceil_div(g.k, E), tiles = g.groups * ceil_div(g.m, E) * col_tiles;
  const unsigned grid = (unsigned)(ceil_div(tiles * splits, hpspmm::kXcds) * hpspmm::kXcds);
  if (direct)
    hipLaunchKernelGGL((hpspmm::grouped_tile_kernel<T, TO, hpspmm::kGradW, E, E, 2, 2, true, 3, 2, true>), dim3(grid), dim3(256), 0,
                       st, g, (int)col_tiles);
  else
    hipLaunchKernelGGL((hpspmm::grouped_tile_kernel<T, TO, hpspmm::kGradW, E, E, 2, 2, false, 2, 2, true>), dim3(grid), dim3(256), 0,
                       st, g, (int)col_tiles);
  hipLaunchKernelGGL((hpspmm::grouped_join_kernel<TO>), dim3((unsigned)tiles, E * E / (4 * hpspmm::kBlock)), dim3(hpspmm::kBlock), 0, st,
                     g, (int)col_tiles);
  return HPSPMM_OK;
}

template <int kMode>
int launch_grouped(const hpspmm::GroupedArgs& g, int dtype, int out_type, hipStream_t st) {
  if (g.groups == 0 || (kMode != hpspmm::kGradW && g.rows == 0)) return HPSPMM_OK;
  const int64_t size = dtype_size(dtype);
  const int64_t wide_a = kMode == hpspmm::kForward ? g.k : g.m;
  const bool direct = chunked(g.a, g.lda, 0, wide_a, size) && chunked(g.b, g.ldb, g.stride_b, g.k, size);
  int rc = dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return dispatch_dtype(out_type, [&](auto o) {
      using TO = decltype(o);
      if constexpr (std::is_same_v<T, TO> || (kMode == hpspmm::kGradW && std::is_same_v<TO, float>)) {
        const auto [edge, splits] = tiling_of(kMode, g, size, direct);
        if constexpr (kMode == hpspmm::kGradW) {
          if (splits > 1) return launch_split<T, TO>(g, splits, direct, st);
        }
        if constexpr (sizeof(T) == 2) {
          if (edge == 256) return launch_tiles<T, TO, kMode, 256, 256, 2, 4, true, 3, 2>(g, st);
        }
        if (edge == 128)
          return direct ? launch_tiles<T, TO, kMode, 128, 128, 2, 2, true, 3, 2>(g, st)
                        : launch_tiles<T, TO, kMode, 128, 128, 2, 2, false, 2, 2>(g, st);
        return direct ? launch_tiles<T, TO, kMode, 64, 64, 2, 2, true, 4, 4>(g, st)
                      : launch_tiles<T, TO, kMode, 64, 64, 2, 2, false, 2, 2>(g, st);
      } else {
        return fail(HPSPMM_ERR_INVALID_ARG, "no product of these types");
      }
    });
  });
  if (rc) return rc;
  HPSPMM_HIP(hipGetLastError());
  return HPSPMM_OK;
}

}  // namespace

HPSPMM_API int hpspmm_grouped_tiling(int product, int64_t rows, int64_t groups, int64_t k, int64_t m, int dtype, int whole16,
                                     int* edge_out, int* parts_out) {
  if (!edge_out || !parts_out) return fail(HPSPMM_ERR_INVALID_ARG, "edge_out or parts_out is NULL");
  *edge_out = *parts_out = 0;
  if (product < hpspmm::kForward || product > hpspmm::kGradW) return fail(HPSPMM_ERR_INVALID_ARG, "unknown product %d", product);
  static const int32_t none = 0;
  if (int rc = check_grouped(rows, groups, k, m, &none, dtype)) return rc;
  if (groups == 0 || (product != hpspmm::kGradW && rows == 0)) return HPSPMM_OK;
  hpspmm::GroupedArgs g{};
  g.rows = rows, g.groups = groups, g.k = (int32_t)k, g.m = (int32_t)m;
  const auto [edge, splits] = tiling_of(product, g, dtype_size(dtype), whole16 != 0);
  *edge_out = edge;
  *parts_out = splits;
  return HPSPMM_OK;
}

HPSPMM_API int hpspmm_grouped_mm(int64_t rows, int64_t groups, int64_t k, int64_t m, const void* d_x, int64_t ld_x,
                                 const void* d_w, int64_t ld_w, int64_t stride_w, const int32_t* d_offsets, void* d_y,
                                 int64_t ld_y, int dtype, void* stream) {
  if (int rc = check_grouped(rows, groups, k, m, d_offsets, dtype)) return rc;
  if (int rc = check_matrix("d_x", d_x, rows, k, ld_x, dtype)) return rc;
  if (int rc = check_weights("d_w", d_w, groups, k, m, ld_w, stride_w, dtype, false)) return rc;
  if (int rc = check_matrix("d_y", d_y, rows, m, ld_y, dtype)) return rc;
  const hpspmm::GroupedArgs g{rows, groups, (int32_t)k, (int32_t)m, d_offsets, d_x, ld_x, d_w, ld_w, stride_w, d_y, ld_y, 0, 0, 1, nullptr};
  return launch_grouped<hpspmm::kForward>(g, dtype, dtype, (hipStream_t)stream);
}

HPSPMM_API int hpspmm_grouped_mm_grad_x(int64_t rows, int64_t groups, int64_t k, int64_t m, const void* d_dy,
                                        int64_t ld_dy, const void* d_w, int64_t ld_w, int64_t stride_w,
                                        const int32_t* d_offsets, void* d_dx, int64_t ld_dx, int dtype, void* stream) {
  if (int rc = check_grouped(rows, groups, k, m, d_offsets, dtype)) return rc;
  if (int rc = check_matrix("d_dy", d_dy, rows, m, ld_dy, dtype)) return rc;
  if (int rc = check_weights("d_w", d_w, groups, k, m, ld_w, stride_w, dtype, false)) return rc;
  if (int rc = check_matrix("d_dx", d_dx, rows, k, ld_dx, dtype)) return rc;
  const hpspmm::GroupedArgs g{rows, groups, (int32_t)k, (int32_t)m, d_offsets, d_dy, ld_dy, d_w, ld_w, stride_w, d_dx, ld_dx, 0, 0, 1, nullptr};
  return launch_grouped<hpspmm::kGradX>(g, dtype, dtype, (hipStream_t)stream);
}

HPSPMM_API int hpspmm_grouped_mm_grad_w(hpspmm_rows_plan* plan, int64_t rows, int64_t groups, int64_t k, int64_t m,
                                        const void* d_dy, int64_t ld_dy, const void* d_x, int64_t ld_x,
                                        const int32_t* d_offsets, void* d_dw, int64_t ld_dw, int64_t stride_dw,
                                        int dtype, int dw_type, int accumulate, void* stream) {
  if (int rc = check_grouped(rows, groups, k, m, d_offsets, dtype)) return rc;
  if (dw_type != dtype && dw_type != HPSPMM_F32)
    return fail(HPSPMM_ERR_INVALID_ARG, "the gradient of the weights has the operands' type or HPSPMM_F32, got %d", dw_type);
  if (int rc = check_matrix("d_dy", d_dy, rows, m, ld_dy, dtype)) return rc;
  if (int rc = check_matrix("d_x", d_x, rows, k, ld_x, dtype)) return rc;
  if (int rc = check_weights("d_dw", d_dw, groups, k, m, ld_dw, stride_dw, dw_type, true)) return rc;
  if (int rc = check_rows_plan(plan, 0, 0, 0)) return rc;
  const hpspmm::GroupedArgs g{rows, groups, (int32_t)k, (int32_t)m, d_offsets, d_dy, ld_dy, d_x, ld_x, 0, d_dw, ld_dw, stride_dw, accumulate != 0,
                              1, plan->d_split};
  return launch_grouped<hpspmm::kGradW>(g, dtype, dw_type, (hipStream_t)stream);
}
