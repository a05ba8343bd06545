// Entry points of the products grouped by expert.
#include "row_ops.hpp"

#include "grouped_kernels.hpp"

using namespace hpspmm_host;

namespace {

// Groups are a grid dimension of the gradient of the weights.
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

template <int kMode>
int launch_grouped(const hpspmm::GroupedArgs& g, int dtype, int out_type, hipStream_t st) {
  const int64_t n_out = kMode == hpspmm::kForward ? g.m : g.k;
  const unsigned nt = (unsigned)ceil_div(n_out, hpspmm::kSimpleTile);
  const dim3 grid = kMode == hpspmm::kGradW
                        ? dim3((unsigned)ceil_div(g.m, hpspmm::kSimpleTile), nt, (unsigned)g.groups)
                        : dim3((unsigned)most_row_tiles(g.rows, g.groups, hpspmm::kSimpleTile), nt, 1);
  if (grid.x == 0 || grid.z == 0) return HPSPMM_OK;
  dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return dispatch_dtype(out_type, [&](auto o) {
      using TO = decltype(o);
      if constexpr (std::is_same_v<T, TO> || (kMode == hpspmm::kGradW && std::is_same_v<TO, float>))
        hipLaunchKernelGGL((hpspmm::grouped_simple_kernel<T, TO, kMode>), grid, dim3(hpspmm::kBlock), 0, st, g);
      return HPSPMM_OK;
    });
  });
  HPSPMM_HIP(hipGetLastError());
  return HPSPMM_OK;
}

}  // namespace

HPSPMM_API int hpspmm_grouped_mm(int64_t rows, int64_t groups, int64_t k, int64_t m, const void* d_x, int64_t ld_x,
                                 const void* d_w, int64_t ld_w, int64_t stride_w, const int32_t* d_offsets, void* d_y,
                                 int64_t ld_y, int dtype, void* stream) {
  if (int rc = check_grouped(rows, groups, k, m, d_offsets, dtype)) return rc;
  if (int rc = check_matrix("d_x", d_x, rows, k, ld_x, dtype)) return rc;
  if (int rc = check_weights("d_w", d_w, groups, k, m, ld_w, stride_w, dtype, false)) return rc;
  if (int rc = check_matrix("d_y", d_y, rows, m, ld_y, dtype)) return rc;
  const hpspmm::GroupedArgs g{rows, groups, (int32_t)k, (int32_t)m, d_offsets, d_x, ld_x, d_w, ld_w, stride_w, d_y, ld_y, 0, 0};
  return launch_grouped<hpspmm::kForward>(g, dtype, dtype, (hipStream_t)stream);
}

HPSPMM_API int hpspmm_grouped_mm_grad_x(int64_t rows, int64_t groups, int64_t k, int64_t m, const void* d_dy,
                                        int64_t ld_dy, const void* d_w, int64_t ld_w, int64_t stride_w,
                                        const int32_t* d_offsets, void* d_dx, int64_t ld_dx, int dtype, void* stream) {
  if (int rc = check_grouped(rows, groups, k, m, d_offsets, dtype)) return rc;
  if (int rc = check_matrix("d_dy", d_dy, rows, m, ld_dy, dtype)) return rc;
  if (int rc = check_weights("d_w", d_w, groups, k, m, ld_w, stride_w, dtype, false)) return rc;
  if (int rc = check_matrix("d_dx", d_dx, rows, k, ld_dx, dtype)) return rc;
  const hpspmm::GroupedArgs g{rows, groups, (int32_t)k, (int32_t)m, d_offsets, d_dy, ld_dy, d_w, ld_w, stride_w, d_dx, ld_dx, 0, 0};
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
  const hpspmm::GroupedArgs g{rows, groups, (int32_t)k, (int32_t)m, d_offsets, d_dy, ld_dy, d_x, ld_x, 0, d_dw, ld_dw, stride_dw, accumulate != 0};
  return launch_grouped<hpspmm::kGradW>(g, dtype, dw_type, (hipStream_t)stream);
}
