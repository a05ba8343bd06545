// Entry points about rows selected by an id: embedding lookup, its gradient, rows sorted by id, and the plan that
// holds their workspace.
#include "row_ops.hpp"

#include "row_kernels.hpp"

using namespace hpspmm_host;

namespace hpspmm_host {

int check_matrix(const char* name, const void* p, int64_t rows, int64_t width, int64_t ld, int dtype) {
  if (width <= 0 || width > kMaxRowLength)
    return fail(HPSPMM_ERR_INVALID_ARG, "%s: rows must have 1 to 2^20 columns, got %lld", name, (long long)width);
  if (ld < width || ld > kMaxStride)
    return fail(HPSPMM_ERR_INVALID_ARG, "%s: leading dimension %lld with rows of %lld columns", name, (long long)ld,
                (long long)width);
  if (rows > 0 && !p) return fail(HPSPMM_ERR_INVALID_ARG, "%s is NULL", name);
  if (!aligned_to(p, dtype_size(dtype)))
    return fail(HPSPMM_ERR_INVALID_ARG, "%s is not at a multiple of its element size", name);
  return HPSPMM_OK;
}

int check_rows_plan(const hpspmm_rows_plan* plan, int64_t rows, int64_t ids, int64_t width) {
  if (!plan) return fail(HPSPMM_ERR_INVALID_ARG, "plan is NULL");
  if (rows > plan->max_rows || ids > plan->max_ids || width > plan->max_width)
    return fail(HPSPMM_ERR_INVALID_ARG,
                "the plan is for up to %lld rows, %lld ids and rows of %lld columns; asked for %lld, %lld, %lld",
                (long long)plan->max_rows, (long long)plan->max_ids, (long long)plan->max_width, (long long)rows,
                (long long)ids, (long long)width);
  int dev = 0;
  HPSPMM_HIP(hipGetDevice(&dev));
  if (dev != plan->device)
    return fail(HPSPMM_ERR_INVALID_ARG, "the plan lives on device %d, the current device is %d", plan->device, dev);
  return HPSPMM_OK;
}

}  // namespace hpspmm_host

namespace {

int check_ids(int64_t n, int64_t ids, const void* d_ids, int id_type) {
  if (n < 0 || ids < 0) return fail(HPSPMM_ERR_INVALID_ARG, "negative size (n=%lld ids=%lld)", (long long)n, (long long)ids);
  if (n >= INT32_MAX || ids >= INT32_MAX)
    return fail(HPSPMM_ERR_INVALID_ARG, "size exceeds the int32 index range (n=%lld ids=%lld)", (long long)n, (long long)ids);
  if (id_type != HPSPMM_I32 && id_type != HPSPMM_I64) return fail(HPSPMM_ERR_INVALID_ARG, "unknown id type %d", id_type);
  if (n > 0 && !d_ids) return fail(HPSPMM_ERR_INVALID_ARG, "d_ids is NULL");
  if (!aligned_to(d_ids, id_type == HPSPMM_I64 ? 8 : 4))
    return fail(HPSPMM_ERR_INVALID_ARG, "d_ids is not at a multiple of its element size");
  return HPSPMM_OK;
}

int key_bits(int64_t ids) {
  int bits = 1;
  while (bits < 32 && (ids >> bits) != 0) ++bits;
  return bits;
}

// The n rows sorted by id, ids outside [0, ids) last, rows of one id in increasing order: *cur = which of the plan's
// buffers holds them.
int sort_rows(hpspmm_rows_plan* plan, int64_t n, int64_t ids, const void* d_ids, int id_type, hipStream_t st, int* cur) {
  *cur = 0;
  if (n == 0) return HPSPMM_OK;
  dispatch_id(id_type, [&](auto id) {
    using Id = decltype(id);
    hipLaunchKernelGGL((hpspmm::row_keys_kernel<Id>), dim3((unsigned)ceil_div(n, hpspmm::kBlock)), dim3(hpspmm::kBlock), 0,
                       st, n, (uint32_t)ids, (const Id*)d_ids, plan->d_keys[0], plan->d_vals[0]);
    return HPSPMM_OK;
  });
  return radix_sort_pairs(n, plan->d_keys, plan->d_vals, plan->d_hist, plan->d_scan, key_bits(ids), st, cur);
}

}  // namespace

HPSPMM_API int hpspmm_rows_plan_create(int64_t max_rows, int64_t max_ids, int64_t max_width, hpspmm_rows_plan** plan_out) {
  if (!plan_out) return fail(HPSPMM_ERR_INVALID_ARG, "plan_out is NULL");
  *plan_out = nullptr;
  if (max_rows < 0 || max_ids < 0 || max_width < 0 || max_rows >= INT32_MAX || max_ids >= INT32_MAX || max_width > kMaxRowLength)
    return fail(HPSPMM_ERR_INVALID_ARG, "bad plan size (max_rows=%lld max_ids=%lld max_width=%lld)", (long long)max_rows,
                (long long)max_ids, (long long)max_width);
  int dev = 0;
  HPSPMM_HIP(hipGetDevice(&dev));
  hpspmm_rows_plan* p = new (std::nothrow) hpspmm_rows_plan;
  if (!p) return fail(HPSPMM_ERR_ALLOC, "out of host memory");
  p->device = dev;
  p->max_rows = max_rows;
  p->max_ids = max_ids;
  p->max_width = max_width;
  const int64_t n = std::max<int64_t>(max_rows, 1), tiles = ceil_div(n, sort_tile());
  const int64_t hist = 256 * tiles + 1, scan = scan_scratch_words(256 * tiles);
  const int64_t words[] = {n, n, n, n, hist, scan};
  int64_t bytes = 0;
  for (int64_t w : words) bytes += (w * 4 + 255) & ~(int64_t)255;
  if (hipMalloc((void**)&p->arena, (size_t)bytes) != hipSuccess) {
    (void)hipGetLastError();
    delete p;
    return fail(HPSPMM_ERR_ALLOC, "device allocation of %lld bytes for the plan failed", (long long)bytes);
  }
  p->workspace_bytes = bytes;
  char* at = p->arena;
  auto take = [&](int64_t w) {
    char* q = at;
    at += (w * 4 + 255) & ~(int64_t)255;
    return q;
  };
  p->d_keys[0] = (uint32_t*)take(n);
  p->d_keys[1] = (uint32_t*)take(n);
  p->d_vals[0] = (int32_t*)take(n);
  p->d_vals[1] = (int32_t*)take(n);
  p->d_hist = (uint32_t*)take(hist);
  p->d_scan = (uint32_t*)take(scan);
  *plan_out = p;
  return HPSPMM_OK;
}

HPSPMM_API int hpspmm_rows_plan_destroy(hpspmm_rows_plan* plan) {
  if (!plan) return HPSPMM_OK;
  const hipError_t e = hipFree(plan->arena);
  delete plan;
  if (e != hipSuccess) return fail(HPSPMM_ERR_HIP, "hipFree: %s", hipGetErrorString(e));
  return HPSPMM_OK;
}

HPSPMM_API int hpspmm_embedding_lookup(int64_t n, int64_t vocab, int64_t width, const void* d_ids, int id_type,
                                       const void* d_table, int64_t ld_table, int dtype, float scale, void* d_out,
                                       int64_t ld_out, void* stream) {
  if (int rc = check_ids(n, vocab, d_ids, id_type)) return rc;
  if (!known_dtype(dtype)) return fail(HPSPMM_ERR_INVALID_ARG, "unknown element type %d", dtype);
  if (int rc = check_matrix("d_table", d_table, vocab, width, ld_table, dtype)) return rc;
  if (int rc = check_matrix("d_out", d_out, n, width, ld_out, dtype)) return rc;
  if (n == 0) return HPSPMM_OK;
  hipStream_t st = (hipStream_t)stream;
  const int64_t size = dtype_size(dtype), per16 = 16 / size;
  const bool aligned = aligned_to(d_table, 16) && aligned_to(d_out, 16) && ld_table % per16 == 0 && ld_out % per16 == 0;
  const int64_t vecs = ceil_div(width, per16);
  int tpr_log2 = 0;
  while (tpr_log2 < 8 && ((int64_t)1 << tpr_log2) < vecs) ++tpr_log2;
  const int64_t col_tiles = ceil_div(vecs, (int64_t)1 << tpr_log2);
  const int64_t per_pass = hpspmm::kBlock >> tpr_log2;
  const bool many = n * col_tiles >= 4 * per_pass * 1024;
  const int64_t blocks = ceil_div(n, per_pass * (many ? 4 : 1));
  dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return dispatch_id(id_type, [&](auto id) {
      using Id = decltype(id);
      auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)col_tiles), dim3(hpspmm::kBlock), 0, st, n, (uint32_t)vocab,
                           (int32_t)width, tpr_log2, (const Id*)d_ids, (const T*)d_table, ld_table, scale, (T*)d_out, ld_out);
      };
      if (aligned) {
        if (many) launch(hpspmm::embedding_lookup_kernel<T, Id, true, 4>);
        else launch(hpspmm::embedding_lookup_kernel<T, Id, true, 1>);
      } else {
        if (many) launch(hpspmm::embedding_lookup_kernel<T, Id, false, 4>);
        else launch(hpspmm::embedding_lookup_kernel<T, Id, false, 1>);
      }
      return HPSPMM_OK;
    });
  });
  HPSPMM_HIP(hipGetLastError());
  return HPSPMM_OK;
}

HPSPMM_API int hpspmm_group_rows(hpspmm_rows_plan* plan, int64_t n, int64_t groups, const void* d_ids, int id_type,
                                 int32_t* d_order, int32_t* d_offsets, void* stream) {
  if (int rc = check_ids(n, groups, d_ids, id_type)) return rc;
  if ((n > 0 && !d_order) || !d_offsets) return fail(HPSPMM_ERR_INVALID_ARG, "d_order or d_offsets is NULL");
  if (!aligned_to(d_order, 4) || !aligned_to(d_offsets, 4))
    return fail(HPSPMM_ERR_INVALID_ARG, "d_order or d_offsets is not at a multiple of 4 bytes");
  if (int rc = check_rows_plan(plan, n, groups, 0)) return rc;
  hipStream_t st = (hipStream_t)stream;
  int cur = 0;
  if (int rc = sort_rows(plan, n, groups, d_ids, id_type, st, &cur)) return rc;
  hipLaunchKernelGGL(hpspmm::row_offsets_kernel, dim3((unsigned)ceil_div(std::max(n, groups + 1), hpspmm::kBlock)),
                     dim3(hpspmm::kBlock), 0, st, n, groups, plan->d_keys[cur], plan->d_vals[cur], d_order, d_offsets);
  HPSPMM_HIP(hipGetLastError());
  return HPSPMM_OK;
}

HPSPMM_API int hpspmm_embedding_grad(hpspmm_rows_plan* plan, int64_t n, int64_t vocab, int64_t width, const void* d_ids,
                                     int id_type, const void* d_grad, int64_t ld_grad, int grad_type, float scale,
                                     void* d_table, int64_t ld_table, int table_type, int accumulate, void* stream) {
  if (int rc = check_ids(n, vocab, d_ids, id_type)) return rc;
  if (!known_dtype(grad_type) || !known_dtype(table_type))
    return fail(HPSPMM_ERR_INVALID_ARG, "unknown element type %d or %d", grad_type, table_type);
  if (int rc = check_matrix("d_grad", d_grad, n, width, ld_grad, grad_type)) return rc;
  if (int rc = check_matrix("d_table", d_table, vocab, width, ld_table, table_type)) return rc;
  if (int rc = check_rows_plan(plan, n, vocab, width)) return rc;
  if (vocab == 0 || (n == 0 && accumulate)) return HPSPMM_OK;
  hipStream_t st = (hipStream_t)stream;
  int cur = 0;
  if (int rc = sort_rows(plan, n, vocab, d_ids, id_type, st, &cur)) return rc;
  dispatch_dtype(grad_type, [&](auto t) {
    using T = decltype(t);
    return dispatch_dtype(table_type, [&](auto o) {
      using TO = decltype(o);
      hipLaunchKernelGGL((hpspmm::embedding_grad_kernel<T, TO>),
                         dim3((unsigned)vocab, (unsigned)std::min<int64_t>(ceil_div(width, hpspmm::kBlock), 64)),
                         dim3(hpspmm::kBlock), 0, st, n, (int32_t)width, plan->d_keys[cur], plan->d_vals[cur],
                         (const T*)d_grad, ld_grad, scale, (TO*)d_table, ld_table, accumulate);
      return HPSPMM_OK;
    });
  });
  HPSPMM_HIP(hipGetLastError());
  return HPSPMM_OK;
}
