// Entry points about rows selected by an id: embedding lookup, its gradient, rows sorted by id, and the plan that
// holds their workspace.
#include "row_ops.hpp"

#include "grouped_kernels.hpp"
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

// Digits of the counting sort for ids below `ids` (and the key `ids` itself): how many, of how many bits each.
void key_digits(int64_t ids, int* digits, int* bits) {
  const int all = key_bits(ids);
  *digits = (int)ceil_div(all, hpspmm::kDigitBits);
  *bits = (int)ceil_div(all, *digits);
}

// The n rows sorted by id, ids outside [0, ids) last, rows of one id in increasing order, in d_keys / d_vals
// (hpspmm_group_rows: the rows straight to d_order, and the groups' offsets; keys are then kept only where it needs them).
struct Sorted {
  const uint32_t* keys;
  const int32_t* rows;
};
// The rows of a table that become zeros, cut into stretches for launches to come.
struct ZeroRows {
  char* at = nullptr;
  int64_t rows = 0, bytes = 0, last = 0, pitch = 0;
  ZeroRows() = default;
  ZeroRows(void* table, int64_t n, int64_t row_bytes, int64_t row_pitch)
      : at((char*)table), rows(n), bytes(row_bytes), last(row_bytes), pitch(row_pitch) {
    if (row_bytes == row_pitch && n > 0) {  // one stretch of memory, in pieces of 16 KB
      const int64_t all = n * row_bytes;
      bytes = pitch = 16384;
      rows = ceil_div(all, bytes);
      last = all - (rows - 1) * bytes;
    }
  }
  // The next of `left` stretches, for a launch of `first` workgroups of `threads` threads; *grid = the workgroups in all.
  hpspmm::ZeroFill next(int64_t first, int left, int threads, unsigned* grid) {
    const int64_t share = ceil_div(rows, left);
    hpspmm::ZeroFill z{at, share, bytes, share == rows ? last : bytes, pitch, (unsigned)first, 0, 4, 0};
    at += share * pitch;
    rows -= share;
    const int64_t apart = (int64_t)(uintptr_t)z.at | z.pitch;
    z.unit_log2 = apart % 16 == 0 ? 4 : apart % 4 == 0 ? 2 : 1;
    // four stores a thread
    while ((1 << z.tpr_log2) < threads && ((int64_t)4 << (z.tpr_log2 + z.unit_log2)) < bytes) ++z.tpr_log2;
    z.blocks = (unsigned)std::min<int64_t>(ceil_div(share << z.tpr_log2, threads), 4096);
    *grid = (unsigned)first + z.blocks;
    return z;
  }
};

int sort_rows(hpspmm_rows_plan* plan, int64_t n, int64_t ids, const void* d_ids, int id_type, int32_t* d_order,
              int32_t* d_offsets, ZeroRows zero, hipStream_t st, Sorted* out) {
  using namespace hpspmm;
  unsigned grid = 0;
  if (out) *out = {plan->d_keys[0], plan->d_vals[0]};
  const int64_t n_offsets = d_offsets ? ids + 1 : 0;
  auto offsets_of = [&](const uint32_t* keys) {
    hipLaunchKernelGGL(row_offsets_kernel, dim3((unsigned)ceil_div(n_offsets, kBlock)), dim3(kBlock), 0, st, n, ids, keys,
                       d_offsets);
  };
  int digits, bits;
  key_digits(ids, &digits, &bits);
  // Counting ranks is one launch of n^2 steps, digits are two dependent launches each.  64 ids (one digit), ranks / digits:
  // 4096 rows 7.9 / 9.9 us, 8192 rows 13.0 / 10.4; 131072 ids (two digits), with the sums of a gradient behind them: 512
  // rows 12 / 24 us, 8192 rows 28 / 41, 16384 rows 46 / 48.
  if (n <= (digits == 1 ? 6144 : kRankMaxRows)) {
    // few groups are counted along as if they were rows, many found in the sorted keys
    const bool counted = n_offsets <= 4 * kRankMaxRows;
    const int64_t count = n + (counted ? n_offsets : 0);
    if (count > 0 || zero.rows > 0) {
      const ZeroFill z = zero.next(ceil_div(count, 64), 1, 64 * kRankWaves, &grid);
      dispatch_id(id_type, [&](auto id) {
        using Id = decltype(id);
        hipLaunchKernelGGL((row_rank_kernel<Id>), dim3(grid), dim3(64 * kRankWaves), 0, st, (int32_t)n,
                           counted ? (int32_t)n_offsets : 0, (uint32_t)ids, (const Id*)d_ids,
                           d_order && counted ? nullptr : plan->d_keys[0], d_order ? d_order : plan->d_vals[0], d_offsets, z);
        return HPSPMM_OK;
      });
    }
    if (!counted) offsets_of(plan->d_keys[0]);
    return HPSPMM_OK;
  }
  const int64_t tiles = ceil_div(n, kDigitTile);
  const bool fused = tiles <= kDigitFused;
  // offsets come with the only digit, or from the sorted keys
  const bool with_offsets = d_offsets && digits == 1 && fused;
  for (int p = 0; p < digits; ++p) {
    const int shift = p * bits, from = (p + 1) & 1, to = p & 1;
    const bool last = p + 1 == digits;
    int rc = dispatch_id(id_type, [&](auto id) {
      using Id = decltype(id);
      const RowKeys<Id> rows{p == 0 ? (const Id*)d_ids : nullptr, plan->d_keys[from], plan->d_vals[from], (uint32_t)ids};
      ZeroFill z = zero.next(tiles, 2 * (digits - p), kDigitThreads, &grid);
      hipLaunchKernelGGL((digit_count_kernel<Id>), dim3(grid), dim3(kDigitThreads), 0, st, n, rows, shift, bits,
                         tiles, fused ? 0 : 1, plan->d_hist, z);
      if (!fused)
        if (int e = exclusive_scan_u32(plan->d_hist, plan->d_hist, tiles << bits, st, plan->d_scan)) return e;
      z = zero.next(tiles, 2 * (digits - p) - 1, kDigitThreads, &grid);
      hipLaunchKernelGGL((digit_scatter_kernel<Id>), dim3(grid), dim3(kDigitThreads), 0, st, n, rows, shift, bits,
                         tiles, fused ? 0 : 1, plan->d_hist, last && d_order && with_offsets ? nullptr : plan->d_keys[to],
                         last && d_order ? d_order : plan->d_vals[to], ids, with_offsets ? d_offsets : nullptr, z);
      return (int)HPSPMM_OK;
    });
    if (rc) return rc;
  }
  const int at = (digits + 1) & 1;
  if (d_offsets && !with_offsets) offsets_of(plan->d_keys[at]);
  if (out) *out = {plan->d_keys[at], plan->d_vals[at]};
  return HPSPMM_OK;
}

// Shape of the sums of a gradient with rows of `width` columns, `per16` of which a thread owns.
struct SumShape {
  int tpr_log2, chunk_log2;
  int64_t col_tiles, chunks, pitch;
};
constexpr int kMinChunkLog2 = 2, kMaxChunkLog2 = 7;
// (a launch holds fewer than 2^32 threads: 2^24 - 1 workgroups, some of which fill rows with zeros beside the sums)
constexpr int64_t kMostChunks = ((int64_t)1 << 24) - ((int64_t)1 << 21);
SumShape sum_shape(int64_t n, int64_t width, int64_t per16) {
  SumShape s{};
  const int64_t vecs = ceil_div(width, per16);
  while (s.tpr_log2 < 8 && ((int64_t)1 << s.tpr_log2) < vecs) ++s.tpr_log2;
  s.col_tiles = ceil_div(vecs, (int64_t)1 << s.tpr_log2);
  // chunks as long as leaves 1024 of them a column tile, at most 128 rows
  s.chunk_log2 = kMinChunkLog2;
  while (s.chunk_log2 < kMaxChunkLog2 && (n * s.col_tiles) >> (s.chunk_log2 + 1) >= 1024) ++s.chunk_log2;
  while (ceil_div(n, (int64_t)1 << s.chunk_log2) > kMostChunks) ++s.chunk_log2;
  if (n <= 32) s.chunk_log2 = 5;  // one chunk: no sum crosses it, one launch less
  s.chunks = ceil_div(n, (int64_t)1 << s.chunk_log2);
  s.pitch = ceil_div(width, 8) * 8;
  return s;
}
// Carry floats that any n <= rows, width <= columns can need.
int64_t most_carry_floats(int64_t rows, int64_t columns) {
  if (rows == 0 || columns == 0) return 0;
  // a column tile has at most 2048 columns; chunks * tiles stays below 4096 (+ one chunk) until chunks are at their longest
  const int64_t tiles = ceil_div(columns, 4 * hpspmm::kBlock), pitch = ceil_div(columns, 8) * 8;
  const int64_t by_rows = 2 * ceil_div(rows, (int64_t)1 << kMinChunkLog2) * pitch;
  const int64_t by_tiles = 2 * 2048 * (std::max<int64_t>(4096, (rows * tiles) >> kMaxChunkLog2) + tiles + 1);
  return std::min(by_rows, by_tiles);
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
  int digits, bits;
  key_digits(max_ids, &digits, &bits);
  const int64_t n = std::max<int64_t>(max_rows, 1), tiles = ceil_div(n, hpspmm::kDigitTile);
  // (fewer ids may make a digit of more bits)
  const int64_t hist = tiles << std::min<int>(hpspmm::kDigitBits, key_bits(max_ids)), scan = scan_scratch_words(hist);
  const int64_t carry = most_carry_floats(max_rows, max_width);
  const int64_t split = hpspmm::kSplitTiles * hpspmm::kSplitEdge * hpspmm::kSplitEdge;
  const int64_t words[] = {n, n, n, n, hist, scan, carry, split};
  int64_t bytes = 0;
  for (int64_t w : words) bytes += (w * 4 + 255) & ~(int64_t)255;
  if (hipMalloc((void**)&p->arena, (size_t)bytes) != hipSuccess) {
    (void)hipGetLastError();
    delete p;
    return fail(HPSPMM_ERR_ALLOC, "device allocation of %lld bytes for the plan failed", (long long)bytes);
  }
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
  p->d_carry = (float*)take(carry);
  p->carry_floats = carry;
  p->d_split = (float*)take(split);
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
  const bool past_caches = aligned && many && n * width * size >= hpspmm::kStreamBytes && aligned_to(d_out, 128) && ld_out * size % 128 == 0;
  // (a launch holds fewer than 2^32 threads: 2^23 workgroups at a time)
  const int64_t per_block = per_pass * (many ? 4 : 1), per_launch = per_block << 23;
  dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return dispatch_id(id_type, [&](auto id) {
      using Id = decltype(id);
      auto launch = [&](auto kernel) {
        for (int64_t r = 0; r < n; r += per_launch) {
          const int64_t rows = std::min(per_launch, n - r);
          hipLaunchKernelGGL(kernel, dim3((unsigned)ceil_div(rows, per_block), (unsigned)col_tiles), dim3(hpspmm::kBlock), 0, st,
                             rows, (uint32_t)vocab, (int32_t)width, tpr_log2, (const Id*)d_ids + r, (const T*)d_table, ld_table,
                             scale, (T*)d_out + r * ld_out, ld_out);
        }
      };
      using hpspmm::embedding_lookup_kernel;
      if (past_caches) launch(embedding_lookup_kernel<T, Id, true, 4, true>);
      else if (aligned && many) launch(embedding_lookup_kernel<T, Id, true, 4, false>);
      else if (aligned) launch(embedding_lookup_kernel<T, Id, true, 1, false>);
      else if (many) launch(embedding_lookup_kernel<T, Id, false, 4, false>);
      else launch(embedding_lookup_kernel<T, Id, false, 1, false>);
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
  if (int rc = sort_rows(plan, n, groups, d_ids, id_type, d_order, d_offsets, ZeroRows{}, (hipStream_t)stream, nullptr)) return rc;
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
  const int64_t grad_size = dtype_size(grad_type), table_size = dtype_size(table_type);
  // Rows that no id points at become zeros either in the launches of the sort, which leave most of the chip idle but know
  // of no row yet (so every row is filled), or beside the sums, where the rows that get one are left out.  The first hides
  // the sort behind the fill and writes the rows that get a sum twice.  Early / late, 2048 columns bf16 -> bf16, as many ids
  // as rows of the table, frequencies of natural text or even ones: 64 MB of rows 58 / 65 or 59 / 62 us, 128 MB 97 / 99 or
  // 104 / 98, 192 MB 136 / 138 or 143 / 132, 256 MB 170 / 170 or 177 / 160, 512 MB 285 / 274 or 312 / 270, 1 GB 531 / 495 or
  // 603 / 505; a fourth as many ids as rows of the table: 64 MB 89 / 110 or 89 / 105, 128 MB 165 / 180 or 171 / 176, 192 MB
  // 239 / 252 or 249 / 245, 256 MB 307 / 310 or 320 / 302, 512 MB 582 / 554 or 624 / 561.  (1000 ids, 50001 x 771 f32 28 / 36;
  // more ids than rows, 262144 over 32768 x 1024 f32: 208 / 196.)
  const bool early = !accumulate && n <= vocab && n * width * table_size <= (int64_t)192 << 20;
  const ZeroRows zero = early ? ZeroRows(d_table, vocab, width * table_size, ld_table * table_size) : ZeroRows();
  const SumShape s = sum_shape(n, width, 16 / grad_size);
  if (2 * s.chunks * s.pitch > plan->carry_floats) return fail(HPSPMM_ERR_INVALID_ARG, "the plan's workspace is too small");
  Sorted sorted{};
  if (int rc = sort_rows(plan, n, vocab, d_ids, id_type, nullptr, nullptr, zero, st, &sorted)) return rc;
  const int64_t per_block = s.tpr_log2 < 6 ? hpspmm::kBlock >> s.tpr_log2 : 1;
  const int64_t sum_blocks = ceil_div(s.chunks, per_block);
  const int64_t zero_blocks = accumulate || early ? 0 : std::min<int64_t>(ceil_div(vocab, hpspmm::kZeroRows), 1 << 20);
  const unsigned threads = s.tpr_log2 < 6 ? hpspmm::kBlock : 1u << s.tpr_log2;
  const bool whole = aligned_to(d_grad, 16) && aligned_to(d_table, 16) && ld_grad * grad_size % 16 == 0 &&
                     ld_table * table_size % 16 == 0 && width * grad_size % 16 == 0;
  const hpspmm::SumArgs g{n, (uint32_t)vocab, (int32_t)width, (int32_t)s.pitch, sorted.keys, sorted.rows, d_grad, ld_grad, scale,
                          d_table, ld_table, accumulate != 0, plan->d_carry, s.chunk_log2, s.tpr_log2, s.chunks, (unsigned)sum_blocks,
                          (unsigned)zero_blocks};
  const dim3 fix_grid((unsigned)s.chunks, (unsigned)ceil_div(width, 256));
  dispatch_dtype(table_type, [&](auto o) {
    using TO = decltype(o);
    if (sum_blocks + zero_blocks > 0) dispatch_dtype(grad_type, [&](auto t) {
      using T = decltype(t);
      auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)(sum_blocks + zero_blocks), (unsigned)s.col_tiles), dim3(threads), 0, st, g);
      };
      using hpspmm::embedding_sum_kernel;
      if (width < 16 / grad_size) launch(embedding_sum_kernel<T, TO, hpspmm::kRowShort, false>);
      else if (s.tpr_log2 >= 6 && whole) launch(embedding_sum_kernel<T, TO, hpspmm::kRowWhole, true>);
      else if (s.tpr_log2 >= 6) launch(embedding_sum_kernel<T, TO, hpspmm::kRowLoose, true>);
      else if (whole) launch(embedding_sum_kernel<T, TO, hpspmm::kRowWhole, false>);
      else launch(embedding_sum_kernel<T, TO, hpspmm::kRowLoose, false>);
      return HPSPMM_OK;
    });
    if (s.chunks > 1) {
      if (whole) hipLaunchKernelGGL((hpspmm::embedding_fix_kernel<TO, true>), fix_grid, dim3(hpspmm::kBlock), 0, st, g);
      else hipLaunchKernelGGL((hpspmm::embedding_fix_kernel<TO, false>), fix_grid, dim3(hpspmm::kBlock), 0, st, g);
    }
    return HPSPMM_OK;
  });
  HPSPMM_HIP(hipGetLastError());
  return HPSPMM_OK;
}
