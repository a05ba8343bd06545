// Kernels of the embedding lookup, of its gradient and of the rows sorted by id.
#pragma once

#include "row_types.hpp"
#include "spmm_kernels.hpp"

namespace hpspmm {

// out[i, :] = scale * table[ids[i], :], rows of zeros for ids outside the table: one product in 32 bits, rounded once.
// Bound by the bytes, n rows read and n written.  A thread owns 16 bytes of a row; 2^tpr_log2 adjacent threads share a
// row's column tile, a workgroup covers kRows rows one after the other, all of whose loads are in flight together.
// kStream: large outputs go past the caches, which they do not fit (32768 rows of 4096 bf16 over 131072, 12651 different
// ones: 87 -> 81 us, 4.6 TB/s of different rows and output; 85 -> 63 us where the same rows come again and stay in the
// caches).  16 rows of 1024 take 7 us from Python, half of it the launch.
template <class T, class Id, bool kAligned, int kRows, bool kStream>
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
      if (row >= n) continue;
      if constexpr (kStream) stream_n<kAligned, T, V>(out + row * ld_out + col, v[r]);
      else store_n<kAligned, T, V>(out + row * ld_out + col, v[r]);
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

// Rows of zeros, for the launches that have workgroups to spare: rows [0, rows) of `bytes` bytes (the last one of
// `last`), `pitch` bytes apart, by `blocks` workgroups from workgroup `first` on, 2^tpr_log2 threads a row.  An all-zero
// word is a zero of every element type.  A quarter of 131072 x 2048 bf16 with each launch of a sort: 21 us, 6.4 TB/s.
struct ZeroFill {
  char* at;
  int64_t rows, bytes, last, pitch;
  unsigned first, blocks;
  int unit_log2, tpr_log2;  // bytes of a store: 16, 4 or 2; address and pitch are multiples of it
};
template <class U>
__device__ __forceinline__ void fill_units(const ZeroFill& z) {
  const int per_block = (int)blockDim.x >> z.tpr_log2, tpr = 1 << z.tpr_log2;
  const U zero{};
  for (int64_t r = (int64_t)(blockIdx.x - z.first) * per_block + ((int)threadIdx.x >> z.tpr_log2); r < z.rows;
       r += (int64_t)z.blocks * per_block) {
    char* row = z.at + r * z.pitch;
    const int64_t bytes = r + 1 == z.rows ? z.last : z.bytes;
    const int64_t units = bytes >> z.unit_log2;
    const int t = (int)threadIdx.x & (tpr - 1);
#pragma unroll 4
    for (int64_t u = t; u < units; u += tpr) ((U*)row)[u] = zero;
    if (t == 0)
#pragma unroll 1
      for (int64_t b = units << z.unit_log2; b < bytes; b += 2) *(uint16_t*)(row + b) = 0;
  }
}
__device__ __forceinline__ void zero_fill(const ZeroFill& z) {
  if (z.unit_log2 == 4) fill_units<uint4>(z);
  else if (z.unit_log2 == 2) fill_units<uint32_t>(z);
  else fill_units<uint16_t>(z);
}

// ---------------------------------------------------------------------------------------------
// Rows sorted by id: keys[q] / vals[q] = id and row of the q-th row in that order, rows of one id in increasing order,
// ids outside [0, ids) as key `ids` behind all others.
// ---------------------------------------------------------------------------------------------

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

// offsets[g] = rows whose key is below g, g = 0 ... groups.
HPSPMM_KERNEL __launch_bounds__(kBlock) void row_offsets_kernel(int64_t n, int64_t groups,
                                                             const uint32_t* __restrict__ keys,
                                                             int32_t* __restrict__ offsets) {
  const int64_t g = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (g <= groups) offsets[g] = (int32_t)lower_bound_u32(keys, n, (uint32_t)g);
}

// Few rows: the place of a row is the number of rows before it, counted - n^2 comparisons, but one launch and no step
// that waits for another (512 rows, 16 groups: 4 us on the device).  Bound by the comparisons, 2 instructions each.  A workgroup places 64 rows, one a lane; its 16 wavefronts count in a sixteenth of the rows
// each, which they hold in LDS.  Rows n ... n + virtual - 1 are the group numbers 0 ...: their place is their offset.
constexpr int kRankWaves = 16;
constexpr int kRankMaxRows = 16384;
template <class Id>
__global__ __launch_bounds__(64 * kRankWaves) void row_rank_kernel(int32_t n, int32_t n_virtual, uint32_t ids,
                                                                  const Id* __restrict__ id, uint32_t* __restrict__ keys,
                                                                  int32_t* __restrict__ vals,
                                                                  int32_t* __restrict__ offsets, ZeroFill zero) {
  if (blockIdx.x >= zero.first) return zero_fill(zero);
  __shared__ __attribute__((aligned(16))) uint32_t s_key[kRankMaxRows];
  __shared__ int32_t s_count[kRankWaves][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int i0 = blockIdx.x * 64, i = i0 + lane;
  const bool real = i < n;
  const uint32_t key = real ? id_key(id[i], ids) : (uint32_t)(i - n);
  // tiles of 64 rows, dealt to the wavefronts in stretches
  const int tiles = (n + 63) / 64, per = (tiles + kRankWaves - 1) / kRankWaves;
  const int first = wave * per, last = min(first + per, tiles);
  uint32_t* mine = s_key + wave * per * 64;
  for (int t = first; t < last; ++t) {
    const int j = t * 64 + lane;
    mine[(t - first) * 64 + lane] = j < n ? id_key(id[j], ids) : 0xFFFFFFFFu;
  }
  // (a wavefront reads what it has written itself: no barrier)
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  int count = 0;
  for (int t = first; t < last; ++t) {
    const uint4* at = reinterpret_cast<const uint4*>(mine + (t - first) * 64);
    const int j0 = t * 64;
    if (j0 == i0 && real) {
#pragma unroll 4
      for (int q = 0; q < 16; ++q) {
        const uint4 v = at[q];
        count += v.x < key + (uint32_t)(q * 4 + 0 < lane);
        count += v.y < key + (uint32_t)(q * 4 + 1 < lane);
        count += v.z < key + (uint32_t)(q * 4 + 2 < lane);
        count += v.w < key + (uint32_t)(q * 4 + 3 < lane);
      }
    } else {
      // rows of the same id count where they lie before this one
      const uint32_t below = key + (uint32_t)(real && j0 < i0);
#pragma unroll 4
      for (int q = 0; q < 16; ++q) {
        const uint4 v = at[q];
        count += v.x < below;
        count += v.y < below;
        count += v.z < below;
        count += v.w < below;
      }
    }
  }
  s_count[wave][lane] = count;
  __syncthreads();
  if (wave != 0) return;
  count = 0;
#pragma unroll
  for (int w = 0; w < kRankWaves; ++w) count += s_count[w][lane];
  if (real) {
    if (keys) keys[count] = key;
    vals[count] = i;
  } else if (i - n < n_virtual) {
    offsets[i - n] = count;
  }
}

// Many rows: stable counting sort by digits of up to 10 bits, least significant first, two launches a digit: counts per
// tile of rows, then the rows to their places.  A tile's rows go to the wavefronts in stretches of 4 x 64; a row's rank
// among the equal digits of its stretch is found by ballots over the digit's bits.  Bound by the chain of its steps: keys,
// counts of the other tiles, places, rows.  524288 rows, 64 groups: 3 + 10 us, 0.5 TB/s (three kernels a digit of 8 bits,
// with a scan between counts and places: 37 us).  Ten bits a digit let 2^20 ids do with two.
constexpr int kDigitBits = 10, kDigitBins = 1 << kDigitBits;
constexpr int kDigitThreads = 1024, kDigitWaves = kDigitThreads / 64, kDigitRounds = 4;
constexpr int kDigitTile = kDigitThreads * kDigitRounds;
constexpr int kDigitFused = 256;  // up to so many tiles every workgroup adds up the counts of the others itself

// The key of row i of this pass: from the ids in the first one.
template <class Id>
struct RowKeys {
  const Id* id;          // first pass
  const uint32_t* keys;  // later ones
  const int32_t* vals;
  uint32_t ids;
  __device__ __forceinline__ uint32_t key(int64_t i) const { return id ? id_key(id[i], ids) : keys[i]; }
  __device__ __forceinline__ int32_t val(int64_t i) const { return id ? (int32_t)i : vals[i]; }
};

// hist[tile * bins + d] (or hist[d * tiles + tile], for a scan over all of it) = rows of the tile with digit d.
template <class Id>
__global__ __launch_bounds__(kDigitThreads) void digit_count_kernel(int64_t n, RowKeys<Id> rows, int shift, int bits,
                                                                   int64_t tiles, int by_digit, uint32_t* __restrict__ hist,
                                                                   ZeroFill zero) {
  if (blockIdx.x >= zero.first) return zero_fill(zero);
  __shared__ uint32_t s_hist[kDigitBins];
  const int bins = 1 << bits;
  for (int d = threadIdx.x; d < bins; d += kDigitThreads) s_hist[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kDigitTile;
#pragma unroll
  for (int q = 0; q < kDigitRounds; ++q) {
    const int64_t i = base + q * kDigitThreads + threadIdx.x;
    if (i < n) atomicAdd(&s_hist[(rows.key(i) >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kDigitThreads)
    hist[by_digit ? (int64_t)d * tiles + blockIdx.x : (int64_t)blockIdx.x * bins + d] = s_hist[d];
}

// Row i of the tile goes to (rows with a lower digit) + (rows of the tiles before with this digit) + (its rank in the
// tile).  scanned: hist holds the first two sums already; otherwise they are added up here.  offsets (only when one
// digit is all there is): offsets[d] = rows with a digit below d, by the first workgroup.
template <class Id>
__global__ __launch_bounds__(kDigitThreads) void digit_scatter_kernel(int64_t n, RowKeys<Id> rows, int shift, int bits,
                                                                     int64_t tiles, int scanned,
                                                                     const uint32_t* __restrict__ hist,
                                                                     uint32_t* __restrict__ keys_out,
                                                                     int32_t* __restrict__ vals_out, int64_t groups,
                                                                     int32_t* __restrict__ offsets, ZeroFill zero) {
  if (blockIdx.x >= zero.first) return zero_fill(zero);
  __shared__ uint32_t s_base[kDigitBins];
  __shared__ uint32_t s_wave[kDigitWaves][kDigitBins];
  __shared__ uint32_t s_part[2][kDigitThreads];
  __shared__ uint32_t s_sum[kDigitWaves];
  const int bins = 1 << bits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tile = blockIdx.x, base = tile * kDigitTile;
  for (int d = threadIdx.x; d < bins * kDigitWaves; d += kDigitThreads) s_wave[d >> bits][d & (bins - 1)] = 0;
  __syncthreads();
  // ranks within the wavefront's stretch (a wavefront counts in its own row of s_wave: no barrier in between)
  uint32_t key[kDigitRounds], rank[kDigitRounds];
  int32_t val[kDigitRounds];
  const uint64_t below = (1ull << lane) - 1ull;
#pragma unroll
  for (int q = 0; q < kDigitRounds; ++q) {
    const int64_t i = base + wave * (64 * kDigitRounds) + q * 64 + lane;
    key[q] = i < n ? rows.key(i) : 0u;
    val[q] = i < n ? rows.val(i) : 0;
  }
#pragma unroll
  for (int q = 0; q < kDigitRounds; ++q) {
    const int64_t i = base + wave * (64 * kDigitRounds) + q * 64 + lane;
    const uint32_t d = (key[q] >> shift) & (bins - 1);
    uint64_t same = __ballot(i < n);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((d >> b) & 1u);
      same &= ((d >> b) & 1u) ? set : ~set;
    }
    const uint32_t before = (uint32_t)__popcll(same & below);
    rank[q] = s_wave[wave][d] + before;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (i < n && before == 0) s_wave[wave][d] += (uint32_t)__popcll(same);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  // where the tile's rows of each digit begin
  if (scanned) {
    for (int d = threadIdx.x; d < bins; d += kDigitThreads) s_base[d] = hist[(int64_t)d * tiles + tile];
  } else {
    // kDigitThreads / bins threads share a bin, each adds up a stretch of the tiles; their sums meet in s_part
    const int d = threadIdx.x & (bins - 1), share = (int)threadIdx.x >> bits, shares = kDigitThreads >> bits;
    const int64_t per = (tiles + shares - 1) / shares, first = share * per, stop = min(first + per, tiles);
    uint32_t all = 0, earlier = 0;
#pragma unroll 16
    for (int64_t t = first; t < stop; ++t) {
      const uint32_t c = hist[t * bins + d];
      all += c;
      if (t < tile) earlier += c;
    }
    s_part[0][threadIdx.x] = all;
    s_part[1][threadIdx.x] = earlier;
    __syncthreads();
    if (share == 0) {
      for (int h = 1; h < shares; ++h) {
        all += s_part[0][(h << bits) + d];
        earlier += s_part[1][(h << bits) + d];
      }
    } else {
      all = 0;
    }
    uint32_t upto = all;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const uint32_t other = __shfl_up(upto, s, 64);
      if (lane >= s) upto += other;
    }
    if (lane == 63) s_sum[wave] = upto;
    __syncthreads();
    uint32_t start = upto - all;
    for (int w = 0; w < wave; ++w) start += s_sum[w];
    if (share == 0) {
      s_base[d] = start + earlier;
      if (offsets && tile == 0 && d <= groups) offsets[d] = (int32_t)start;
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kDigitThreads) {
    uint32_t at = s_base[d];
#pragma unroll
    for (int w = 0; w < kDigitWaves; ++w) {
      const uint32_t c = s_wave[w][d];
      s_wave[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kDigitRounds; ++q) {
    const int64_t i = base + wave * (64 * kDigitRounds) + q * 64 + lane;
    if (i >= n) continue;
    const uint32_t to = s_wave[wave][(key[q] >> shift) & (bins - 1)] + rank[q];
    if (keys_out) keys_out[to] = key[q];
    vals_out[to] = val[q];
  }
}

// ---------------------------------------------------------------------------------------------
// Gradient of the lookup: sums over the stretches of equal keys of the sorted rows.  A chunk of 2^chunk_log2 sorted rows
// is added up by one group of threads, 16 bytes of a row each; a sum that lies within the chunk goes to the table, one
// that began before it to carry slot 2c, one that goes on behind it to slot 2c + 1 (32 bits), and a second kernel adds
// those up in order.  No atomics: the same ids give the same bits.  Sums are held in 32 bits and rounded once.
//
// Bound by the bytes: rows of the gradient in a random order, rows of the table written.  262144 rows of 1024 bf16 over
// 32768 rows of f32: 537 + 134 MB in 150 us, 4.5 TB/s (an addition over all of a large array reads at 4.0); one workgroup
// for each row of the table that walks its rows: 4300 us, the frequent ids being one chain.  Chunks of 16 to 128 rows:
// the fewer, the less is carried (32768 rows of 2048, 16 / 32 / 64 rows a chunk: 165 / 161 / 160 us in all).  16 instead
// of 8 rows in flight: fewer workgroups on a CU, 268 -> 380 us.
// ---------------------------------------------------------------------------------------------

constexpr int kSumFlight = 8;  // rows in flight (4: the same times)

// Sorted keys and rows, as the kernel finds them: reads at addresses that a whole workgroup shares go through scalar
// registers.
template <class T>
using Fixed = const __attribute__((address_space(4))) T*;

// Elements [lo, hi) of at[0 .. kN) = (accumulate ? at : 0) + scale * v.  kWhole: all of them, at a multiple of their size.
template <class TO, int kN, bool kWhole>
__device__ __forceinline__ void store_sum(TO* at, int lo, int hi, const float (&v)[kN], float scale, int accumulate) {
  constexpr int kPart = kN < kPer16<TO> ? kN : kPer16<TO>;
  if (kWhole || (lo == 0 && hi >= kN)) {
#pragma unroll
    for (int p = 0; p < kN; p += kPart) {
      float out[kPart];
#pragma unroll
      for (int i = 0; i < kPart; ++i) out[i] = scale * v[p + i];
      if (accumulate) {
        const auto old = *reinterpret_cast<const typename Pack<TO, kPart, kWhole>::type*>(at + p);
#pragma unroll
        for (int i = 0; i < kPart; ++i) out[i] += (float)old[i];
      }
      store_n<kWhole, TO, kPart>(at + p, out);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (i >= lo && i < hi) {
        float out = scale * v[i];
        if (accumulate) out += (float)at[i];
        at[i] = (TO)out;
      }
  }
}

// How the rows lie: whole 16-byte pieces at multiples of 16 bytes; any alignment and length, but at least one piece (the
// last thread of a row then reads the row's last 16 bytes and leaves out what its neighbour owns); shorter rows.
enum RowForm { kRowWhole = 0, kRowLoose = 1, kRowShort = 2 };

struct SumArgs {
  int64_t n;
  uint32_t vocab;
  int32_t width, pitch;  // columns; floats from one carry slot to the next
  const uint32_t* keys;
  const int32_t* pos;
  const void* grad;
  int64_t ld_grad;
  float scale;
  void* d_table;
  int64_t ld_table;
  int accumulate;
  float* carry;
  int chunk_log2, tpr_log2;
  int64_t chunks;
  unsigned sum_blocks;   // workgroups that add up
  unsigned zero_blocks;  // workgroups behind them that fill the rows of the table that no id points at with zeros
};

constexpr int kZeroRows = 64;  // rows of the table a workgroup looks at for that

template <class T, class TO, int kForm, bool kWide>
__global__ __launch_bounds__(kBlock) void embedding_sum_kernel(SumArgs g) {
  constexpr int V = kPer16<T>;
  constexpr bool kWhole = kForm == kRowWhole;
  const int tpr = 1 << g.tpr_log2;
  if (blockIdx.x >= g.sum_blocks) {
    // (all column tiles of a row by one workgroup)
    if (blockIdx.y != 0) return;
    const int lane = threadIdx.x & 63;
    constexpr int kPart = kPer16<TO>;
    const float zero[kPart] = {};
    for (int64_t v0 = (int64_t)(blockIdx.x - g.sum_blocks) * kZeroRows; v0 < g.vocab; v0 += (int64_t)g.zero_blocks * kZeroRows) {
      bool empty = false;
      if (v0 + lane < g.vocab) {
        const int64_t at = lower_bound_u32(g.keys, g.n, (uint32_t)(v0 + lane));
        empty = at == g.n || g.keys[at] != (uint32_t)(v0 + lane);
      }
      uint64_t rows = __ballot(empty);
      while (rows) {
        const int r = __ffsll((unsigned long long)rows) - 1;
        rows &= rows - 1;
        TO* row = (TO*)g.d_table + (v0 + r) * g.ld_table;
        for (int c = (int)threadIdx.x * kPart; c < g.width; c += (int)blockDim.x * kPart)
          store_sum<TO, kPart, false>(row + c, 0, g.width - c, zero, 0.f, 0);
      }
    }
    return;
  }
  const int64_t c = kWide ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x << (8 - g.tpr_log2)) + ((int)threadIdx.x >> g.tpr_log2);
  const int own = ((int)blockIdx.y * tpr + ((int)threadIdx.x & (tpr - 1))) * V;  // first column of this thread's
  if (c >= g.chunks || own >= g.width) return;
  const int col = kForm == kRowLoose ? min(own, g.width - V) : own;              // first column that it reads
  const int lo = own - col, hi = kForm == kRowShort ? g.width : V;
  const int64_t begin = c << g.chunk_log2, end = min(begin + ((int64_t)1 << g.chunk_log2), g.n);
  const Fixed<uint32_t> keys = (Fixed<uint32_t>)(uintptr_t)g.keys;
  const Fixed<int32_t> pos = (Fixed<int32_t>)(uintptr_t)g.pos;
  uint32_t cur = keys[begin];
  bool open = keys[begin > 0 ? begin - 1 : 0] == cur && begin > 0;  // the sum began in an earlier chunk
  float acc[V] = {};
  const T* grad = (const T*)g.grad + col;
  auto close = [&](int slot) {
    if (slot >= 0) store_sum<float, V, kWhole>(g.carry + (2 * c + slot) * (int64_t)g.pitch + col, lo, hi, acc, 1.f, 0);
    else store_sum<TO, V, kWhole>((TO*)g.d_table + (int64_t)cur * g.ld_table + col, lo, hi, acc, g.scale, g.accumulate);
  };
  for (int64_t q0 = begin; q0 < end && cur < g.vocab; q0 += kSumFlight) {
    // (all loads are asked for before the first is used: none is conditional, behind the end the last row is read again)
    uint32_t key[kSumFlight];
    int32_t from[kSumFlight];
    typename Pack<T, V, true>::type row[kSumFlight];
#pragma unroll
    for (int u = 0; u < kSumFlight; ++u) {
      const int64_t q = min(q0 + u, end - 1);
      key[u] = keys[q];
      from[u] = pos[q];
    }
    if constexpr (kWide) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < kSumFlight; ++u) {
      const T* p = grad + (int64_t)from[u] * g.ld_grad;
      if constexpr (kForm == kRowShort) {
#pragma unroll
        for (int i = 0; i < V; ++i) row[u][i] = i < hi ? p[i] : (T)0.f;
      } else {
        row[u] = *reinterpret_cast<const typename Pack<T, V, kWhole>::type*>(p);
      }
    }
#pragma unroll
    for (int u = 0; u < kSumFlight; ++u) {
      if (q0 + u >= end) break;
      if (key[u] != cur) {
        close(open ? 0 : -1);
        open = false;
        cur = key[u];
        if (cur >= g.vocab) break;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += (float)row[u][i];
    }
  }
  if (cur >= g.vocab) return;
  const bool goes_on = end < g.n && keys[end] == cur;
  close(open ? 0 : goes_on ? 1 : -1);
}

// The sums that cross chunks: the chunk in which one begins adds up its slots.  One workgroup per chunk and 256 columns
// (most have nothing to do); its wavefronts take a stretch of the slots each, and their sums are added in that order.
// Bound by its chain of loads, 3 to 11 us: keys around the chunk's end, keys at the starts of the next 64 chunks, slots.
// (Workgroups that looked at 8 chunks each and searched for a sum's end: 41 to 48 us.)
template <class TO, bool kWhole>
__global__ __launch_bounds__(kBlock) void embedding_fix_kernel(SumArgs g) {
  __shared__ float s_part[kWavesPerBlock][64][4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int64_t c = blockIdx.x, begin = c << g.chunk_log2, end = begin + ((int64_t)1 << g.chunk_log2);
  if (end >= g.n) return;
  const uint32_t key = g.keys[end - 1], next = g.keys[end], first_key = g.keys[begin], before = g.keys[begin > 0 ? begin - 1 : 0];
  if (key >= g.vocab || next != key) return;                     // it ends here
  if (begin > 0 && first_key == key && before == key) return;    // it began earlier
  // chunks behind this one that begin within the sum, 64 a step
  int64_t slots = 0;
  for (;;) {
    const int64_t at = (c + 1 + slots + lane) << g.chunk_log2;
    const uint64_t within = __ballot(at < g.n && g.keys[min(at, g.n - 1)] == key);
    const int more = __popcll(within);
    slots += more;
    if (more < 64) break;
  }
  const int col = ((int)blockIdx.y * 64 + lane) * 4, there = g.width - col;
  const int64_t per = (slots + kWavesPerBlock - 1) / kWavesPerBlock;
  const int64_t first = wave * per, last = min(first + per, slots);
  float acc[4] = {};
  if (there > 0) {
    if (wave == 0) load16<true>(g.carry + (2 * c + 1) * (int64_t)g.pitch + col, acc);
#pragma unroll 8
    for (int64_t s = first; s < last; ++s) {
      float v[4];
      load16<true>(g.carry + 2 * (c + 1 + s) * (int64_t)g.pitch + col, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += v[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s_part[wave][lane][i] = acc[i];
  __syncthreads();
  if (wave != 0 || there <= 0) return;
#pragma unroll
  for (int w = 1; w < kWavesPerBlock; ++w)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += s_part[w][lane][i];
  store_sum<TO, 4, kWhole>((TO*)g.d_table + (int64_t)key * g.ld_table + col, 0, there, acc, g.scale, g.accumulate);
}

}  // namespace hpspmm
