// The tile kernel of the products grouped by expert: one workgroup per kBM x kBN tile of the output.
//
// Both operands of a step of the contraction (64 terms of 16-bit, 32 of 32-bit elements) lie in LDS in the layout they
// have in memory, 16-byte chunks permuted within a row:
//   row operand  kB rows of the tile, 128 bytes (8 chunks) of the contraction each      x, dy and w^T (forward)
//   col operand  the step's rows, kB columns of the tile each                           w (gradient of x), dy and x (of w)
// A fragment of a row operand is one 16-byte read a lane.  One of a col operand is read transposed: 16-bit elements with
// the transposing 8-byte read (lane s of 16 gives the address of columns 4 (s % 4) ... + 3 of row s / 4 and receives
// column s of the four rows), 32-bit ones word by word.  The permutations put what one read touches into different
// banks: chunk c of row r lies at c ^ (r % 8) in a row operand; in a col operand the 32-byte (16-bit elements) or 64-byte
// (32-bit) segments of the rows that a read meets are spread.
//
// Rows beyond the group and columns beyond the matrix repeat the last one that exists - what they give is not stored;
// terms beyond the contraction are zeros in both operands, whatever lies there in memory.
//
// Sums are held in 32 bits by the matrix instructions (16 x 16 x 32 for 16-bit, 16 x 16 x 4 for 32-bit elements) and
// rounded once.  bf16, 32768 rows, 32 groups, k 2048, m 4096, tiles of 256, a call among many on three sets of operands in
// turn: product 544 us (995 TFLOP/s), gradient of x 543 us, of w in 32 bits 736 us; 16384 rows, 16 groups: 292, 304 and 374.
// The matrix cores are busy 55 % of the product's time (of the gradients' at 16384 rows 46 and 41 %), an eighth of it with
// rows beyond the ends of groups.  What bounds it is the way of the operands into LDS: without the products the same loads
// take 510 us, without the loads the products 405 us (one set of operands again and again); a CU has about 64 lines under
// way, at 570 cycles each (a larger tile, fewer bytes, does not fit 160 KB of LDS).  The steps' reads of LDS meet no bank
// conflicts in any of the three.  On the way, likewise on one set: loads with
// the builtin, whose counter every transposed read waits for, 715 / 944 us for the gradients; steps of 32 terms, half a
// line a row, 650 / 870 / 1155 us; tiles in rows instead of panels, a third more requests to memory, 575 instead of 562 us.
#pragma once

#include "grouped_kernels.hpp"

namespace hpspmm {

typedef float float4_t __attribute__((ext_vector_type(4)));

template <class T>
struct Mfma;
template <>
struct Mfma<bf16_t> {
  typedef bf16_t frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float4_t mul(frag a, frag b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma<f16_t> {
  typedef f16_t frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float4_t mul(frag a, frag b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma<float> {
  typedef float frag __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ float4_t mul(frag a, frag b, float4_t c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

typedef __attribute__((address_space(3))) char lds_char;
typedef short short4_t __attribute__((ext_vector_type(4)));

constexpr int kStepChunks = 8;  // 16-byte chunks of the contraction a step: whole lines of a row operand

// One operand of one output tile.
template <class T, bool kCol, int kB, int kThreads, bool kDirect>
struct Operand {
  static constexpr int kSize = (int)sizeof(T);
  static constexpr int kChunk = 16 / kSize;    // elements of a 16-byte chunk
  static constexpr int kDepth = kStepChunks * kChunk;  // terms of the contraction a step
  static constexpr int kBytes = kB * kStepChunks * 16;  // of LDS a step
  static constexpr int kPer = kB * kStepChunks / kThreads;  // chunks a thread brings in a step
  static constexpr int kRowChunks = kCol ? kB / kChunk : kStepChunks;  // chunks of a row in LDS
  static constexpr uint32_t kNowhere = 0xFFFFFFF0u;  // an offset beyond the buffer: the load gives zeros
  using Chunk = typename Pack<T, kChunk, true>::type;

  const char* base;    // first element of the step to be loaded
  int64_t step;        // bytes from one step to the next
  int64_t ld;          // bytes from row to row
  int valid;           // rows (row operand) or columns (col operand) of the tile that exist
  uint32_t offset[kDirect ? kPer : 1];

  static __device__ __forceinline__ int swizzle(int r) {
    if constexpr (!kCol) return r & 7;
    else if constexpr (kSize == 2) return (((r & 3) | ((r >> 1) & 4)) << 1) & (kRowChunks - 1);
    else return (((r >> 2) & 3) << 2) & (kRowChunks - 1);
  }
  // Row of LDS and chunk of that row in memory that this thread's i-th chunk is.
  static __device__ __forceinline__ void place(int i, int& r, int& c) {
    const int q = i * kThreads + (int)threadIdx.x;
    r = q / kRowChunks;
    c = (q % kRowChunks) ^ swizzle(r);
  }

  // first: first element of the tile; valid_: its rows or columns that exist, at least 1.
  __device__ __forceinline__ void init(const T* first, int64_t ld_, int64_t valid_) {
    base = (const char*)first;
    ld = ld_ * kSize;
    step = kCol ? ld * kDepth : (int64_t)kDepth * kSize;
    valid = (int)min(valid_, (int64_t)kB);
    if constexpr (kDirect) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        int r, c;
        place(i, r, c);
        offset[i] = kCol ? (uint32_t)r * (uint32_t)ld + (uint32_t)(min(c * kChunk, valid - kChunk) * kSize)
                         : (uint32_t)min(r, valid - 1) * (uint32_t)ld + (uint32_t)c * 16u;
      }
    }
  }

  // Before the first load of a step of which only `left` terms are left: what lies behind them becomes zeros, in this
  // step and all later ones.
  __device__ __forceinline__ void end_after(int64_t left) {
    if (left >= kDepth) return;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int r, c;
      place(i, r, c);
      if ((kCol ? r : c * kChunk) >= left) offset[i] = kNowhere;
    }
  }
  // Brings this thread's i-th chunk of a step into LDS without passing registers: a wavefront's 64 chunks land one behind
  // the other.  (Written out: behind the builtin the compiler lets every transposed read of LDS wait for all loads that
  // are under way.  The load has no output register; wait_loads() waits for it.  One wait state lies between the write of
  // m0 and its use; nothing else in the kernel uses m0.)
  __device__ __forceinline__ void load_direct(uint32_t lds, int i) const {
    typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));
    const uint64_t at = (uint64_t)base;
    const uint4_t rsrc = {(uint32_t)at, (uint32_t)(at >> 32) & 0xFFFFu, 0x7FFFFFFFu, 0x00020000u};
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds + i * kThreads * 16), "v"(offset[i]), "s"(rsrc)
                 : "memory");
  }

  // The same for rows at any alignment and of any length, through registers.  Inner steps are those whose chunks stay
  // within the matrix: there a chunk that runs over the end of its row reads on into the next rows - what it gives is not
  // stored -, and no load hangs on a condition, for which it would wait.  The one or two steps behind them go by elements.
  __device__ __forceinline__ int64_t inner_steps(int64_t depth) const {
    if constexpr (!kCol) return depth / kDepth;
    // bytes that the last chunk of a row runs over its end, and the rows that they reach into
    const int64_t over = (int64_t)(((valid - 1) / kChunk + 1) * kChunk - valid) * kSize;
    return max(depth - (over + ld - 1) / ld, (int64_t)0) / kDepth;
  }
  __device__ __forceinline__ void load_inner(Chunk (&regs)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int r, c;
      place(i, r, c);
      if constexpr (kCol) c = min(c, (valid - 1) / kChunk);
      else r = min(r, valid - 1);
      regs[i] = *reinterpret_cast<const typename Pack<T, kChunk, false>::type*>((const T*)(base + (int64_t)r * ld) + c * kChunk);
    }
    base += step;
  }
  __device__ __forceinline__ void load_last(Chunk (&regs)[kPer], int64_t left) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      int r, c;
      place(i, r, c);
      // elements of the chunk that exist
      const int64_t there = kCol ? (r < left ? (int64_t)valid - c * kChunk : 0) : left - c * kChunk;
      const T* p = (const T*)(base + (int64_t)(kCol ? r : min(r, valid - 1)) * ld) + c * kChunk;
#pragma unroll
      for (int e = 0; e < kChunk; ++e) regs[i][e] = e < there ? p[e] : (T)0.f;
    }
    base += step;
  }
  static __device__ __forceinline__ void put(char* lds, const Chunk (&regs)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) *reinterpret_cast<Chunk*>(lds + (i * kThreads + (int)threadIdx.x) * 16) = regs[i];
  }

  // Fragment of 16 rows or columns from `at` on, half `h` of the step's terms.
  static __device__ __forceinline__ typename Mfma<T>::frag fragment(const char* lds, int at, int h) {
    using Frag = typename Mfma<T>::frag;
    const int lane = threadIdx.x & 63, low = lane & 15, high = lane >> 4;
    if constexpr (!kCol) {
      const int r = at + low;
      return *reinterpret_cast<const Frag*>(lds + r * (kStepChunks * 16) + (((h * 4 + high) ^ swizzle(r)) << 4));
    } else if constexpr (kSize == 2) {
      Frag f;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int r = h * 32 + high * 8 + q * 4 + (low >> 2);
        const int byte = (at + (low & 3) * 4) * 2;
        const short4_t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) short4_t*)(lds + r * (kB * 2) + (byte ^ (swizzle(r) << 4))));
        const auto t = __builtin_bit_cast(typename Pack<T, 4, true>::type, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[q * 4 + e] = t[e];
      }
      return f;
    } else {
      Frag f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = h * 16 + high * 4 + e;
        f[e] = *reinterpret_cast<const float*>(lds + r * (kB * 4) + (((at + low) * 4) ^ (swizzle(r) << 4)));
      }
      return f;
    }
  }
};

// Waits until at most n of the loads that this wavefront has asked for are under way, and none of its reads of LDS.
template <int n>
__device__ __forceinline__ void wait_loads() {
  static_assert(n >= 0 && n < 64, "six bits count them");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(n) : "memory");
}
// A barrier that waits for no loads by itself.
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The largest part of `all` rows, halved as often as needed, that fits `room` rows.
constexpr int whole_rows(int room, int all) { return all <= room ? all : whole_rows(room, all / 2); }

// Workgroup -> output tile: the tiles in use are cut into one contiguous stretch for each XCD, so that the tiles that an
// XCD works on at a time share rows of x and columns of w in its L2.
__device__ __forceinline__ int64_t xcd_tile(int64_t tiles) {
  const int64_t per = (tiles + kXcds - 1) / kXcds, b = blockIdx.x;
  const int64_t t = (b % kXcds) * per + b / kXcds;
  return b / kXcds < per && t < tiles ? t : -1;
}

template <class T, class TO, int kMode, int kBM, int kBN, int kWM, int kWN, bool kDirect, int kStagesA, int kStagesB, bool kSplit = false>
__global__ __launch_bounds__(64 * kWM * kWN, 2) void grouped_tile_kernel(GroupedArgs g, int col_tiles) {
  constexpr int kThreads = 64 * kWM * kWN;
  using OpA = Operand<T, kMode == kGradW, kBM, kThreads, kDirect>;
  using OpB = Operand<T, kMode != kForward, kBN, kThreads, kDirect>;
  using Frag = typename Mfma<T>::frag;
  constexpr int FM = kBM / kWM / 16, FN = kBN / kWN / 16, kDepth = OpA::kDepth;
  constexpr int kLdsA = kStagesA * OpA::kBytes, kLds = kLdsA + kStagesB * OpB::kBytes;
  __shared__ __attribute__((aligned(1024))) char lds[kLds];

  // the tile of the output, its operands, the length of the contraction
  int64_t e, row0 = 0, end = 0, depth, m_left, n_left;
  const int n_out = kMode == kForward ? g.m : g.k;
  OpA a;
  OpB b;
  TO* c;
  float* out_part = nullptr;
  if constexpr (kMode == kGradW) {
    const int row_tiles = (g.m + kBM - 1) / kBM;
    const int64_t tiles = g.groups * row_tiles * col_tiles;
    const int64_t tp = xcd_tile(kSplit ? tiles * g.splits : tiles);
    if (tp < 0) return;
    const int64_t part = kSplit ? tp / tiles : 0, t = kSplit ? tp - part * tiles : tp;
    e = t / (row_tiles * col_tiles);
    int64_t mt;
    int nt;
    panel_tile(t - e * row_tiles * col_tiles, row_tiles, col_tiles, mt, nt);
    group_rows_of(g, e, row0, end);
    if constexpr (kSplit) {
      // the part's steps of the contraction
      const int64_t per = ((end - row0 + kDepth - 1) / kDepth + g.splits - 1) / g.splits * kDepth;
      row0 = min(row0 + part * per, end);
      end = min(row0 + per, end);
      out_part = g.parts + tp * (kBM * kBN);
    }
    depth = end - row0;
    m_left = g.m - mt * kBM;
    n_left = n_out - (int64_t)nt * kBN;
    a.init((const T*)g.a + row0 * g.lda + mt * kBM, g.lda, m_left);
    b.init((const T*)g.b + row0 * g.ldb + (int64_t)nt * kBN, g.ldb, n_left);
    c = (TO*)g.c + e * g.stride_c + mt * kBM * g.ldc + (int64_t)nt * kBN;
  } else {
    const int64_t row_tiles = count_row_tiles(g, kBM);
    const int64_t t = xcd_tile(row_tiles * col_tiles);
    if (t < 0) return;
    int64_t first, mt;
    int nt;
    if (!find_group(g, t / col_tiles, kBM, e, row0, end, first)) return;
    panel_tile(t - first * col_tiles, (end - row0 + kBM - 1) / kBM, col_tiles, mt, nt);
    row0 += mt * kBM;
    depth = kMode == kForward ? g.k : g.m;
    m_left = end - row0;
    n_left = n_out - (int64_t)nt * kBN;
    a.init((const T*)g.a + row0 * g.lda, g.lda, m_left);
    const T* w = (const T*)g.b + e * g.stride_b;
    b.init(kMode == kForward ? w + (int64_t)nt * kBN * g.ldb : w + (int64_t)nt * kBN, g.ldb, n_left);
    c = (TO*)g.c + row0 * g.ldc + (int64_t)nt * kBN;
  }

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int am = wave / kWN * (kBM / kWM), bn = wave % kWN * (kBN / kWN);
  float4_t acc[FM][FN] = {};
  // The products of one step, sum by sum of 16 rows; `between(i)` after the i-th.  The next half of the step is read
  // while this one is multiplied.
  constexpr int H = kStepChunks / 4;
  auto multiply = [&](const char* lds_a, const char* lds_b, auto between) {
    Frag fa[H][FM], fb[H][FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) fb[0][j] = OpB::fragment(lds_b, bn + j * 16, 0);
#pragma unroll
    for (int i = 0; i < FM; ++i) fa[0][i] = OpA::fragment(lds_a, am + i * 16, 0);
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        // (the operands exchanged: a lane then holds four neighbouring columns of one row of the output)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = Mfma<T>::mul(fb[h][j], fa[h][i], acc[i][j]);
        between(h * FM + i);
        if (h + 1 < H) {
          fa[h + 1][i] = OpA::fragment(lds_a, am + i * 16, h + 1);
          if (i < FN) fb[h + 1][i] = OpB::fragment(lds_b, bn + i * 16, h + 1);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
  };

  // Some steps of each operand in LDS: one is multiplied while the next ones are on their way.  The barrier at the head
  // of a step says that its operands are there, and that nobody reads the step before it any more, whose places the steps
  // brought in then take.  Loads past the registers are counted: those of later steps may still be under way (steps beyond
  // the last one are asked for as well, as zeros, so that the count holds to the end).  One operand may be a step further
  // ahead than the other: three steps of a and two of b fill the 160 KB of LDS in tiles of 256, and what is behind the
  // next step keeps the loads flowing while that one is waited for.
  static_assert(kStagesA == kStagesB || kStagesA == kStagesB + 1, "a is asked for after b, and at most a step further ahead");
  static_assert(kDirect || (kStagesA == 2 && kStagesB == 2), "loads through registers are one step ahead");
  const int64_t steps = (depth + kDepth - 1) / kDepth;
  typename OpA::Chunk ra[OpA::kPer];
  typename OpB::Chunk rb[OpB::kPer];
  const int64_t inner = kDirect ? 0 : min(a.inner_steps(depth), b.inner_steps(depth));
  auto load_loose = [&](int64_t s) {
    if (s < inner) {
      a.load_inner(ra);
      b.load_inner(rb);
    } else {
      a.load_last(ra, depth - s * kDepth);
      b.load_last(rb, depth - s * kDepth);
    }
  };
  auto put_loose = [&](int64_t s) {
    OpA::put(lds + (s & 1) * OpA::kBytes, ra);
    OpB::put(lds + kLdsA + (s & 1) * OpB::kBytes, rb);
  };
  const uint32_t lds_wave = (uint32_t)(uintptr_t)(lds_char*)lds + (uint32_t)wave * 1024u;  // where this wavefront's chunks go
  static_assert(FN <= FM, "the fragments of a half are read between the sums of the half before");
  int next_a = 0, next_b = 0;  // steps asked for
  auto ask_a = [&](int i) {
    if (i == 0) a.end_after(depth - (int64_t)next_a * kDepth);
    a.load_direct(lds_wave + (uint32_t)(next_a % kStagesA * OpA::kBytes), i);
    if (i + 1 == OpA::kPer) {
      a.base += a.step;
      ++next_a;
    }
  };
  auto ask_b = [&](int i) {
    if (i == 0) b.end_after(depth - (int64_t)next_b * kDepth);
    b.load_direct(lds_wave + (uint32_t)(kLdsA + next_b % kStagesB * OpB::kBytes), i);
    if (i + 1 == OpB::kPer) {
      b.base += b.step;
      ++next_b;
    }
  };
  auto ask_both = [&](bool with_b) {
#pragma unroll
    for (int i = 0; i < OpB::kPer; ++i)
      if (with_b) ask_b(i);
#pragma unroll
    for (int i = 0; i < OpA::kPer; ++i) ask_a(i);
  };
  if (steps > 0) {
    if constexpr (kDirect) {
#pragma unroll
      for (int s = 0; s < kStagesA - 1; ++s) ask_both(s >= kStagesA - kStagesB);
    } else {
      load_loose(0);
      put_loose(0);
    }
  }
  if constexpr (kDirect) {
    int at_a = 0, at_b = 0;  // places of the step at hand
    for (int64_t s = 0; s < steps; ++s) {
      wait_loads<(kStagesA - 2) * OpA::kPer + (kStagesB - 2) * OpB::kPer>();
      meet();
      multiply(lds + at_a * OpA::kBytes, lds + kLdsA + at_b * OpB::kBytes, [&](int i) {
        if (i == 0) ask_both(true);
      });
      at_a = at_a + 1 == kStagesA ? 0 : at_a + 1;
      at_b = at_b + 1 == kStagesB ? 0 : at_b + 1;
    }
  } else {
    for (int64_t s = 0; s < steps; ++s) {
      __syncthreads();
      if (s + 1 < steps) load_loose(s + 1);
      multiply(lds + (s & 1) * OpA::kBytes, lds + kLdsA + (s & 1) * OpB::kBytes, [](int) {});
      if (s + 1 < steps) put_loose(s + 1);
    }
  }
  // (nothing may be on its way into LDS when the workgroup ends)
  if constexpr (kDirect) wait_loads<0>();

  const int lane = threadIdx.x & 63;
  if constexpr (kSplit) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
        *reinterpret_cast<float4_t*>(out_part + (am + i * 16 + (lane & 15)) * kBN + bn + j * 16 + (lane >> 4) * 4) = acc[i][j];
    return;
  }
  // To the output through LDS, so that a store covers whole lines: each wavefront has a share of the stages for itself,
  // kRows rows of its kCols columns at a time, 16-byte pieces permuted by row.
  constexpr int kCols = kBN / kWN, kPiece = kPer16<TO>, kPieces = kCols / kPiece, kRowBytes = kCols * (int)sizeof(TO);
  constexpr int kShare = kLds / (kWM * kWN), kRows = whole_rows(kShare / kRowBytes, kBM / kWM);
  static_assert(kRows % 16 == 0 && kBM / kWM % kRows == 0 && kPieces <= 64, "whole fragments and rows");
  __syncthreads();
  char* mine = lds + wave * kShare;
#pragma unroll
  for (int part = 0; part < kBM / kWM / kRows; ++part) {
#pragma unroll
    for (int i = 0; i < kRows / 16; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int r = i * 16 + (lane & 15), byte = (j * 16 + (lane >> 4) * 4) * (int)sizeof(TO);
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = acc[part * (kRows / 16) + i][j][q];
        // (accumulated values are rounded after the sum)
        if constexpr (kMode == kGradW && sizeof(TO) == 2) {
          if (g.accumulate) {
            const int row = am + part * kRows + r, col = bn + j * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (row < m_left && col + q < n_left) v[q] += (float)c[(int64_t)row * g.ldc + col + q];
          }
        }
        store_n<true, TO, 4>(
            reinterpret_cast<TO*>(mine + r * kRowBytes + ((byte & 15) | (((byte >> 4) ^ (r & (kPieces - 1))) << 4))), v);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the share is the wavefront's own: no barrier)
    constexpr int kAtOnce = 64 / kPieces;  // rows a step
#pragma unroll 4
    for (int r0 = 0; r0 < kRows; r0 += kAtOnce) {
      const int r = r0 + lane / kPieces, p = lane % kPieces;
      const int row = am + part * kRows + r, col = bn + p * kPiece;
      const auto v = *reinterpret_cast<const typename Pack<TO, kPiece, true>::type*>(mine + r * kRowBytes +
                                                                                  ((p ^ (r & (kPieces - 1))) << 4));
      if (row >= m_left || col >= n_left) continue;
      TO* at = c + (int64_t)row * g.ldc + col;
      using Loose = typename Pack<TO, kPiece, false>::type;
      if (col + kPiece <= n_left) {
        if constexpr (kMode == kGradW && sizeof(TO) == 4) {
          if (g.accumulate) {
            *reinterpret_cast<Loose*>(at) = *reinterpret_cast<const Loose*>(at) + v;
            continue;
          }
        }
        // Gradients of large weights go past the caches, which they do not fit: 16 matrices of 4096 x 2048 in 32 bits from
        // 16384 rows 389 -> 374 us (402 -> 355 where the same operands come again and stay in the caches), of 4096 x 4096
        // 768 -> 733 us (798 -> 704); products and gradients of x gain nothing by it.
        if constexpr (kMode == kGradW && kBM == 256) __builtin_nontemporal_store(v, reinterpret_cast<Loose*>(at));
        else *reinterpret_cast<Loose*>(at) = v;
      } else {
#pragma unroll
        for (int q = 0; q < kPiece; ++q)
          if (col + q < n_left) {
            if constexpr (kMode == kGradW && sizeof(TO) == 4) at[q] = g.accumulate ? at[q] + v[q] : v[q];
            else at[q] = v[q];
          }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

}  // namespace hpspmm
