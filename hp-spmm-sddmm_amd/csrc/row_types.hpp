// Element types of the row operators (lookup, gradient of the lookup, products grouped by expert): loads into and
// stores from 32-bit registers, 16 bytes at a time, at the alignment that the caller's rows have.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace hpspmm {

using bf16_t = __bf16;
using f16_t = _Float16;

// kN consecutive elements as they lie in memory.  kAligned: at a multiple of 16 bytes; otherwise at any multiple of
// the element's size (gfx950 serves 16-byte loads and stores at any address, more slowly across a line).
template <class T, int kN, bool kAligned>
struct Pack {
  typedef T vec __attribute__((ext_vector_type(kN)));
  typedef vec loose __attribute__((aligned(sizeof(T))));
  using type = std::conditional_t<kAligned, vec, loose>;
};

// Elements of T in 16 bytes.
template <class T>
inline constexpr int kPer16 = 16 / (int)sizeof(T);

template <bool kAligned, class T>
__device__ __forceinline__ void load16(const T* p, float (&out)[kPer16<T>]) {
  const auto v = *reinterpret_cast<const typename Pack<T, kPer16<T>, kAligned>::type*>(p);
#pragma unroll
  for (int i = 0; i < kPer16<T>; ++i) out[i] = (float)v[i];
}

// (rounds each value once, to nearest even)
template <bool kAligned, class T, int kN>
__device__ __forceinline__ void store_n(T* p, const float* in) {
  typename Pack<T, kN, true>::type v;
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = (T)in[i];
  *reinterpret_cast<typename Pack<T, kN, kAligned>::type*>(p) = v;
}

// The same past the caches: for outputs that do not fit them, in whole lines (pieces of lines cost more than they save).
template <bool kAligned, class T, int kN>
__device__ __forceinline__ void stream_n(T* p, const float* in) {
  typename Pack<T, kN, true>::type v;
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = (T)in[i];
  __builtin_nontemporal_store(v, reinterpret_cast<typename Pack<T, kN, kAligned>::type*>(p));
}
constexpr int64_t kStreamBytes = (int64_t)64 << 20;  // outputs from this size on are written past the caches

// Key of one id: the id itself, or `ids` for one outside [0, ids).
template <class Id>
__device__ __forceinline__ uint32_t id_key(Id id, uint32_t ids) {
  return (uint64_t)(int64_t)id < (uint64_t)ids ? (uint32_t)id : ids;
}

}  // namespace hpspmm
