// Vectors of VE elements as the 32-bit words that loads and stores move (a struct of 16-bit
// elements may be moved one by one), and their elements in fp32.
#pragma once

#include <stdint.h>

#include <type_traits>

#include "kf_common.cuh"

namespace kf {
namespace {

// 16-bit elements are held two by two.
template <typename T, int VE>
struct alignas(sizeof(T) * VE) Vec {
  static constexpr bool PAIRS = sizeof(T) == 2 && VE > 1;
  using Word = std::conditional_t<PAIRS, uint32_t, T>;
  static constexpr int WORDS = PAIRS ? VE / 2 : VE;
  Word w[WORDS];
};

template <typename T, int VE>
__device__ __forceinline__ void widen(const Vec<T, VE>& x, float (&f)[VE]) {
#pragma unroll
  for (int i = 0; i < Vec<T, VE>::WORDS; ++i) {
    if constexpr (!Vec<T, VE>::PAIRS) {
      f[i] = to_f32(x.w[i]);
    } else if constexpr (std::is_same_v<T, __half>) {
      const __half2 two = *reinterpret_cast<const __half2*>(&x.w[i]);
      f[2 * i] = __low2float(two), f[2 * i + 1] = __high2float(two);
    } else {  // the upper half of a fp32 number
      f[2 * i] = __uint_as_float(x.w[i] << 16), f[2 * i + 1] = __uint_as_float(x.w[i] & 0xffff0000u);
    }
  }
}

template <typename T, int VE>
__device__ __forceinline__ void narrow(const float (&f)[VE], Vec<T, VE>& x) {
#pragma unroll
  for (int i = 0; i < Vec<T, VE>::WORDS; ++i) {
    if constexpr (Vec<T, VE>::PAIRS) x.w[i] = pack_pair<T>(f[2 * i], f[2 * i + 1]);
    else x.w[i] = from_f32<T>(f[i]);
  }
}


// A vector that this kernel does not read again, and one that it does not read: the first to leave the cache.
template <typename V>
__device__ __forceinline__ V load_once(const void* from) {
  V x;
  if constexpr (sizeof(V) == 16) {
    const uint4 u = __ldcs(static_cast<const uint4*>(from));
    memcpy(&x, &u, 16);
  } else {
    x = *static_cast<const V*>(from);
  }
  return x;
}
// One that many threads read and nobody writes.
template <typename V>
__device__ __forceinline__ V load_common(const void* from) {
  V x;
  if constexpr (sizeof(V) == 16) {
    const uint4 u = __ldg(static_cast<const uint4*>(from));
    memcpy(&x, &u, 16);
  } else {
    x = *static_cast<const V*>(from);
  }
  return x;
}
template <typename V>
__device__ __forceinline__ void store_once(void* to, const V& x) {
  if constexpr (sizeof(V) == 16) {
    uint4 u;
    memcpy(&u, &x, 16);
    __stcs(static_cast<uint4*>(to), u);
  } else {
    *static_cast<V*>(to) = x;
  }
}

// VE elements in fp32, two to a register pair, for the packed arithmetic that does two in one instruction (kf_common.cuh).
template <int VE>
struct Floats {
  static constexpr int N = VE == 1 ? 1 : VE / 2;
  using E = std::conditional_t<VE == 1, float, uint64_t>;
  E e[N];
};
__device__ __forceinline__ float p_mul(float a, float b) { return a * b; }
__device__ __forceinline__ uint64_t p_mul(uint64_t a, uint64_t b) { return f2_mul(a, b); }
__device__ __forceinline__ float p_fma(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ uint64_t p_fma(uint64_t a, uint64_t b, uint64_t c) { return f2_fma(a, b, c); }
__device__ __forceinline__ float p_neg(float a) { return -a; }
__device__ __forceinline__ uint64_t p_neg(uint64_t a) { return a ^ 0x8000000080000000ull; }
__device__ __forceinline__ float p_sum(float a) { return a; }
__device__ __forceinline__ float p_sum(uint64_t a) {
  const float2 f = f2_unpack(a);
  return f.x + f.y;
}
template <int VE>
__device__ __forceinline__ typename Floats<VE>::E p_splat(float a) {
  if constexpr (VE == 1) return a;
  else return f2_splat(a);
}
template <int VE>
__device__ __forceinline__ typename Floats<VE>::E p_at(const float (&f)[VE], int i) {
  if constexpr (VE == 1) return f[0];
  else return f2_pack(f[2 * i], f[2 * i + 1]);
}

template <typename T, int VE>
__device__ __forceinline__ Floats<VE> floats(const Vec<T, VE>& x) {
  float f[VE];
  widen<T, VE>(x, f);
  Floats<VE> to;
#pragma unroll
  for (int i = 0; i < Floats<VE>::N; ++i) to.e[i] = p_at<VE>(f, i);
  return to;
}
template <typename T, int VE>
__device__ __forceinline__ void narrow(const Floats<VE>& x, Vec<T, VE>& to) {
  float f[VE];
#pragma unroll
  for (int i = 0; i < Floats<VE>::N; ++i) {
    if constexpr (VE == 1) {
      f[0] = x.e[0];
    } else {
      const float2 two = f2_unpack(x.e[i]);
      f[2 * i] = two.x, f[2 * i + 1] = two.y;
    }
  }
  narrow<T, VE>(f, to);
}

}  // namespace
}  // namespace kf
