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

}  // namespace
}  // namespace kf
