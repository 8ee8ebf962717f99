// The softmax step of the tcgen05 attention kernels: a thread has one row's 128
// scores in registers and writes its weights, 16 bit, over them in TMEM.
// All of its arithmetic but the exponential runs two values to an instruction, or
// three to a maximum.
//
// 2^x on the special-function unit takes 8 cycles per warp and quarter SM, 1024
// for a tile of 128 x 128, as long as the tile's two products. Where two tiles
// share an SM a quarter of the exponentials is computed on the FMA pipe instead
// (EMULATE): x = n + f with n the nearest integer, 2^f by the degree-4 polynomial
// with constant term 1 of least relative error on [-1/2, 1/2] (2.9e-6 as computed),
// and n added to the exponent. One 8192-token prompt at 32/8 heads of 128 in bursts: 465 us
// without it, 450 with it.
#pragma once

#include "kf_common.cuh"

namespace kf {

// A row's maximum is raised, and its sums rescaled, when it grew by more than this.
constexpr float RAISE_LOG2 = 8.0f;
// By so much are the weights made smaller, and the row's maximum (for its sums' base) larger.
// bf16 weights stay at one or below: a value near the end of the type's range, which is
// fp32's, would overflow the sums times 2^8. fp16's values are far from that, and its
// weights would lose bits.
template <typename T>
constexpr float WEIGHT_SHIFT = DType<T>::code == KF_BF16 ? RAISE_LOG2 : 0.0f;

// Maxima that a NaN among their operands makes NaN.
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16],"
      " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}

// The largest of `m` and the row's scores; NaN if one of them is.
__device__ __forceinline__ float row_max(const float (&s)[128], float m) {
  float top[4] = {m, s[0], s[1], s[2]};
  top[0] = max2(top[0], s[3]);
#pragma unroll
  for (int x = 4; x < 124; x += 8) {
#pragma unroll
    for (int y = 0; y < 4; ++y) top[y] = max3(top[y], s[x + y], s[x + 4 + y]);
  }
#pragma unroll
  for (int y = 0; y < 4; ++y) top[y] = max2(top[y], s[124 + y]);
  return max2(max3(top[0], top[1], top[2]), top[3]);
}

// 2^x of two values without the special-function unit; x = -127 and below (a key
// that the row does not see) give exactly zero, and so does NaN: a row that has
// one is known by its maximum.
__device__ __forceinline__ uint64_t ex2_poly2(float2 v) {
  // n = -127, f = 0 make the polynomial 1, whose exponent field the addition clears. Down to
  // there f is not negative, so the field does not wrap: what is below 2^-126 comes out as
  // some number from zero to that.
  const uint64_t x = f2_pack(fmaxf(v.x, -127.0f), fmaxf(v.y, -127.0f));
  const uint64_t magic = f2_splat(12582912.0f);  // 1.5 x 2^23: adding it leaves the nearest integer in the low bits
  const uint64_t t = f2_add(x, magic);
  const uint64_t f = f2_add(x, f2_fma(t, f2_splat(-1.0f), magic));
  uint64_t r = f2_fma(f, f2_splat(0.009582852944731712f), f2_splat(0.055906426161527634f));
  r = f2_fma(r, f, f2_splat(0.24024099111557007f));
  r = f2_fma(r, f, f2_splat(0.6931241750717163f));
  r = f2_fma(r, f, f2_splat(1.0f));
  const float2 tf = f2_unpack(t), rf = f2_unpack(r);
  return f2_pack(__int_as_float(__float_as_int(rf.x) + (__float_as_int(tf.x) << 23)),
                 __int_as_float(__float_as_int(rf.y) + (__float_as_int(tf.y) << 23)));
}

// P = 2^(c s - cm) of 32 keys to TMEM at `to`, 16 columns; returns the sums of the
// unrounded weights (two of them, to be added). A masked key, whose score is
// -infinity, weighs exactly zero either way.
template <typename T, bool EMULATE>
__device__ __forceinline__ uint64_t weights_32(const float* s, uint64_t c2, uint64_t minus_cm2, uint32_t to) {
  uint64_t sum[2] = {0ull, 0ull};
  uint32_t w[16];
#pragma unroll
  for (int y = 0; y < 32; y += 2) {
    const float2 e = f2_unpack(f2_fma(f2_pack(s[y], s[y + 1]), c2, minus_cm2));
    const uint64_t v = EMULATE && (y / 2) % 4 == 3 ? ex2_poly2(e) : f2_pack(ex2_ftz(e.x), ex2_ftz(e.y));
    sum[(y / 2) & 1] = f2_add(sum[(y / 2) & 1], v);
    const float2 vf = f2_unpack(v);
    w[y / 2] = pack_pair<T>(vf.x, vf.y);
  }
  tmem_st_16(to, w);
  return f2_add(sum[0], sum[1]);
}

// The warp's weights so far are in TMEM: arrive on `bar`.
__device__ __forceinline__ void weights_done(uint32_t bar, int lane) {
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

// All 128 keys' weights, with an arrival on `half` after 64 and on `all` at the end
// (half 0: at the end alone); returns their sum.
template <typename T, bool EMULATE>
__device__ __forceinline__ float row_weights(const float (&s)[128], float c, float cm, uint32_t to, uint32_t half,
                                             uint32_t all, int lane) {
  const uint64_t c2 = f2_splat(c), minus_cm2 = f2_splat(-cm);
  uint64_t sum = weights_32<T, EMULATE>(s, c2, minus_cm2, to);
#pragma unroll
  for (int x = 32; x < 128; x += 32) {
    sum = f2_add(sum, weights_32<T, EMULATE>(s + x, c2, minus_cm2, to + x / 2));
    if (x == 32 && half != 0) weights_done(half, lane);
  }
  weights_done(all, lane);
  const float2 f = f2_unpack(sum);
  return f.x + f.y;
}

}  // namespace kf
