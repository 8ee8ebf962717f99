// The softmax step of the tcgen05 attention kernels: a thread has one row's 128
// scores in registers and writes its weights, 16 bit, over them in TMEM.
//
// All of its arithmetic but the exponential runs two values to an instruction, or
// three to a maximum.
#pragma once

#include "kf_common.cuh"

namespace kf {

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  uint32_t r;
  if constexpr (DType<T>::code == KF_BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  }
  return r;
}

// The largest of `m` and the row's scores.
__device__ __forceinline__ float row_max(const float (&s)[128], float m) {
  float top[4] = {m, s[0], s[1], s[2]};
  top[0] = fmaxf(top[0], s[3]);
#pragma unroll
  for (int x = 4; x < 124; x += 8) {
#pragma unroll
    for (int y = 0; y < 4; ++y) top[y] = max3(top[y], s[x + y], s[x + 4 + y]);
  }
#pragma unroll
  for (int y = 0; y < 4; ++y) top[y] = fmaxf(top[y], s[124 + y]);
  return fmaxf(max3(top[0], top[1], top[2]), top[3]);
}

// P = 2^(c s - cm) to TMEM at `to`, 64 columns; returns the sum of the unrounded
// weights. The warp arrives on `done` when its weights are there.
template <typename T>
__device__ __forceinline__ float row_weights(const float (&s)[128], float c, float cm, uint32_t to, uint32_t done, int lane) {
  const uint64_t c2 = f2_splat(c), cm2 = f2_splat(-cm);
  uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
  for (int x = 0; x < 128; x += 32) {
    uint32_t w[16];
#pragma unroll
    for (int y = 0; y < 32; y += 2) {
      const float2 e = f2_unpack(f2_fma(f2_pack(s[x + y], s[x + y + 1]), c2, cm2));
      const float2 v = make_float2(ex2_ftz(e.x), ex2_ftz(e.y));
      sum[(y / 2) & 1] = f2_add(sum[(y / 2) & 1], f2_pack(v.x, v.y));
      w[y / 2] = pack_pair<T>(v.x, v.y);
    }
    tmem_st_16(to + x / 2, w);
  }
  tmem_st_wait();
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(done);
  const float2 f = f2_unpack(f2_add(sum[0], sum[1]));
  return f.x + f.y;
}

}  // namespace kf
