// What the rotary kernels share: a head as units of two vectors, the turn of a
// unit's pairs, a token's angles and its place in the cache, and the widest
// vectors that a call's layouts allow.
#pragma once

#include <cuda.h>

#include <initializer_list>
#include <type_traits>

#include "kf_common.cuh"
#include "kf_internal.h"
#include "packed.cuh"

namespace kf {
namespace {

// A thread turns one unit of a token's heads: the two vectors of VE elements
// that hold VE pairs, or two plain vectors of the rest of the head.

// The pairs of two vectors' elements turned by their cosines and sines.
template <int VE>
__device__ __forceinline__ void turn(float (&a)[VE], float (&b)[VE], const float (&c)[VE], const float (&s)[VE],
                                     int interleaved) {
  if (interleaved && VE > 1) {
#pragma unroll
    for (int i = 0; i + 1 < VE; i += 2) {
      const float a0 = a[i], b0 = b[i];
      a[i] = fmaf(a0, c[i / 2], -(a[i + 1] * s[i / 2]));
      a[i + 1] = fmaf(a0, s[i / 2], a[i + 1] * c[i / 2]);
      b[i] = fmaf(b0, c[(VE + i) / 2], -(b[i + 1] * s[(VE + i) / 2]));
      b[i + 1] = fmaf(b0, s[(VE + i) / 2], b[i + 1] * c[(VE + i) / 2]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const float a0 = a[i];
      a[i] = fmaf(a0, c[i], -(b[i] * s[i]));
      b[i] = fmaf(a0, s[i], b[i] * c[i]);
    }
  }
}
template <int VE>
__device__ __forceinline__ void turn(Floats<VE>& a, Floats<VE>& b, const float (&c)[VE], const float (&s)[VE], int interleaved) {
#pragma unroll
  for (int i = 0; i < Floats<VE>::N; ++i) {
    if constexpr (VE > 1) {
      if (interleaved) {  // a pair's two elements lie side by side
        const float2 x = f2_unpack(a.e[i]), y = f2_unpack(b.e[i]);
        const float cx = c[i], sx = s[i], cy = c[VE / 2 + i], sy = s[VE / 2 + i];
        a.e[i] = f2_pack(fmaf(x.x, cx, -(x.y * sx)), fmaf(x.x, sx, x.y * cx));
        b.e[i] = f2_pack(fmaf(y.x, cy, -(y.y * sy)), fmaf(y.x, sy, y.y * cy));
        continue;
      }
    }
    const auto cs = p_at<VE>(c, i), sn = p_at<VE>(s, i), x = a.e[i];
    a.e[i] = p_fma(x, cs, p_neg(p_mul(b.e[i], sn)));
    b.e[i] = p_fma(x, sn, p_mul(b.e[i], cs));
  }
}
template <typename T, int VE>
__device__ __forceinline__ void turn(Vec<T, VE>& x, Vec<T, VE>& y, const float (&c)[VE], const float (&s)[VE],
                                     int interleaved) {
  float a[VE], b[VE];
  widen<T, VE>(x, a);
  widen<T, VE>(y, b);
  turn<VE>(a, b, c, s, interleaved);
  narrow<T, VE>(a, x);
  narrow<T, VE>(b, y);
}

// Cosines and sines of VE pairs from column `pairs` on of a position's table row; NaN for a position outside the table.
template <int VE>
__device__ __forceinline__ void load_angles(const RotaryArgs& p, int pos, int pairs, float (&c)[VE], float (&s)[VE]) {
  const int rot = static_cast<int>(p.rot), half = rot / 2;
  if (pos < 0 || pos >= p.table_rows) {
#pragma unroll
    for (int i = 0; i < VE; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
    return;
  }
  const float* row = p.table + static_cast<long long>(pos) * rot + pairs;
  if constexpr (VE >= 4) {
#pragma unroll
    for (int i = 0; i < VE; i += 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(row + i));
      const float4 b = __ldg(reinterpret_cast<const float4*>(row + half + i));
      c[i] = a.x, c[i + 1] = a.y, c[i + 2] = a.z, c[i + 3] = a.w;
      s[i] = b.x, s[i + 1] = b.y, s[i + 2] = b.z, s[i + 3] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      c[i] = __ldg(row + i);
      s[i] = __ldg(row + half + i);
    }
  }
}

// A unit's two vectors by their first element, and its first pair's column in the table. Units of a head: `turned`
// ones first, then plain ones of what is not turned, the last of which may have one vector only.
struct Unit {
  int e0, e1, pairs;
  bool turned, second;
};
template <int VE>
__device__ __forceinline__ Unit unit_of(int unit, int turned, int rot, int dim, int interleaved) {
  Unit u;
  u.turned = unit < turned;
  u.second = true;
  u.pairs = VE * unit;
  if (u.turned) {
    u.e0 = interleaved ? 2 * VE * unit : VE * unit;
    u.e1 = interleaved ? u.e0 + VE : u.e0 + rot / 2;
  } else {
    u.e0 = rot + 2 * VE * (unit - turned);
    u.e1 = u.e0 + VE;
    u.second = u.e1 < dim;
  }
  return u;
}

// A token's page and its place in it; page -1 where its slot is none of the cache's.
struct Place {
  long long page, slot;
};
__device__ __forceinline__ Place place_of(const RotaryArgs& p, long long t) {
  Place at{-1, 0};
  if (p.slots == nullptr) return at;
  const long long n = __ldg(reinterpret_cast<const long long*>(p.slots) + t);
  if (n < 0 || n >= p.pages * p.block_size) return at;
  if (((n | p.block_size) >> 32) == 0) {
    at.page = static_cast<uint32_t>(n) / static_cast<uint32_t>(p.block_size);
  } else {
    at.page = n / p.block_size;
  }
  at.slot = n - at.page * p.block_size;
  return at;
}

inline bool on_grid(const void* ptr, int64_t vec, int elem, std::initializer_list<int64_t> strides) {
  if (ptr == nullptr) return true;
  if (reinterpret_cast<uintptr_t>(ptr) % (vec * elem) != 0) return false;
  for (int64_t s : strides)
    if (s % vec != 0) return false;
  return true;
}

// Whether heads, halves, table rows and strides hold whole vectors of VE elements.
template <typename T, int VE>
bool whole_vectors(const RotaryArgs& a) {
  const int elem = static_cast<int>(sizeof(T));
  return a.dim % VE == 0 && a.rot % (2 * VE) == 0 &&
         (VE < 4 || reinterpret_cast<uintptr_t>(a.table) % 16 == 0) && on_grid(a.q, VE, elem, {a.sq_t, a.sq_h}) &&
         on_grid(a.q_out, VE, elem, {a.sqo_t, a.sqo_h}) && on_grid(a.k, VE, elem, {a.sk_t, a.sk_h}) &&
         on_grid(a.k_out, VE, elem, {a.sko_t, a.sko_h}) && on_grid(a.v, VE, elem, {a.sv_t, a.sv_h}) &&
         on_grid(a.k_cache, VE, elem, {a.skc_p, a.skc_h, a.skc_s}) &&
         on_grid(a.v_cache, VE, elem, {a.svc_p, a.svc_h, a.svc_s});
}

}  // namespace
}  // namespace kf
