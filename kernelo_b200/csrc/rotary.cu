// Rotary positions: each pair (a, b) of a head's first `rot` elements is turned
// by its position's angle,
//
//   a' = a cos - b sin,   b' = a sin + b cos   (sin negated for the inverse),
//
// pairs being (i, i + rot/2) or, interleaved, (2i, 2i + 1); the rest of the head
// is copied. cos and sin come from a table [position][rot] in fp32, made once in
// 64 bits (an angle of a late position keeps no bits as fp32 position x
// frequency); a position outside the table gives NaN, never a read outside it.
// The inverse is the gradient, since the rotation is orthogonal. With a cache,
// the turned k and the v of each token also go to its slot (none if negative).
//
// Bound by bytes: every element is read once and written once to each place.
#include <cuda.h>

#include <initializer_list>

#include "kf_common.cuh"
#include "kf_internal.h"

namespace kf {
namespace {

constexpr int ROTARY_THREADS = 256;

// A thread turns one unit of a token's heads: the two vectors of VE elements
// that hold VE pairs, or two plain vectors of the rest of the head.
template <typename T, int VE>
struct alignas(sizeof(T) * VE) Vec {
  T e[VE];
};

struct RotaryPlan {
  int units;         // per head: turned ones first, then plain ones
  int turned;
  int head_lanes;    // threads that share a token's heads, each taking every head_lanes-th
  int per_token;     // units * head_lanes
};

template <typename T, int VE>
__device__ __forceinline__ void turn(Vec<T, VE>& x, Vec<T, VE>& y, const float (&c)[VE], const float (&s)[VE],
                                     int interleaved) {
  if (interleaved && VE > 1) {
#pragma unroll
    for (int i = 0; i + 1 < VE; i += 2) {
      const float a = to_f32(x.e[i]), b = to_f32(x.e[i + 1]);
      x.e[i] = from_f32<T>(fmaf(a, c[i / 2], -(b * s[i / 2])));
      x.e[i + 1] = from_f32<T>(fmaf(a, s[i / 2], b * c[i / 2]));
      const float d = to_f32(y.e[i]), e = to_f32(y.e[i + 1]);
      y.e[i] = from_f32<T>(fmaf(d, c[(VE + i) / 2], -(e * s[(VE + i) / 2])));
      y.e[i + 1] = from_f32<T>(fmaf(d, s[(VE + i) / 2], e * c[(VE + i) / 2]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < VE; ++i) {
    const float a = to_f32(x.e[i]), b = to_f32(y.e[i]);
    x.e[i] = from_f32<T>(fmaf(a, c[i], -(b * s[i])));
    y.e[i] = from_f32<T>(fmaf(a, s[i], b * c[i]));
  }
}

template <typename T, int VE>
__global__ void __launch_bounds__(ROTARY_THREADS) rotary_kernel(const RotaryArgs p, const RotaryPlan plan) {
  using V = Vec<T, VE>;
  const long long at = static_cast<long long>(blockIdx.x) * ROTARY_THREADS + threadIdx.x;
  const long long t = at / plan.per_token;
  if (t >= p.tokens) return;
  const int rest = static_cast<int>(at - t * plan.per_token);
  const int unit = rest % plan.units, lane = rest / plan.units;
  const int rot = static_cast<int>(p.rot), half = rot / 2;

  // The unit's two vectors by their first element; `pairs` its table column.
  int e0, e1, pairs = 0;
  bool second = true;
  const bool turned = unit < plan.turned;
  if (turned) {
    e0 = p.interleaved ? 2 * VE * unit : VE * unit;
    e1 = p.interleaved ? e0 + VE : e0 + half;
    pairs = VE * unit;
  } else {
    e0 = rot + 2 * VE * (unit - plan.turned);
    e1 = e0 + VE;
    second = e1 < p.dim;
  }
  float c[VE], s[VE];
  if (turned) {
    const int pos = __ldg(p.positions + t);
    const bool known = pos >= 0 && pos < p.table_rows;
    const float* row = p.table + static_cast<long long>(known ? pos : 0) * rot + pairs;
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      c[i] = known ? __ldg(row + i) : __int_as_float(0x7fc00000);
      s[i] = known ? __ldg(row + half + i) : __int_as_float(0x7fc00000);
      if (p.inverse) s[i] = -s[i];
    }
  }
  long long page = -1, slot = 0;
  if (p.slots != nullptr) {
    const long long n = __ldg(reinterpret_cast<const long long*>(p.slots) + t);
    if (n >= 0 && n < p.pages * p.block_size) {
      page = n / p.block_size;
      slot = n - page * p.block_size;
    }
  }
  const int hq = static_cast<int>(p.heads), hk = static_cast<int>(p.kv_heads);
  const int all = hq + hk + (p.slots != nullptr ? hk : 0);
  for (int h = lane; h < all; h += plan.head_lanes) {
    const T* src;
    T *to, *cached = nullptr;
    bool turn_it = turned;
    if (h < hq) {
      src = static_cast<const T*>(p.q) + t * p.sq_t + h * p.sq_h;
      to = static_cast<T*>(p.q_out) + t * p.sqo_t + h * p.sqo_h;
    } else if (h < hq + hk) {
      const int g = h - hq;
      src = static_cast<const T*>(p.k) + t * p.sk_t + g * p.sk_h;
      to = p.k_out != nullptr ? static_cast<T*>(p.k_out) + t * p.sko_t + g * p.sko_h : nullptr;
      if (page >= 0) cached = static_cast<T*>(p.k_cache) + page * p.skc_p + g * p.skc_h + slot * p.skc_s;
    } else {
      const int g = h - hq - hk;
      src = static_cast<const T*>(p.v) + t * p.sv_t + g * p.sv_h;
      to = nullptr;
      if (page >= 0) cached = static_cast<T*>(p.v_cache) + page * p.svc_p + g * p.svc_h + slot * p.svc_s;
      turn_it = false;
    }
    if (to == nullptr && cached == nullptr) continue;
    V x = *reinterpret_cast<const V*>(src + e0), y{};
    if (second) y = *reinterpret_cast<const V*>(src + e1);
    if (turn_it) turn<T, VE>(x, y, c, s, p.interleaved);
    if (to != nullptr) {
      *reinterpret_cast<V*>(to + e0) = x;
      if (second) *reinterpret_cast<V*>(to + e1) = y;
    }
    if (cached != nullptr) {
      *reinterpret_cast<V*>(cached + e0) = x;
      if (second) *reinterpret_cast<V*>(cached + e1) = y;
    }
  }
}

bool on_grid(const void* ptr, int64_t vec, int elem, std::initializer_list<int64_t> strides) {
  if (ptr == nullptr) return true;
  if (reinterpret_cast<uintptr_t>(ptr) % (vec * elem) != 0) return false;
  for (int64_t s : strides)
    if (s % vec != 0) return false;
  return true;
}

template <typename T, int VE>
int launch_typed(const RotaryArgs& a, cudaStream_t stream) {
  RotaryPlan plan;
  plan.turned = static_cast<int>(a.rot / 2 / VE);
  plan.units = plan.turned + static_cast<int>(ceil_div(a.dim - a.rot, 2 * VE));
  plan.head_lanes = 1;
  plan.per_token = plan.units * plan.head_lanes;
  const int64_t blocks = ceil_div(a.tokens * plan.per_token, ROTARY_THREADS);
  if (blocks > 0x7fffffffll) return set_error(KF_ERR_UNSUPPORTED, "rotary: tokens beyond the grid");
  rotary_kernel<T, VE><<<static_cast<unsigned>(blocks), ROTARY_THREADS, 0, stream>>>(a, plan);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(rotary)");
}

template <typename T>
int pick(const RotaryArgs& a, cudaStream_t stream) {
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  const int elem = static_cast<int>(sizeof(T));
  // 16-byte vectors where heads, halves and strides hold whole ones; the turned
  // part is VE pairs a unit in both layouts
  const bool whole = a.dim % VE == 0 && a.rot % (2 * VE) == 0 && on_grid(a.q, VE, elem, {a.sq_t, a.sq_h}) &&
                     on_grid(a.q_out, VE, elem, {a.sqo_t, a.sqo_h}) && on_grid(a.k, VE, elem, {a.sk_t, a.sk_h}) &&
                     on_grid(a.k_out, VE, elem, {a.sko_t, a.sko_h}) && on_grid(a.v, VE, elem, {a.sv_t, a.sv_h}) &&
                     on_grid(a.k_cache, VE, elem, {a.skc_p, a.skc_h, a.skc_s}) &&
                     on_grid(a.v_cache, VE, elem, {a.svc_p, a.svc_h, a.svc_s});
  return whole ? launch_typed<T, VE>(a, stream) : launch_typed<T, 1>(a, stream);
}

}  // namespace

int launch_rotary(const RotaryArgs& a, const DeviceInfo&, cudaStream_t stream) {
  switch (a.dtype) {
    case KF_FP16: return pick<__half>(a, stream);
    case KF_BF16: return pick<__nv_bfloat16>(a, stream);
    default: return pick<float>(a, stream);
  }
}

}  // namespace kf
