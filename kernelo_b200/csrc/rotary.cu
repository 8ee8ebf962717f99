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
// Bound by bytes: every element is read once and written once to each place. A
// thread turns the two vectors (16 bytes each where layout and alignment allow)
// that hold its pairs for several heads: its cosines and sines are loaded once for
// all of them. 8192 tokens of 32 query and 8 key heads of 128 bf16 elements with the
// cache written: 42.5 us, 5.2 TB/s (80% of a copy's rate); 2048 tokens of 64 heads in
// fp32, inverse: 25.5 us, 5.3 TB/s; 64 tokens 3.0 us.
#include <cuda.h>

#include "kf_common.cuh"
#include "kf_internal.h"
#include "rotary.cuh"

namespace kf {
namespace {

constexpr int ROTARY_THREADS = 256;  // of a block at most
constexpr int BATCH = 2;       // heads whose loads are in flight together (4: 84 us for 8192 tokens, with spills)
constexpr int HEADS_EACH = 6;  // that a thread turns with one load of its angles

// Threads of a block: units of a head (turned ones first, then plain ones) x
// heads side by side x tokens.
struct RotaryPlan {
  int units, turned, lanes, tokens;
};

template <typename T, int VE>
__global__ void __launch_bounds__(ROTARY_THREADS, 4)
    rotary_kernel(const __grid_constant__ RotaryArgs p, const RotaryPlan plan) {
  using V = Vec<T, VE>;
  const long long t = static_cast<long long>(blockIdx.x) * plan.tokens + threadIdx.z;
  if (t >= p.tokens) return;
  const Unit u = unit_of<VE>(threadIdx.x, plan.turned, static_cast<int>(p.rot), static_cast<int>(p.dim), p.interleaved);
  const int e0 = u.e0, e1 = u.e1;
  const bool turned = u.turned, second = u.second;
  float c[VE], s[VE];
  if (turned) {
    load_angles<VE>(p, __ldg(p.positions + t), u.pairs, c, s);
    if (p.inverse) {
#pragma unroll
      for (int i = 0; i < VE; ++i) s[i] = -s[i];
    }
  }
  const int hq = static_cast<int>(p.heads), hk = static_cast<int>(p.kv_heads), lanes = plan.lanes;
  int h = threadIdx.y;
  {
    const T* q = static_cast<const T*>(p.q) + t * p.sq_t;
    T* q_out = static_cast<T*>(p.q_out) + t * p.sqo_t;
    for (; h < hq; h += BATCH * lanes) {
      V x[BATCH], y[BATCH];
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (h + i * lanes < hq) {
          const T* from = q + (h + i * lanes) * p.sq_h;
          x[i] = *reinterpret_cast<const V*>(from + e0);
          if (second) y[i] = *reinterpret_cast<const V*>(from + e1);
        }
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (h + i * lanes < hq) {
          if (turned) turn<T, VE>(x[i], y[i], c, s, p.interleaved);
          T* to = q_out + (h + i * lanes) * p.sqo_h;
          *reinterpret_cast<V*>(to + e0) = x[i];
          if (second) *reinterpret_cast<V*>(to + e1) = y[i];
        }
      }
    }
    // on with the heads of k where this thread's stride left q
    while (h - lanes >= hq) h -= lanes;
  }
  const Place at = place_of(p, t);
  const long long page = at.page, slot = at.slot;
  if (page < 0 && p.k_out == nullptr) return;
  for (; h < hq + hk; h += lanes) {
    const int g = h - hq;
    const T* from = static_cast<const T*>(p.k) + t * p.sk_t + g * p.sk_h;
    V x = *reinterpret_cast<const V*>(from + e0), y;
    if (second) y = *reinterpret_cast<const V*>(from + e1);
    if (turned) turn<T, VE>(x, y, c, s, p.interleaved);
    if (p.k_out != nullptr) {
      T* to = static_cast<T*>(p.k_out) + t * p.sko_t + g * p.sko_h;
      *reinterpret_cast<V*>(to + e0) = x;
      if (second) *reinterpret_cast<V*>(to + e1) = y;
    }
    if (page >= 0) {
      T* to = static_cast<T*>(p.k_cache) + page * p.skc_p + g * p.skc_h + slot * p.skc_s;
      *reinterpret_cast<V*>(to + e0) = x;
      if (second) *reinterpret_cast<V*>(to + e1) = y;
    }
  }
  if (page < 0) return;
  for (; h < hq + 2 * hk; h += lanes) {
    const int g = h - hq - hk;
    const T* from = static_cast<const T*>(p.v) + t * p.sv_t + g * p.sv_h;
    T* to = static_cast<T*>(p.v_cache) + page * p.svc_p + g * p.svc_h + slot * p.svc_s;
    *reinterpret_cast<V*>(to + e0) = *reinterpret_cast<const V*>(from + e0);
    if (second) *reinterpret_cast<V*>(to + e1) = *reinterpret_cast<const V*>(from + e1);
  }
}

template <typename T, int VE>
int launch_typed(const RotaryArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t turned = a.rot / 2 / VE, units = turned + ceil_div(a.dim - a.rot, 2 * VE);
  if (units > ROTARY_THREADS) return set_error(KF_ERR_UNSUPPORTED, "rotary: heads too wide for their alignment");
  // Heads side by side: HEADS_EACH heads a thread, or one where that leaves the
  // GPU without threads to cover its latency (a decoding step: 64 tokens 3.0 us, 3.6 the
  // other way; 8192 tokens 42.5 us, 46.3 with one head a thread).
  const int64_t all = a.heads + a.kv_heads * (a.slots != nullptr ? 2 : 1);
  const bool few = a.tokens * units * ceil_div(all, HEADS_EACH) < static_cast<int64_t>(dev.sm_count) * 1024;
  RotaryPlan plan;
  plan.units = static_cast<int>(units);
  plan.turned = static_cast<int>(turned);
  // small blocks: a prompt of 8192 tokens 42.5 us, with blocks of 256 threads 44.0
  const int threads = units <= 128 ? 128 : ROTARY_THREADS;
  const int64_t most = threads / units;
  const int64_t lanes = few ? all : ceil_div(all, HEADS_EACH);
  plan.lanes = static_cast<int>(lanes < most ? lanes : most);
  plan.tokens = threads / (plan.units * plan.lanes);
  if (plan.tokens > 64) plan.tokens = 64;  // the limit of a block's third extent
  const int64_t blocks = ceil_div(a.tokens, plan.tokens);
  if (blocks > 0x7fffffffll) return set_error(KF_ERR_UNSUPPORTED, "rotary: tokens beyond the grid");
  rotary_kernel<T, VE><<<static_cast<unsigned>(blocks), dim3(plan.units, plan.lanes, plan.tokens), 0, stream>>>(a, plan);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(rotary)");
}

template <typename T>
int pick(const RotaryArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (whole_vectors<T, 8>(a)) return launch_typed<T, 8>(a, dev, stream);
  if (whole_vectors<T, 4>(a)) return launch_typed<T, 4>(a, dev, stream);
  if (whole_vectors<T, 2>(a)) return launch_typed<T, 2>(a, dev, stream);
  return launch_typed<T, 1>(a, dev, stream);
}

}  // namespace

int launch_rotary(const RotaryArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  switch (a.dtype) {
    case KF_FP16: return pick<__half>(a, dev, stream);
    case KF_BF16: return pick<__nv_bfloat16>(a, dev, stream);
    default: return pick<float>(a, dev, stream);
  }
}

}  // namespace kf
