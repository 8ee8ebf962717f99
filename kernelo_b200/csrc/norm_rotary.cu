// Norms of each head of q and k with the rotary turn (and the cache write) in
// one pass, and the gradient of both in one pass.
//
//   y = R_p (w u),   u = x / s,   s = sqrt(mean x^2 + eps)   per head of dim elements
//
// with R_p the turn of rotary.cu (elements behind `rot` are not turned), w one
// weight for all heads of q and one for those of k, everything in fp32 and rounded
// once. Backward, with g = R_p^T dy (the turn back):
//
//   dx = (g w - u mean(g w u)) / s,   dw = sum over tokens and heads of g u.
//
// A head is held by a power of two of lanes, each with the two vectors of a unit
// (rotary.cuh), so that the sums are shuffles among them and nothing is read twice.
//
// Bound by bytes. Forward: a group of lanes takes several heads of a token with one load
// of its angles, two heads' loads in flight. Backward: the blocks that are resident at once
// share the tokens, those of q and those of k apart, so that a thread sums its own
// columns of dw in registers over all of its heads and tokens; a block adds its
// groups in shared memory, and a second small launch the blocks, each in a
// fixed order: no atomics, the same bits from call to call.
#include <cuda.h>

#include "kf_common.cuh"
#include "kf_internal.h"
#include "rotary.cuh"

namespace kf {
namespace {

constexpr int NORM_THREADS = 128;
constexpr int BATCH = 2;       // heads whose loads are in flight together
constexpr int HEADS_EACH = 6;  // heads that a group takes with one load of its angles

// Lanes of a head, units in it (and turned ones), heads side by side, tokens of a block.
struct NormPlan {
  int width, units, turned, lanes, tokens;
};

// Units that a lane holds where heads of up to NORM_ROTARY_MAX_DIM elements have no wider vectors.
template <int VE>
constexpr int UNITS_EACH = VE >= 4 ? 1 : NORM_ROTARY_MAX_DIM / 2 / VE / 32;

// The lanes of this thread's head.
__device__ __forceinline__ unsigned group_mask(int width) {
  const int thread = threadIdx.x + blockDim.x * (threadIdx.y + blockDim.y * threadIdx.z);
  const unsigned lanes = width == 32 ? 0xffffffffu : (1u << width) - 1;
  return lanes << (thread & 31 & ~(width - 1));
}
__device__ __forceinline__ float group_sum(float v, int width, unsigned mask) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
  return v;
}

// Elements whose squares' sum is beyond fp32 (never fp16's) are taken by this power of two less: u does not change, and
// eps is nothing beside them.
constexpr float FAR = 0x1p-70f;
template <typename T>
__device__ __forceinline__ bool too_far(float sum) {
  return sizeof(T) == 4 || DType<T>::code == KF_BF16 ? !(sum < __int_as_float(0x7f800000)) : false;
}

template <typename T, int VE>
struct HeadWeight {
  Vec<T, VE> first[UNITS_EACH<VE>], second[UNITS_EACH<VE>];
};

// One thread's part of a head: its units' elements and angles.
template <typename T, int VE>
struct Lane {
  static constexpr int U = UNITS_EACH<VE>;
  using V = Vec<T, VE>;
  Unit u[U];
  bool active[U];
  float c[U][VE], s[U][VE];

  __device__ __forceinline__ void init(const RotaryArgs& p, const NormPlan& plan) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int unit = threadIdx.x + j * plan.width;
      active[j] = unit < plan.units;
      u[j] = unit_of<VE>(unit, plan.turned, static_cast<int>(p.rot), static_cast<int>(p.dim), p.interleaved);
    }
  }
  template <bool BACK = false>
  __device__ __forceinline__ void angles(const RotaryArgs& p, long long t) {
    if (p.rot == 0) return;
    const int pos = __ldg(p.positions + t);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (!active[j] || !u[j].turned) continue;
      load_angles<VE>(p, pos, u[j].pairs, c[j], s[j]);
      if constexpr (BACK) {
#pragma unroll
        for (int i = 0; i < VE; ++i) s[j][i] = -s[j][i];
      }
    }
  }
  // Vectors that a head does not have are zeros.
  __device__ __forceinline__ void load(const T* head, V (&x)[U], V (&y)[U]) const {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (active[j]) x[j] = *reinterpret_cast<const V*>(head + u[j].e0);
      else x[j] = V{};
      if (active[j] && u[j].second) y[j] = *reinterpret_cast<const V*>(head + u[j].e1);
      else y[j] = V{};
    }
  }
  __device__ __forceinline__ void store(T* head, const V (&x)[U], const V (&y)[U]) const {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (active[j]) *reinterpret_cast<V*>(head + u[j].e0) = x[j];
      if (active[j] && u[j].second) *reinterpret_cast<V*>(head + u[j].e1) = y[j];
    }
  }
  // x, y: the head's vectors, left as its outputs.
  __device__ __forceinline__ void forward(V (&x)[U], V (&y)[U], const HeadWeight<T, VE>& w, float eps, float inv_dim,
                                          int width, unsigned mask, int interleaved) const {
    float a[U][VE], b[U][VE], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      widen<T, VE>(x[j], a[j]);
      widen<T, VE>(y[j], b[j]);
#pragma unroll
      for (int i = 0; i < VE; ++i) sum = fmaf(a[j][i], a[j][i], fmaf(b[j][i], b[j][i], sum));
    }
    sum = group_sum(sum, width, mask);
    if (too_far<T>(sum)) {
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          a[j][i] *= FAR, b[j][i] *= FAR;
          sum = fmaf(a[j][i], a[j][i], fmaf(b[j][i], b[j][i], sum));
        }
      sum = group_sum(sum, width, mask);
    }
    const float r = rsqrtf(fmaf(sum, inv_dim, eps));
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float wa[VE], wb[VE];
      widen<T, VE>(w.first[j], wa);
      widen<T, VE>(w.second[j], wb);
#pragma unroll
      for (int i = 0; i < VE; ++i) {
        a[j][i] = a[j][i] * r * wa[i];
        b[j][i] = b[j][i] * r * wb[i];
      }
      if (u[j].turned) turn<VE>(a[j], b[j], c[j], s[j], interleaved);
      narrow<T, VE>(a[j], x[j]);
      narrow<T, VE>(b[j], y[j]);
    }
  }
};

template <typename T, int VE>
__global__ void __launch_bounds__(NORM_THREADS, VE == 8 ? 5 : 4)
    norm_rotary_kernel(const __grid_constant__ RotaryArgs p, const NormArgs n, const NormPlan plan) {
  using L = Lane<T, VE>;
  constexpr int U = L::U;
  const long long t = static_cast<long long>(blockIdx.x) * plan.tokens + threadIdx.z;
  if (t >= p.tokens) return;  // a head's lanes have one token: they leave together
  const unsigned mask = group_mask(plan.width);
  const int width = plan.width;
  L me;
  me.init(p, plan);
  me.angles(p, t);
  HeadWeight<T, VE> w;
  const float eps = n.eps, inv_dim = n.inv_dim;
  const int hq = static_cast<int>(p.heads), hk = static_cast<int>(p.kv_heads), lanes = plan.lanes;
  int h = threadIdx.y;
  if (h < hq) {
    me.load(static_cast<const T*>(n.q_weight), w.first, w.second);
    const T* q = static_cast<const T*>(p.q) + t * p.sq_t;
    T* q_out = static_cast<T*>(p.q_out) + t * p.sqo_t;
    for (; h < hq; h += BATCH * lanes) {
      typename L::V x[BATCH][U], y[BATCH][U];
#pragma unroll
      for (int i = 0; i < BATCH; ++i)
        if (h + i * lanes < hq) me.load(q + (h + i * lanes) * p.sq_h, x[i], y[i]);
#pragma unroll
      for (int i = 0; i < BATCH; ++i) {
        if (h + i * lanes < hq) {
          me.forward(x[i], y[i], w, eps, inv_dim, width, mask, p.interleaved);
          me.store(q_out + (h + i * lanes) * p.sqo_h, x[i], y[i]);
        }
      }
    }
    // on with the heads of k where this group's stride left q
    while (h - lanes >= hq) h -= lanes;
  }
  const Place at = place_of(p, t);
  if (at.page < 0 && p.k_out == nullptr) return;
  if (h < hq + hk) me.load(static_cast<const T*>(n.k_weight), w.first, w.second);
  for (; h < hq + hk; h += lanes) {
    const int g = h - hq;
    typename L::V x[U], y[U];
    me.load(static_cast<const T*>(p.k) + t * p.sk_t + g * p.sk_h, x, y);
    me.forward(x, y, w, eps, inv_dim, width, mask, p.interleaved);
    if (p.k_out != nullptr) me.store(static_cast<T*>(p.k_out) + t * p.sko_t + g * p.sko_h, x, y);
    if (at.page >= 0)
      me.store(static_cast<T*>(p.k_cache) + at.page * p.skc_p + g * p.skc_h + at.slot * p.skc_s, x, y);
  }
  if (at.page < 0) return;
  for (; h < hq + 2 * hk; h += lanes) {
    const int g = h - hq - hk;
    typename L::V x[U], y[U];
    me.load(static_cast<const T*>(p.v) + t * p.sv_t + g * p.sv_h, x, y);
    me.store(static_cast<T*>(p.v_cache) + at.page * p.svc_p + g * p.svc_h + at.slot * p.svc_s, x, y);
  }
}

// ---------------------------------------------------------------- gradient
// Blocks of q first, then those of k. `partial` gets a row of dim sums from each.
template <typename T, int VE>
__global__ void __launch_bounds__(NORM_THREADS, 4)
    norm_rotary_grad_kernel(const __grid_constant__ NormGradArgs a, const NormPlan plan, int q_blocks, int k_blocks) {
  using L = Lane<T, VE>;
  constexpr int U = L::U;
  __shared__ float sums[2 * VE * U * NORM_THREADS];
  const RotaryArgs& p = a.rotary;  // q and k: the inputs; q_out and k_out: their gradients
  const bool of_q = static_cast<int>(blockIdx.x) < q_blocks;
  const int block = of_q ? blockIdx.x : blockIdx.x - q_blocks, blocks = of_q ? q_blocks : k_blocks;
  const T* const x_all = static_cast<const T*>(of_q ? p.q : p.k);
  const T* const d_all = static_cast<const T*>(of_q ? a.dq : a.dk);
  T* const out_all = static_cast<T*>(of_q ? p.q_out : p.k_out);
  const long long sx_t = of_q ? p.sq_t : p.sk_t, sx_h = of_q ? p.sq_h : p.sk_h;
  const long long sd_t = of_q ? a.sdq_t : a.sdk_t, sd_h = of_q ? a.sdq_h : a.sdk_h;
  const long long so_t = of_q ? p.sqo_t : p.sko_t, so_h = of_q ? p.sqo_h : p.sko_h;
  const int heads = static_cast<int>(of_q ? p.heads : p.kv_heads);
  const unsigned mask = group_mask(plan.width);
  // groups of lanes: heads side by side x tokens
  const int width = plan.width, group = threadIdx.y, groups = blockDim.y;
  const int lanes = min(heads, groups), tokens = groups / lanes, lane = group % lanes, token = group / lanes;
  L me;
  me.init(p, plan);
  HeadWeight<T, VE> w;
  me.load(static_cast<const T*>(of_q ? a.norm.q_weight : a.norm.k_weight), w.first, w.second);
  float wsum_a[U][VE] = {}, wsum_b[U][VE] = {};
  for (long long t = static_cast<long long>(block) * tokens + token; t < p.tokens && token < tokens;
       t += static_cast<long long>(blocks) * tokens) {
    me.template angles<true>(p, t);
    for (int h = lane; h < heads; h += lanes) {
      typename L::V x[U], y[U], dx[U], dy[U];
      me.load(x_all + t * sx_t + h * sx_h, x, y);
      me.load(d_all + t * sd_t + h * sd_h, dx, dy);
      float xa[U][VE], xb[U][VE], ga[U][VE], gb[U][VE], square = 0.0f, along = 0.0f;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        widen<T, VE>(x[j], xa[j]);
        widen<T, VE>(y[j], xb[j]);
        widen<T, VE>(dx[j], ga[j]);
        widen<T, VE>(dy[j], gb[j]);
        if (me.u[j].turned) turn<VE>(ga[j], gb[j], me.c[j], me.s[j], p.interleaved);
        float wa[VE], wb[VE];
        widen<T, VE>(w.first[j], wa);
        widen<T, VE>(w.second[j], wb);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          square = fmaf(xa[j][i], xa[j][i], fmaf(xb[j][i], xb[j][i], square));
          along = fmaf(ga[j][i] * wa[i], xa[j][i], fmaf(gb[j][i] * wb[i], xb[j][i], along));
        }
      }
      square = group_sum(square, width, mask);
      along = group_sum(along, width, mask);
      float scale = 1.0f;
      if (too_far<T>(square)) {
        scale = FAR, square = along = 0.0f;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          float wa[VE], wb[VE];
          widen<T, VE>(w.first[j], wa);
          widen<T, VE>(w.second[j], wb);
#pragma unroll
          for (int i = 0; i < VE; ++i) {
            xa[j][i] *= FAR, xb[j][i] *= FAR;
            square = fmaf(xa[j][i], xa[j][i], fmaf(xb[j][i], xb[j][i], square));
            along = fmaf(ga[j][i] * wa[i], xa[j][i], fmaf(gb[j][i] * wb[i], xb[j][i], along));
          }
        }
        square = group_sum(square, width, mask);
        along = group_sum(along, width, mask);
      }
      const float r = rsqrtf(fmaf(square, a.norm.inv_dim, a.norm.eps));
      const float r_true = r * scale;                         // 1 / s
      const float back = along * r * a.norm.inv_dim * r_true;  // mean(g w u) / s
#pragma unroll
      for (int j = 0; j < U; ++j) {
        float wa[VE], wb[VE];
        widen<T, VE>(w.first[j], wa);
        widen<T, VE>(w.second[j], wb);
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          const float ua = xa[j][i] * r, ub = xb[j][i] * r;
          wsum_a[j][i] = fmaf(ga[j][i], ua, wsum_a[j][i]);
          wsum_b[j][i] = fmaf(gb[j][i], ub, wsum_b[j][i]);
          xa[j][i] = fmaf(ga[j][i] * wa[i], r_true, -(ua * back));
          xb[j][i] = fmaf(gb[j][i] * wb[i], r_true, -(ub * back));
        }
        narrow<T, VE>(xa[j], x[j]);
        narrow<T, VE>(xb[j], y[j]);
      }
      me.store(out_all + t * so_t + h * so_h, x, y);
    }
  }
  // The block's groups of lanes, one after another.
  const int row = 2 * VE * U * width;  // of a group: [unit of the lane][lane][first and second vector]
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      float* const at = sums + group * row + (j * width + threadIdx.x) * 2 * VE;
      at[i] = wsum_a[j][i];
      at[VE + i] = wsum_b[j][i];
    }
  __syncthreads();
  float* const partial = a.partial + static_cast<long long>(blockIdx.x) * p.dim;
  const int thread = threadIdx.x + width * group, threads = width * groups;
  for (int e = thread; e < row; e += threads) {
    const Unit u = unit_of<VE>(e / (2 * VE), plan.turned, static_cast<int>(p.rot), static_cast<int>(p.dim), p.interleaved);
    const int in = e % (2 * VE);
    if (e / (2 * VE) >= plan.units || (in >= VE && !u.second)) continue;
    float sum = 0.0f;
    for (int g = 0; g < groups; ++g) sum += sums[g * row + e];
    partial[in < VE ? u.e0 + in : u.e1 + in - VE] = sum;
  }
}

// Sums of the blocks' rows, 32 columns to a block; the first half of the grid q's.
constexpr int SUM_ROWS = 32;
__global__ void __launch_bounds__(32 * SUM_ROWS)
    norm_weight_sum_kernel(const float* __restrict__ partial, int q_blocks, int k_blocks, int dim, float* q_grad, float* k_grad) {
  __shared__ float sums[SUM_ROWS][33];
  const int half = gridDim.x / 2;
  const bool of_q = static_cast<int>(blockIdx.x) < half;
  const int column = (of_q ? blockIdx.x : blockIdx.x - half) * 32 + threadIdx.x;
  const float* rows = partial + (of_q ? 0ll : static_cast<long long>(q_blocks) * dim);
  const int n = of_q ? q_blocks : k_blocks;
  float sum = 0.0f;
  if (column < dim) {
#pragma unroll 4
    for (int r = threadIdx.y; r < n; r += SUM_ROWS) sum += rows[static_cast<long long>(r) * dim + column];
  }
  sums[threadIdx.y][threadIdx.x] = sum;
  __syncthreads();
  // lane i of warp w now holds row i's sum of column w
  sum = sums[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int mine = (of_q ? blockIdx.x : blockIdx.x - half) * 32 + threadIdx.y;
  if (threadIdx.x == 0 && mine < dim) (of_q ? q_grad : k_grad)[mine] = sum;
}

template <typename T, int VE>
bool whole(const RotaryArgs& a, const NormArgs& n) {
  const int elem = static_cast<int>(sizeof(T));
  return whole_vectors<T, VE>(a) && on_grid(n.q_weight, VE, elem, {}) && on_grid(n.k_weight, VE, elem, {});
}

// Calls f(VE) with the widest vectors that fit.
template <typename T, typename Fits, typename Launch>
int widest(const Fits& fits, const Launch& launch) {
  if constexpr (sizeof(T) == 2)
    if (fits(std::integral_constant<int, 8>{})) return launch(std::integral_constant<int, 8>{});
  if (fits(std::integral_constant<int, 4>{})) return launch(std::integral_constant<int, 4>{});
  if (fits(std::integral_constant<int, 2>{})) return launch(std::integral_constant<int, 2>{});
  return launch(std::integral_constant<int, 1>{});
}

template <int VE>
NormPlan head_plan(const RotaryArgs& a) {
  NormPlan plan{};
  plan.turned = static_cast<int>(a.rot / 2 / VE);
  plan.units = plan.turned + static_cast<int>(ceil_div(a.dim - a.rot, 2 * VE));
  plan.width = 1;
  while (plan.width < 32 && plan.width < plan.units) plan.width *= 2;
  return plan;
}

template <typename T, int VE>
int launch_typed(const RotaryArgs& a, const NormArgs& n, const DeviceInfo& dev, cudaStream_t stream) {
  NormPlan plan = head_plan<VE>(a);
  // Heads side by side: HEADS_EACH heads a group, or one where that leaves the GPU without threads to cover its latency.
  const int64_t all = a.heads + a.kv_heads * (a.slots != nullptr ? 2 : 1);
  const bool few = a.tokens * plan.width * ceil_div(all, HEADS_EACH) < static_cast<int64_t>(dev.sm_count) * 1024;
  const int64_t most = NORM_THREADS / plan.width, lanes = few ? all : ceil_div(all, HEADS_EACH);
  plan.lanes = static_cast<int>(lanes < most ? lanes : most);
  plan.tokens = NORM_THREADS / (plan.width * plan.lanes);
  if (plan.tokens > 64) plan.tokens = 64;  // the limit of a block's third extent
  const int64_t blocks = ceil_div(a.tokens, plan.tokens);
  if (blocks > 0x7fffffffll) return set_error(KF_ERR_UNSUPPORTED, "norm_rotary: tokens beyond the grid");
  norm_rotary_kernel<T, VE><<<static_cast<unsigned>(blocks), dim3(plan.width, plan.lanes, plan.tokens), 0, stream>>>(
      a, n, plan);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(norm_rotary)");
}

template <typename T>
int pick(const RotaryArgs& a, const NormArgs& n, const DeviceInfo& dev, cudaStream_t stream) {
  return widest<T>([&](auto ve) { return whole<T, decltype(ve)::value>(a, n); },
                   [&](auto ve) { return launch_typed<T, decltype(ve)::value>(a, n, dev, stream); });
}

// Blocks of the gradient: as many as are resident at once, shared out by heads; from the sizes alone.
struct GradBlocks {
  int q, k;
};
GradBlocks grad_blocks(int64_t tokens, int64_t heads, int64_t kv_heads, int sm_count) {
  const int64_t resident = 4ll * sm_count;
  auto share = [&](int64_t mine) -> int {
    if (mine == 0 || tokens == 0) return 0;
    const int64_t n = ceil_div(resident * mine, heads + kv_heads);
    return static_cast<int>(n < tokens ? n : tokens);
  };
  return {share(heads), share(kv_heads)};
}

template <typename T, int VE>
int launch_grad_typed(const NormGradArgs& a, const GradBlocks& blocks, cudaStream_t stream) {
  const NormPlan plan = head_plan<VE>(a.rotary);
  norm_rotary_grad_kernel<T, VE><<<static_cast<unsigned>(blocks.q + blocks.k), dim3(plan.width, NORM_THREADS / plan.width), 0,
                                   stream>>>(a, plan, blocks.q, blocks.k);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(norm_rotary gradient)");
}

template <typename T>
int pick_grad(const NormGradArgs& a, const GradBlocks& blocks, cudaStream_t stream) {
  const int elem = static_cast<int>(sizeof(T));
  return widest<T>(
      [&](auto ve) {
        constexpr int VE = decltype(ve)::value;
        return whole<T, VE>(a.rotary, a.norm) && on_grid(a.dq, VE, elem, {a.sdq_t, a.sdq_h}) &&
               on_grid(a.dk, VE, elem, {a.sdk_t, a.sdk_h});
      },
      [&](auto ve) { return launch_grad_typed<T, decltype(ve)::value>(a, blocks, stream); });
}

}  // namespace

int launch_norm_rotary(const RotaryArgs& a, const NormArgs& n, const DeviceInfo& dev, cudaStream_t stream) {
  switch (a.dtype) {
    case KF_FP16: return pick<__half>(a, n, dev, stream);
    case KF_BF16: return pick<__nv_bfloat16>(a, n, dev, stream);
    default: return pick<float>(a, n, dev, stream);
  }
}

int64_t norm_rotary_grad_workspace_bytes(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim,
                                         const DeviceInfo& dev) {
  const GradBlocks blocks = grad_blocks(tokens, heads, kv_heads, dev.sm_count);
  return static_cast<int64_t>(blocks.q + blocks.k) * dim * 4;
}

int launch_norm_rotary_grad(const NormGradArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  const RotaryArgs& r = a.rotary;
  const GradBlocks blocks = grad_blocks(r.tokens, r.heads, r.kv_heads, dev.sm_count);
  if (blocks.q + blocks.k > 0) {
    int rc;
    switch (r.dtype) {
      case KF_FP16: rc = pick_grad<__half>(a, blocks, stream); break;
      case KF_BF16: rc = pick_grad<__nv_bfloat16>(a, blocks, stream); break;
      default: rc = pick_grad<float>(a, blocks, stream); break;
    }
    if (rc != KF_OK) return rc;
  }
  const unsigned columns = static_cast<unsigned>(ceil_div(r.dim, 32));
  norm_weight_sum_kernel<<<2 * columns, dim3(32, SUM_ROWS), 0, stream>>>(a.partial, blocks.q, blocks.k,
                                                                       static_cast<int>(r.dim), a.q_weight_grad,
                                                                       a.k_weight_grad);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(norm weight sums)");
}

}  // namespace kf
