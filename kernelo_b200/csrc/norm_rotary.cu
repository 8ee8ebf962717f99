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
// Forward: bound by bytes. A group of lanes takes several heads of a token with one load of its angles, two heads'
// loads in flight. 8192 tokens of 32 query and 8 key heads of 128 bf16 with the cache written: 47 us, 4.7 TB/s (72% of
// a copy's rate; the turn alone, without norms, 42); 64 tokens 4.7 us. Operands and outputs pass through the cache as the
// first to leave it, weights and angles stay: alone 44.4 us where plain stores take 47.5, and what follows loses nothing
// (with the prompt's attention 468 us either way, four prompts of 512 38.3 and 38.7, a step of 64 59 to 61).
// Backward: rows (token, head) are dealt out in runs, those of q and of k apart, so that a thread sums its own
// columns of dw in registers over its rows, its next rows on their way to shared memory meanwhile; a
// block adds its groups, and a second small launch the blocks, each in a fixed order: no atomics, the
// same bits from call to call. 4096 tokens: 43-45 us (2.9 TB/s) with the sums: some 12 us for a block's begin and end (first
// angles and rows, sums, the second launch) and 7.5 for each 1024 tokens (4.2 TB/s; 16384 tokens 136 us). The latencies of
// a row's chain, with 16 warps resident to an SM, bound that part; issue slots are half used.
#include <cuda.h>

#include "kf_common.cuh"
#include "kf_internal.h"
#include "rotary.cuh"

namespace kf {
namespace {

constexpr int NORM_THREADS = 128;
constexpr int HEADS_EACH = 6;  // heads that a group takes with one load of its angles
constexpr int BATCH = 2;       // of them, whose loads are in flight together
constexpr int FWD_BLOCKS = 7;  // of an SM, for 72 registers (with plain accesses 49.3 us; 6 blocks 51.0, 8 65.3: spills)

// Lanes of a head, units in it (and turned ones); forward: heads side by side, tokens of a block, rounds through the heads.
struct NormPlan {
  int width, units, turned, lanes, tokens, rounds;
};

// Units that a lane holds where heads of up to NORM_ROTARY_MAX_DIM elements have no wider vectors.
template <int VE>
constexpr int UNITS_EACH = VE >= 4 ? 1 : NORM_ROTARY_MAX_DIM / 2 / VE / 32;

// Sum over the lanes of each head of a warp. All lanes of the warp take part, those without a head too: with shuffles
// among the lanes of one head alone the warp's heads may run one after another (4096 tokens of 64 heads of 80: 57 us
// where this takes 51).
__device__ __forceinline__ float group_sum(float v, int width) {
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Heads whose mean square with eps is beyond fp32 (never fp16's) are taken by this power of two less, and eps by its
// square: u does not change. (The mean is then 2^-20 at least, so a usual eps is nothing only once it is scaled as well.)
constexpr float FAR = 0x1p-70f;
template <typename T>
__device__ __forceinline__ bool too_far(float mean) {
  return sizeof(T) == 4 || DType<T>::code == KF_BF16 ? !(mean < __int_as_float(0x7f800000)) : false;
}

// One thread's part of a head: its units' elements and angles.
template <typename T, int VE>
struct Lane {
  static constexpr int U = UNITS_EACH<VE>;
  using V = Vec<T, VE>;
  Unit u[U];
  bool active[U];
  float c[U][VE], s[U][VE];

  __device__ __forceinline__ void init(const RotaryArgs& p, const NormPlan& plan, int lane) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int unit = lane + j * plan.width;
      active[j] = unit < plan.units;
      u[j] = unit_of<VE>(unit, plan.turned, static_cast<int>(p.rot), static_cast<int>(p.dim), p.interleaved);
    }
  }
  __device__ __forceinline__ void angles(const RotaryArgs& p, long long t) {
    if (p.rot == 0) return;
    const int pos = __ldg(p.positions + t);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (active[j] && u[j].turned) load_angles<VE>(p, pos, u[j].pairs, c[j], s[j]);
    }
  }
  // Vectors that a head does not have are zeros.
  template <bool COMMON = false>  // weights
  __device__ __forceinline__ void load(const T* head, V (&x)[U], V (&y)[U]) const {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const T *const at = head + u[j].e0, *const second = head + u[j].e1;
      if (active[j]) x[j] = COMMON ? load_common<V>(at) : load_once<V>(at);
      else x[j] = V{};
      if (active[j] && u[j].second) y[j] = COMMON ? load_common<V>(second) : load_once<V>(second);
      else y[j] = V{};
    }
  }
  __device__ __forceinline__ void store(T* head, const V (&x)[U], const V (&y)[U]) const {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if (active[j]) store_once(head + u[j].e0, x[j]);
      if (active[j] && u[j].second) store_once(head + u[j].e1, y[j]);
    }
  }
  // x, y: the head's vectors, left as its outputs.
  __device__ __forceinline__ void forward(V (&x)[U], V (&y)[U], const V (&wx)[U], const V (&wy)[U], float eps, float inv_dim,
                                          int width, int interleaved) const {
    float a[U][VE], b[U][VE], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      widen<T, VE>(x[j], a[j]);
      widen<T, VE>(y[j], b[j]);
#pragma unroll
      for (int i = 0; i < VE; ++i) sum = fmaf(a[j][i], a[j][i], fmaf(b[j][i], b[j][i], sum));
    }
    float mean = fmaf(group_sum(sum, width), inv_dim, eps);
    if (__any_sync(0xffffffffu, too_far<T>(mean))) {
      const bool far = too_far<T>(mean);
      const float less = far ? FAR : 1.0f;
      sum = 0.0f;
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          a[j][i] *= less, b[j][i] *= less;
          sum = fmaf(a[j][i], a[j][i], fmaf(b[j][i], b[j][i], sum));
        }
      mean = fmaf(group_sum(sum, width), inv_dim, eps * less * less);
    }
    const float r = rsqrtf(mean);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float wa[VE], wb[VE];
      widen<T, VE>(wx[j], wa);
      widen<T, VE>(wy[j], wb);
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
__global__ void __launch_bounds__(NORM_THREADS, FWD_BLOCKS)
    norm_rotary_kernel(const __grid_constant__ RotaryArgs p, const NormArgs n, const NormPlan plan) {
  using L = Lane<T, VE>;
  constexpr int U = L::U;
  const int width = plan.width, lanes = plan.lanes, group = threadIdx.x / width;
  const long long t = static_cast<long long>(blockIdx.x) * plan.tokens + group / lanes;
  const bool has_token = t < p.tokens && group / lanes < plan.tokens;
  L me;
  me.init(p, plan, threadIdx.x % width);
  const Place at = has_token ? place_of(p, t) : Place{-1, 0};
  // Heads of q, then of k, then of v: as far as they go anywhere.
  const int hq = static_cast<int>(p.heads), hk = static_cast<int>(p.kv_heads);
  const int normed = !has_token ? 0 : hq + (p.k_out != nullptr || at.page >= 0 ? hk : 0);
  const int all = normed + (at.page >= 0 ? hk : 0);
  const T* const q = static_cast<const T*>(p.q) + t * p.sq_t;
  const T* const k = static_cast<const T*>(p.k) + t * p.sk_t;
  const T* const v = static_cast<const T*>(p.v) + t * p.sv_t;
  if (has_token) me.angles(p, t);
  // (the same rounds for all groups of a warp)
  for (int round = 0; round < plan.rounds; ++round) {
    const int h0 = group % lanes + round * BATCH * lanes;
    typename L::V x[BATCH][U], y[BATCH][U];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = h0 + i * lanes;
      if (h < all) me.load(h < hq ? q + h * p.sq_h : h < normed ? k + (h - hq) * p.sk_h : v + (h - normed) * p.sv_h, x[i], y[i]);
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int h = h0 + i * lanes;
      if (__any_sync(0xffffffffu, h < normed)) {
        typename L::V wx[U], wy[U], ox[U], oy[U];  // weights from L1: all heads have them in common
        me.template load<true>(static_cast<const T*>(h < hq ? n.q_weight : n.k_weight), wx, wy);
#pragma unroll
        for (int j = 0; j < U; ++j) ox[j] = x[i][j], oy[j] = y[i][j];
        me.forward(ox, oy, wx, wy, n.eps, n.inv_dim, width, p.interleaved);
        if (h < normed) {
#pragma unroll
          for (int j = 0; j < U; ++j) x[i][j] = ox[j], y[i][j] = oy[j];
        }
      }
      if (h < min(hq, normed)) {
        me.store(static_cast<T*>(p.q_out) + t * p.sqo_t + h * p.sqo_h, x[i], y[i]);
      } else if (h < normed) {
        const int g = h - hq;
        if (p.k_out != nullptr) me.store(static_cast<T*>(p.k_out) + t * p.sko_t + g * p.sko_h, x[i], y[i]);
        if (at.page >= 0) me.store(static_cast<T*>(p.k_cache) + at.page * p.skc_p + g * p.skc_h + at.slot * p.skc_s, x[i], y[i]);
      } else if (h < all) {
        me.store(static_cast<T*>(p.v_cache) + at.page * p.svc_p + (h - normed) * p.svc_h + at.slot * p.svc_s, x[i], y[i]);
      }
    }
  }
}

// ---------------------------------------------------------------- gradient
// Rows (token, head) of q or of k in order, a run of them to each group of lanes. A thread's vectors of the next rows
// are on their way to its own places in shared memory (nobody else reads them: no barriers) while it computes.
constexpr int STAGES = 4;
// Blocks of an SM, and how many times as many the rows are dealt out to: those that run beside slower ones then end
// earlier. 4096 tokens of 40 heads of 128 bf16, in one comparison: 43.8 us; 1 wave 50.4, 4 waves 50.5; 3 blocks 44.4.
constexpr int GRAD_BLOCKS = 4, GRAD_WAVES = 2;

__device__ __forceinline__ void copy_async(uint32_t to, const void* from, int bytes) {
  if (bytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else if (bytes == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from) : "memory");
}

// `partial` gets a row of dim sums from each block, q's first. Blocks of the two kinds are mixed: those of k change
// token oftener, and a few SMs that had only those would end last.
template <typename T, int VE>
__global__ void __launch_bounds__(NORM_THREADS, GRAD_BLOCKS)
    norm_rotary_grad_kernel(const __grid_constant__ NormGradArgs a, const NormPlan plan, int q_blocks, int k_blocks) {
  using L = Lane<T, VE>;
  using V = typename L::V;
  constexpr int U = L::U;
  griddep_launch_dependents();  // the sums' blocks wait for this grid's end
  __shared__ __align__(16) V ring[STAGES][4][U][NORM_THREADS];
  static_assert(sizeof(ring) >= 2 * VE * U * NORM_THREADS * sizeof(float), "the sums lie in the ring when it is done");
  const RotaryArgs& p = a.rotary;  // q and k: the inputs; q_out and k_out: their gradients
  const int n_k = static_cast<int>(static_cast<long long>(blockIdx.x) * k_blocks / (q_blocks + k_blocks));  // in front
  const bool of_q = static_cast<int>(static_cast<long long>(blockIdx.x + 1) * k_blocks / (q_blocks + k_blocks)) == n_k;
  const int block = of_q ? blockIdx.x - n_k : n_k, blocks = of_q ? q_blocks : k_blocks;
  const T* const x_all = static_cast<const T*>(of_q ? p.q : p.k);
  const T* const d_all = static_cast<const T*>(of_q ? a.dq : a.dk);
  T* const out_all = static_cast<T*>(of_q ? p.q_out : p.k_out);
  const long long sx_t = of_q ? p.sq_t : p.sk_t, sx_h = of_q ? p.sq_h : p.sk_h;
  const long long sd_t = of_q ? a.sdq_t : a.sdk_t, sd_h = of_q ? a.sdq_h : a.sdk_h;
  const long long so_t = of_q ? p.sqo_t : p.sko_t, so_h = of_q ? p.sqo_h : p.sko_h;
  const int heads = static_cast<int>(of_q ? p.heads : p.kv_heads);
  const int width = plan.width, groups = NORM_THREADS / width, thread = threadIdx.x, group = thread / width;
  L me;
  me.init(p, plan, thread % width);
  using F = Floats<VE>;
  F wa[U], wb[U];
  {
    V wx[U], wy[U];
    me.template load<true>(static_cast<const T*>(of_q ? a.norm.q_weight : a.norm.k_weight), wx, wy);
#pragma unroll
    for (int j = 0; j < U; ++j) wa[j] = floats<T, VE>(wx[j]), wb[j] = floats<T, VE>(wy[j]);
  }
  // This group's run of rows, and the next one to fetch. (The rounds are the same for all groups of a warp.)
  const long long rows = p.tokens * heads, runs = static_cast<long long>(blocks) * groups;
  const long long run = static_cast<long long>(block) * groups + group;
  const long long first = rows / runs * run + min(rows % runs, run);
  const int mine = static_cast<int>(rows / runs + (run < rows % runs ? 1 : 0));
  const int rounds = static_cast<int>((rows + runs - 1) / runs);
  long long t = first / heads, t_next = t;
  int h = static_cast<int>(first - t * heads), h_next = h;
  const auto fetch = [&](int stage) {
    const T* const x = x_all + t_next * sx_t + h_next * sx_h;
    const T* const d = d_all + t_next * sd_t + h_next * sd_h;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const auto piece = [&](int which, const T* from) {
        V* const to = &ring[stage][which][j][thread];
        if constexpr (sizeof(V) >= 4) copy_async(smem_u32(to), from, sizeof(V));
        else *to = *reinterpret_cast<const V*>(from);
      };
      if (!me.active[j]) continue;
      piece(0, x + me.u[j].e0);
      piece(2, d + me.u[j].e0);
      if (!me.u[j].second) continue;
      piece(1, x + me.u[j].e1);
      piece(3, d + me.u[j].e1);
    }
    if (++h_next == heads) h_next = 0, ++t_next;
  };
  // places that no row fills are zeros, and those of a group that has no row left are as an earlier row left them
#pragma unroll
  for (int s = 0; s < STAGES; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < U; ++j) ring[s][i][j][thread] = V{};
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (s < mine) fetch(s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  F sum_a[U], sum_b[U];
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int i = 0; i < F::N; ++i) sum_a[j].e[i] = sum_b[j].e[i] = p_splat<VE>(0.0f);
  long long angles_of = -1;
  for (int r = 0; r < rounds; ++r) {
    const bool here = r < mine;  // not in the last round, it may be: zeros then
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    if (here && t != angles_of) {
      me.angles(p, t);
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int i = 0; i < VE; ++i) me.s[j][i] = -me.s[j][i];  // the turn back
      angles_of = t;
    }
    const int stage = r % STAGES;
    F xa[U], xb[U], ga[U], gb[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      xa[j] = floats<T, VE>(ring[stage][0][j][thread]), xb[j] = floats<T, VE>(ring[stage][1][j][thread]);
      V gx = ring[stage][2][j][thread], gy = ring[stage][3][j][thread];
      if (!here) gx = gy = V{};
      ga[j] = floats<T, VE>(gx), gb[j] = floats<T, VE>(gy);
    }
    // into the places that were read in the last round
    if (r + STAGES - 1 < mine) fetch((r + STAGES - 1) % STAGES);
    asm volatile("cp.async.commit_group;" ::: "memory");
    // This lane's sums of x^2 and of g w x.
    const auto sums_of = [&](float& square, float& along) {
      auto xx = p_splat<VE>(0.0f), gwx = p_splat<VE>(0.0f);
#pragma unroll
      for (int j = 0; j < U; ++j) {
#pragma unroll
        for (int i = 0; i < F::N; ++i) {
          xx = p_fma(xa[j].e[i], xa[j].e[i], p_fma(xb[j].e[i], xb[j].e[i], xx));
          gwx = p_fma(p_mul(ga[j].e[i], wa[j].e[i]), xa[j].e[i], p_fma(p_mul(gb[j].e[i], wb[j].e[i]), xb[j].e[i], gwx));
        }
      }
      square = group_sum(p_sum(xx), width);
      along = group_sum(p_sum(gwx), width);
    };
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (here && me.u[j].turned) turn<VE>(ga[j], gb[j], me.c[j], me.s[j], p.interleaved);
    float square, along, scale = 1.0f;
    sums_of(square, along);
    float mean = fmaf(square, a.norm.inv_dim, a.norm.eps);
    if (__any_sync(0xffffffffu, too_far<T>(mean))) {
      if (too_far<T>(mean)) scale = FAR;
      const auto less = p_splat<VE>(scale);
#pragma unroll
      for (int j = 0; j < U; ++j)
#pragma unroll
        for (int i = 0; i < F::N; ++i) xa[j].e[i] = p_mul(xa[j].e[i], less), xb[j].e[i] = p_mul(xb[j].e[i], less);
      sums_of(square, along);
      mean = fmaf(square, a.norm.inv_dim, a.norm.eps * scale * scale);
    }
    const float inv = rsqrtf(mean);
    const float inv_true = inv * scale;                            // 1 / s
    const float back = along * inv * a.norm.inv_dim * inv_true;  // mean(g w u) / s
    const auto inv2 = p_splat<VE>(inv), true2 = p_splat<VE>(inv_true), back2 = p_splat<VE>(-back);
    V x[U], y[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
#pragma unroll
      for (int i = 0; i < F::N; ++i) {
        const auto ua = p_mul(xa[j].e[i], inv2), ub = p_mul(xb[j].e[i], inv2);
        sum_a[j].e[i] = p_fma(ga[j].e[i], ua, sum_a[j].e[i]);
        sum_b[j].e[i] = p_fma(gb[j].e[i], ub, sum_b[j].e[i]);
        xa[j].e[i] = p_fma(p_mul(ga[j].e[i], wa[j].e[i]), true2, p_mul(ua, back2));
        xb[j].e[i] = p_fma(p_mul(gb[j].e[i], wb[j].e[i]), true2, p_mul(ub, back2));
      }
      narrow<T, VE>(xa[j], x[j]);
      narrow<T, VE>(xb[j], y[j]);
    }
    if (here) me.store(out_all + t * so_t + h * so_h, x, y);
    if (++h == heads) h = 0, ++t;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // The block's groups of lanes, one after another.
  float* const sums = reinterpret_cast<float*>(ring);
  const int row = 2 * VE * U * width;  // of a group: [unit of the lane][lane][first and second vector]
#pragma unroll
  for (int j = 0; j < U; ++j)
#pragma unroll
    for (int i = 0; i < F::N; ++i) {
      auto* const at = reinterpret_cast<typename F::E*>(sums + group * row + (j * width + thread % width) * 2 * VE);
      at[i] = sum_a[j].e[i];
      at[F::N + i] = sum_b[j].e[i];
    }
  __syncthreads();
  float* const partial = a.partial + static_cast<long long>(of_q ? block : q_blocks + block) * p.dim;
  for (int e = thread; e < row; e += width * groups) {
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
  griddep_wait();
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
  plan.rounds = static_cast<int>(ceil_div(all, BATCH * plan.lanes));
  const int64_t blocks = ceil_div(a.tokens, plan.tokens);
  if (blocks > 0x7fffffffll) return set_error(KF_ERR_UNSUPPORTED, "norm_rotary: tokens beyond the grid");
  norm_rotary_kernel<T, VE><<<static_cast<unsigned>(blocks), NORM_THREADS, 0, stream>>>(a, n, plan);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(norm_rotary)");
}

template <typename T>
int pick(const RotaryArgs& a, const NormArgs& n, const DeviceInfo& dev, cudaStream_t stream) {
  return widest<T>([&](auto ve) { return whole<T, decltype(ve)::value>(a, n); },
                   [&](auto ve) { return launch_typed<T, decltype(ve)::value>(a, n, dev, stream); });
}

// Blocks of the gradient, shared out by heads; fewer where each of their groups would have less than ROWS_EACH rows.
constexpr int ROWS_EACH = 4;
struct GradBlocks {
  int q, k;
};
GradBlocks grad_blocks(int64_t tokens, int64_t heads, int64_t kv_heads, int groups, int sm_count) {
  const int64_t resident = static_cast<int64_t>(GRAD_BLOCKS) * GRAD_WAVES * sm_count;
  auto share = [&](int64_t mine) -> int {
    const int64_t n = ceil_div(resident * mine, heads + kv_heads > 0 ? heads + kv_heads : 1);
    const int64_t most = ceil_div(tokens * mine, ROWS_EACH * groups);
    return static_cast<int>(n < most ? n : most);
  };
  return {share(heads), share(kv_heads)};
}

template <typename T, int VE>
int launch_grad_typed(const NormGradArgs& a, const DeviceInfo& dev, GradBlocks* used, cudaStream_t stream) {
  const NormPlan plan = head_plan<VE>(a.rotary);
  const RotaryArgs& r = a.rotary;
  const GradBlocks blocks = *used = grad_blocks(r.tokens, r.heads, r.kv_heads, NORM_THREADS / plan.width, dev.sm_count);
  norm_rotary_grad_kernel<T, VE><<<static_cast<unsigned>(blocks.q + blocks.k), NORM_THREADS, 0, stream>>>(a, plan, blocks.q, blocks.k);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(norm_rotary gradient)");
}

template <typename T>
int pick_grad(const NormGradArgs& a, const DeviceInfo& dev, GradBlocks* used, cudaStream_t stream) {
  const int elem = static_cast<int>(sizeof(T));
  return widest<T>(
      [&](auto ve) {
        constexpr int VE = decltype(ve)::value;
        return whole<T, VE>(a.rotary, a.norm) && on_grid(a.dq, VE, elem, {a.sdq_t, a.sdq_h}) &&
               on_grid(a.dk, VE, elem, {a.sdk_t, a.sdk_h});
      },
      [&](auto ve) { return launch_grad_typed<T, decltype(ve)::value>(a, dev, used, stream); });
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
  const GradBlocks blocks = grad_blocks(tokens, heads, kv_heads, NORM_THREADS / 32, dev.sm_count);  // the most that are used
  return static_cast<int64_t>(blocks.q + blocks.k) * dim * 4;
}

int launch_norm_rotary_grad(const NormGradArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  const RotaryArgs& r = a.rotary;
  GradBlocks blocks{0, 0};
  if (r.tokens > 0 && r.heads + r.kv_heads > 0) {
    int rc;
    switch (r.dtype) {
      case KF_FP16: rc = pick_grad<__half>(a, dev, &blocks, stream); break;
      case KF_BF16: rc = pick_grad<__nv_bfloat16>(a, dev, &blocks, stream); break;
      default: rc = pick_grad<float>(a, dev, &blocks, stream); break;
    }
    if (rc != KF_OK) return rc;
  }
  const unsigned columns = static_cast<unsigned>(ceil_div(r.dim, 32));
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(2 * columns);
  config.blockDim = dim3(32, SUM_ROWS);
  config.stream = stream;
  cudaLaunchAttribute behind{};
  behind.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  behind.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &behind;
  config.numAttrs = blocks.q + blocks.k > 0 ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&config, norm_weight_sum_kernel, static_cast<const float*>(a.partial), blocks.q,
                                             blocks.k, static_cast<int>(r.dim), a.q_weight_grad, a.k_weight_grad);
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(norm weight sums)");
}

}  // namespace kf
