// Attention, a warp or several per row and head: packed prompts and paged caches,
// every type, stride, head dimension up to 256 and mask.
//
//   o_i = sum_j p_ij v_j / l_i,  p_ij = 2^(s_ij - m_i),  s_ij = scale log2(e) q_i . k_j
//
// over the keys j that row i sees, in one pass with the running maximum m and
// sum l (fp32). A row reads its keys once itself, so the kernel is bound by its
// own instructions: it is what the tile kernels do not take. Where rows x heads
// leave the GPU without warps, up to 16 share a row's keys and join their sums in
// the order of the keys.
#include <cuda.h>

#include "attention.cuh"

namespace kf {
namespace {

constexpr int ROW_WARPS = 4;
constexpr int MAX_PARTS = 16;

template <typename T, int NE>
__global__ void __launch_bounds__(MAX_PARTS * 32) attention_rows_kernel(const __grid_constant__ AttnArgs p, int parts) {
  __shared__ float part_m[MAX_PARTS], part_l[MAX_PARTS];
  __shared__ float part_o[MAX_PARTS][NE * 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const long long unit = parts > 1 ? blockIdx.x : static_cast<long long>(blockIdx.x) * warps + warp;
  if (unit >= p.rows * p.heads) return;  // parts > 1: the whole block, or none of it
  const int t = static_cast<int>(unit / p.heads);
  const int head = static_cast<int>(unit - t * p.heads);
  float acc[NE], m, l;
  attend_row<T, NE, NE <= 4 ? 4 : 2>(p, t, head, lane, acc, &m, &l, parts > 1 ? warp : 0, parts);
  if (parts > 1) {
    if (lane == 0) {
      part_m[warp] = m;
      part_l[warp] = l;
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) part_o[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    if (warp > 0) return;
    for (int w = 1; w < parts; ++w) {
      const float other = part_m[w];
      if (other == -INFINITY && part_l[w] == 0.0f) continue;
      const float top = other > m ? other : m;
      const float fix = m == -INFINITY ? 0.0f : ex2_ftz(m - top), take = other == -INFINITY ? 1.0f : ex2_ftz(other - top);
      l = fmaf(l, fix, part_l[w] * take);
#pragma unroll
      for (int i = 0; i < NE; ++i) acc[i] = fmaf(acc[i], fix, part_o[w][lane + 32 * i] * take);
      m = top;
    }
  }
  write_row<T, NE>(p, t, head, lane, acc, m, l);
}

template <typename T>
int launch_typed(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t units = a.rows * a.heads;
  // warps to a row: as many as keep 16 on every SM busy, for caches (whose rows are few)
  int parts = 1;
  if (a.paged)
    while (parts < MAX_PARTS && units * parts * 2 <= 16ll * dev.sm_count) parts *= 2;
  const int64_t blocks = parts > 1 ? units : ceil_div(units, ROW_WARPS);
  if (blocks > 0x7fffffffll) return set_error(KF_ERR_UNSUPPORTED, "attention: rows x heads beyond the grid");
  const dim3 grid(static_cast<unsigned>(blocks)), block(32 * (parts > 1 ? parts : ROW_WARPS));
  if (a.dim <= 32) attention_rows_kernel<T, 1><<<grid, block, 0, stream>>>(a, parts);
  else if (a.dim <= 64) attention_rows_kernel<T, 2><<<grid, block, 0, stream>>>(a, parts);
  else if (a.dim <= 128) attention_rows_kernel<T, 4><<<grid, block, 0, stream>>>(a, parts);
  else attention_rows_kernel<T, 8><<<grid, block, 0, stream>>>(a, parts);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(attention_rows)");
}

}  // namespace

int launch_attention_rows(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  switch (a.dtype) {
    case KF_FP16: return launch_typed<__half>(a, dev, stream);
    case KF_BF16: return launch_typed<__nv_bfloat16>(a, dev, stream);
    default: return launch_typed<float>(a, dev, stream);
  }
}

}  // namespace kf
