// Attention, one warp per row and head, key by key: packed prompts and paged
// caches, every type, stride, head dimension up to 256 and mask.
//
//   o_i = sum_j p_ij v_j / l_i,  p_ij = 2^(s_ij - m_i),  s_ij = scale log2(e) q_i . k_j
//
// over the keys j that row i sees, in one pass with the running maximum m and
// sum l (fp32). A row reads its keys once itself, so the kernel is bound by its
// own instructions (about 30 a key): it is what the tile kernels do not take.
#include <cuda.h>

#include "attention.cuh"

namespace kf {
namespace {

constexpr int ROW_WARPS = 4;

template <typename T, int NE>
__global__ void __launch_bounds__(ROW_WARPS * 32) attention_rows_kernel(const AttnArgs p) {
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * ROW_WARPS + (threadIdx.x >> 5);
  if (unit >= p.rows * p.heads) return;
  const int t = static_cast<int>(unit / p.heads);
  const int head = static_cast<int>(unit - t * p.heads);
  float acc[NE], m, l;
  attend_row<T, NE>(p, t, head, lane, acc, &m, &l);
  write_row<T, NE>(p, t, head, lane, acc, m, l);
}

template <typename T>
int launch_typed(const AttnArgs& a, cudaStream_t stream) {
  const int64_t blocks = ceil_div(a.rows * a.heads, ROW_WARPS);
  if (blocks > 0x7fffffffll) return set_error(KF_ERR_UNSUPPORTED, "attention: rows x heads beyond the grid");
  const dim3 grid(static_cast<unsigned>(blocks)), block(ROW_WARPS * 32);
  if (a.dim <= 32) attention_rows_kernel<T, 1><<<grid, block, 0, stream>>>(a);
  else if (a.dim <= 64) attention_rows_kernel<T, 2><<<grid, block, 0, stream>>>(a);
  else if (a.dim <= 128) attention_rows_kernel<T, 4><<<grid, block, 0, stream>>>(a);
  else attention_rows_kernel<T, 8><<<grid, block, 0, stream>>>(a);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(attention_rows)");
}

}  // namespace

int launch_attention_rows(const AttnArgs& a, cudaStream_t stream) {
  switch (a.dtype) {
    case KF_FP16: return launch_typed<__half>(a, stream);
    case KF_BF16: return launch_typed<__nv_bfloat16>(a, stream);
    default: return launch_typed<float>(a, stream);
  }
}

}  // namespace kf
