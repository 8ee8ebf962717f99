// Tensor maps of the attention kernels' operands.
#include <cudaTypedefs.h>

#include <mutex>
#include <string>

#include "kf_internal.h"

namespace kf {
namespace {

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(sym);
  });
  return fn;
}

CUtensorMapDataType type_of(int dtype) {
  return dtype == KF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

}  // namespace

int encode_heads(CUtensorMap* map, int dtype, const void* ptr, int64_t rows, int64_t heads, int64_t dim, int64_t s_row,
                 int64_t s_head, int box_heads, int box_rows) {
  auto enc = encoder();
  if (enc == nullptr) return set_error(KF_ERR_LAUNCH, "cuTensorMapEncodeTiled unavailable");
  // a dimension of one has no stride to speak of
  const auto bytes = [](int64_t s, int64_t n) { return static_cast<cuuint64_t>(n > 1 ? 2 * s : 16); };
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {bytes(s_head, heads), bytes(s_row, rows)};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_rows)}, unit[3] = {1, 1, 1};
  const CUresult r = enc(map, type_of(dtype), 3, const_cast<void*>(ptr), dims, strides, box, unit,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(KF_ERR_UNALIGNED, "attention: cuTensorMapEncodeTiled rejected an operand (error " +
                                           std::to_string(r) + ")");
  return KF_OK;
}

bool encode_pages(CUtensorMap* map, const AttnArgs& a, const void* ptr, int64_t s_page, int64_t s_head, int64_t s_slot,
                  int box_rows, int width) {
  auto enc = encoder();
  if (enc == nullptr) return false;
  // strides outside of what a tensor map may have are not left to the encoder to find: a head or
  // a page that stands for several has one of zero
  const auto fits = [](int64_t s, int64_t n) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
  if (!fits(s_slot, a.block_size) || !fits(s_head, a.kv_heads) || !fits(s_page, a.pages)) return false;
  const auto bytes = [](int64_t s, int64_t n) { return static_cast<cuuint64_t>(n > 1 ? 2 * s : 16); };
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.block_size),
                              static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.pages)};
  const cuuint64_t strides[3] = {bytes(s_slot, a.block_size), bytes(s_head, a.kv_heads), bytes(s_page, a.pages)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(width), static_cast<cuuint32_t>(box_rows), 1, 1};
  const cuuint32_t unit[4] = {1, 1, 1, 1};
  return enc(map, type_of(a.dtype), 4, const_cast<void*>(ptr), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
             width == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace kf
