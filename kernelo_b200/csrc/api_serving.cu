// extern "C" entry points of the serving operators: prompt attention, tree
// attention over a paged cache, rotary positions with the cache write, and
// block tables with slot maps. Argument checks here, kernels in their own files.
#include <cmath>
#include <string>

#include "kf_common.cuh"
#include "kf_internal.h"

namespace kf {
namespace {

int invalid(const std::string& message) { return set_error(KF_ERR_INVALID_ARGUMENT, message); }

bool known_dtype(int d) { return d == KF_FP16 || d == KF_BF16 || d == KF_FP32; }

int this_device(DeviceInfo** dev) {
  int device = 0;
  const int rc = current_device(&device);
  return rc != KF_OK ? rc : device_info(device, dev);
}

constexpr int64_t INT32_LIMIT = 0x7fffffffll;

int check_heads(int dtype, int64_t rows, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t dim) {
  if (!known_dtype(dtype)) return invalid("unknown dtype code");
  if (rows < 0 || seqs < 0 || heads < 0 || kv_heads < 0 || dim < 0) return invalid("negative size");
  if (rows > INT32_LIMIT || seqs > INT32_LIMIT) return invalid("rows and requests are counted in 32 bits");
  if (heads > 0 && (kv_heads == 0 || heads % kv_heads != 0))
    return invalid("query heads must be a multiple of key heads; got " + std::to_string(heads) + " and " +
                   std::to_string(kv_heads));
  if (dim > ATTN_MAX_DIM)
    return set_error(KF_ERR_UNSUPPORTED, "attention heads of at most " + std::to_string(ATTN_MAX_DIM) +
                                             " elements; got " + std::to_string(dim));
  return KF_OK;
}

}  // namespace
}  // namespace kf

using namespace kf;

extern "C" {

int32_t kf_prefill_attention(int32_t dtype, const void* q, int64_t sq_row, int64_t sq_head, const void* k,
                             int64_t sk_row, int64_t sk_head, const void* v, int64_t sv_row, int64_t sv_head,
                             void* out, int64_t so_row, int64_t so_head, float* lse, const int32_t* cu_q,
                             const int32_t* cu_k, int64_t seqs, int64_t rows, int64_t keys, int64_t heads,
                             int64_t kv_heads, int64_t dim, float scale, int32_t causal, void* stream) {
  int rc = check_heads(dtype, rows, seqs, heads, kv_heads, dim);
  if (rc != KF_OK) return rc;
  if (keys < 0 || keys > INT32_LIMIT) return invalid("keys are counted in 32 bits");
  if (!std::isfinite(scale)) return invalid("scale must be finite");
  if (rows == 0 || heads == 0 || dim == 0) return KF_OK;
  if (q == nullptr || out == nullptr || cu_q == nullptr || cu_k == nullptr ||
      (keys > 0 && (k == nullptr || v == nullptr)))
    return invalid("null pointer");
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  AttnArgs a;
  a.dtype = dtype;
  a.q = q, a.sq_t = sq_row, a.sq_h = sq_head;
  a.k = k, a.sk_t = sk_row, a.sk_h = sk_head;
  a.v = v, a.sv_t = sv_row, a.sv_h = sv_head;
  a.out = out, a.so_t = so_row, a.so_h = so_head;
  a.lse = lse;
  a.cu_q = cu_q, a.cu_k = cu_k;
  a.seqs = seqs, a.rows = rows, a.keys = keys, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.causal = causal != 0;
  if (attention_prefill_supported(a)) return launch_attention_prefill(a, *dev, static_cast<cudaStream_t>(stream));
  return launch_attention_rows(a, static_cast<cudaStream_t>(stream));
}

int32_t kf_tree_attention(int32_t dtype, const void* q, int64_t sq_row, int64_t sq_head, const void* k_cache,
                          int64_t sk_page, int64_t sk_head, int64_t sk_slot, const void* v_cache, int64_t sv_page,
                          int64_t sv_head, int64_t sv_slot, void* out, int64_t so_row, int64_t so_head, float* lse,
                          const int32_t* block_table, int64_t table_stride, int64_t table_cols, int64_t pages,
                          int64_t block_size, const int32_t* context, const int32_t* cu_q, const int64_t* tree_mask,
                          int64_t mask_words, int64_t seqs, int64_t rows, int64_t heads, int64_t kv_heads,
                          int64_t dim, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  int rc = check_heads(dtype, rows, seqs, heads, kv_heads, dim);
  if (rc != KF_OK) return rc;
  if (table_cols < 0 || pages < 0 || mask_words < 0) return invalid("negative size");
  if (block_size < 1 || block_size > INT32_LIMIT) return invalid("block_size must be positive and fit 32 bits");
  if (!std::isfinite(scale)) return invalid("scale must be finite");
  if (rows == 0 || heads == 0 || dim == 0) return KF_OK;
  if (q == nullptr || out == nullptr || (seqs > 0 && context == nullptr) ||
      (seqs > 0 && table_cols > 0 && block_table == nullptr) ||
      (pages > 0 && (k_cache == nullptr || v_cache == nullptr)) || (mask_words > 0 && tree_mask == nullptr))
    return invalid("null pointer");
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  AttnArgs a;
  a.dtype = dtype;
  a.q = q, a.sq_t = sq_row, a.sq_h = sq_head;
  a.k = k_cache, a.sk_p = sk_page, a.sk_h = sk_head, a.sk_t = sk_slot;
  a.v = v_cache, a.sv_p = sv_page, a.sv_h = sv_head, a.sv_t = sv_slot;
  a.out = out, a.so_t = so_row, a.so_h = so_head;
  a.lse = lse;
  a.cu_q = cu_q;
  a.paged = 1;
  a.table = block_table, a.table_stride = table_stride, a.table_cols = table_cols;
  a.pages = pages, a.block_size = block_size;
  a.context = context;
  a.mask = mask_words > 0 ? reinterpret_cast<const unsigned long long*>(tree_mask) : nullptr;
  a.mask_words = mask_words;
  a.seqs = seqs, a.rows = rows, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.workspace = workspace, a.workspace_bytes = workspace_bytes;
  if (attention_tree_supported(a)) return launch_attention_tree(a, *dev, static_cast<cudaStream_t>(stream));
  return launch_attention_rows(a, static_cast<cudaStream_t>(stream));
}

int64_t kf_tree_attention_workspace_bytes(int32_t device, int32_t dtype, int64_t seqs, int64_t rows, int64_t heads,
                                          int64_t kv_heads, int64_t dim) {
  int rc = check_heads(dtype, rows, seqs, heads, kv_heads, dim);
  if (rc != KF_OK) return -rc;
  if (heads == 0 || dtype == KF_FP32) return 0;
  DeviceInfo* dev = nullptr;
  rc = device_info(device, &dev);
  if (rc != KF_OK) return -rc;
  AttnArgs a;
  a.dtype = dtype;
  a.seqs = seqs, a.rows = rows, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
  return attention_tree_workspace_bytes(a, *dev);
}

int32_t kf_rotary(int32_t dtype, const void* q, int64_t sq_row, int64_t sq_head, void* q_out, int64_t sqo_row,
                  int64_t sqo_head, const void* k, int64_t sk_row, int64_t sk_head, void* k_out, int64_t sko_row,
                  int64_t sko_head, const int32_t* positions, const float* table, int64_t table_rows, int64_t rot,
                  int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim, int32_t interleaved, int32_t inverse,
                  const kf_rotary_cache* cache, void* stream) {
  if (!known_dtype(dtype)) return invalid("unknown dtype code");
  if (tokens < 0 || heads < 0 || kv_heads < 0 || dim < 0 || table_rows < 0 || rot < 0) return invalid("negative size");
  if (rot % 2 != 0 || rot > dim)
    return invalid("the turned part must be even and at most the head; got " + std::to_string(rot) + " of " +
                   std::to_string(dim));
  if (tokens == 0 || dim == 0 || heads + kv_heads == 0) return KF_OK;
  if ((heads > 0 && (q == nullptr || q_out == nullptr)) || (kv_heads > 0 && k == nullptr) ||
      (rot > 0 && (positions == nullptr || (table_rows > 0 && table == nullptr))))
    return invalid("null pointer");
  if (kv_heads > 0 && k_out == nullptr && cache == nullptr) return invalid("k needs an output or a cache");
  if (heads > INT32_LIMIT || kv_heads > INT32_LIMIT / 2 || dim > INT32_LIMIT / 4)
    return invalid("heads and their elements are counted in 32 bits");
  RotaryArgs a;
  a.dtype = dtype;
  a.q = q, a.sq_t = sq_row, a.sq_h = sq_head;
  a.q_out = q_out, a.sqo_t = sqo_row, a.sqo_h = sqo_head;
  a.k = k, a.sk_t = sk_row, a.sk_h = sk_head;
  a.k_out = k_out, a.sko_t = sko_row, a.sko_h = sko_head;
  a.positions = positions, a.table = table, a.table_rows = table_rows, a.rot = rot;
  if (cache != nullptr && kv_heads > 0) {
    if (cache->block_size < 1) return invalid("block_size must be positive");
    if (cache->pages < 0) return invalid("negative size");
    if (cache->v == nullptr || cache->slots == nullptr ||
        (cache->pages > 0 && (cache->k_cache == nullptr || cache->v_cache == nullptr)))
      return invalid("null pointer");
    a.v = cache->v, a.sv_t = cache->sv_row, a.sv_h = cache->sv_head;
    a.k_cache = cache->k_cache, a.skc_p = cache->sk_page, a.skc_h = cache->sk_head, a.skc_s = cache->sk_slot;
    a.v_cache = cache->v_cache, a.svc_p = cache->sv_page, a.svc_h = cache->svc_head, a.svc_s = cache->sv_slot;
    a.pages = cache->pages, a.block_size = cache->block_size;
    a.slots = cache->slots;
  }
  a.tokens = tokens, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
  a.interleaved = interleaved != 0, a.inverse = inverse != 0;
  DeviceInfo* dev = nullptr;
  const int rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  return launch_rotary(a, *dev, static_cast<cudaStream_t>(stream));
}

int32_t kf_build_slots(const int32_t* context, const int32_t* added, int64_t seqs, int32_t* block_table,
                       int64_t table_stride, int64_t table_cols, const int32_t* free_blocks, int64_t n_free,
                       int64_t block_size, int64_t max_tokens, int32_t* cu_new, int32_t* positions, int64_t* slots,
                       int32_t* counts, void* stream) {
  if (seqs < 0 || table_cols < 0 || n_free < 0 || max_tokens < 0) return invalid("negative size");
  if (max_tokens > INT32_LIMIT) return invalid("tokens are counted in 32 bits");
  if (block_size < 1) return invalid("block_size must be positive");
  if (cu_new == nullptr || counts == nullptr || (seqs > 0 && (context == nullptr || added == nullptr)) ||
      (seqs > 0 && table_cols > 0 && block_table == nullptr) || (n_free > 0 && free_blocks == nullptr) ||
      (max_tokens > 0 && (positions == nullptr || slots == nullptr)))
    return invalid("null pointer");
  DeviceInfo* dev = nullptr;
  const int rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  SlotsArgs a;
  a.context = context, a.added = added, a.seqs = seqs;
  a.table = block_table, a.table_stride = table_stride, a.table_cols = table_cols;
  a.free_blocks = free_blocks, a.n_free = n_free;
  a.block_size = block_size, a.max_tokens = max_tokens;
  a.cu_new = cu_new, a.positions = positions, a.slots = slots, a.counts = counts;
  return launch_slots(a, *dev, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
