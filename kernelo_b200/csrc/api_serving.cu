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

bool known_dtype(int64_t d) { return d == KF_FP16 || d == KF_BF16 || d == KF_FP32; }

int this_device(DeviceInfo** dev) {
  int device = 0;
  const int rc = current_device(&device);
  return rc != KF_OK ? rc : device_info(device, dev);
}

constexpr double LOG2_E = 1.4426950408889634;
constexpr int64_t INT32_LIMIT = 0x7fffffffll;
// Rows, keys and requests: steps of up to 256 beyond the last one still fit 32 bits.
constexpr int64_t COUNT_LIMIT = 0x7fffff00ll;

int check_heads(int64_t dtype, int64_t rows, int64_t seqs, int64_t heads, int64_t kv_heads, int64_t dim) {
  if (!known_dtype(dtype)) return invalid("unknown dtype code");
  if (rows < 0 || seqs < 0 || heads < 0 || kv_heads < 0 || dim < 0) return invalid("negative size");
  if (rows > COUNT_LIMIT || seqs > COUNT_LIMIT) return invalid("rows and requests are counted in 32 bits");
  if (heads > 0 && (kv_heads == 0 || heads % kv_heads != 0))
    return invalid("query heads must be a multiple of key heads; got " + std::to_string(heads) + " and " +
                   std::to_string(kv_heads));
  if (dim > ATTN_MAX_DIM)
    return set_error(KF_ERR_UNSUPPORTED, "attention heads of at most " + std::to_string(ATTN_MAX_DIM) +
                                             " elements; got " + std::to_string(dim));
  return KF_OK;
}

// Rows may be computed again from q when others have been written, and every element by one
// thread alone. (Partial overlaps are the caller's to avoid.)
int check_output(const void* q, const void* out, int64_t rows, int64_t so_row, int64_t heads, int64_t so_head) {
  if (out == q) return invalid("out must not be q");
  if ((rows > 1 && so_row == 0) || (heads > 1 && so_head == 0)) return invalid("out overlaps itself: a stride of zero");
  return KF_OK;
}

}  // namespace
}  // namespace kf

using namespace kf;

extern "C" {

int32_t kf_prefill_attention(const kf_prefill_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_prefill_args& g = *args;
  int rc = check_heads(g.dtype, g.rows, g.seqs, g.heads, g.kv_heads, g.dim);
  if (rc != KF_OK) return rc;
  if (g.keys < 0 || g.keys > COUNT_LIMIT) return invalid("keys are counted in 32 bits");
  if (!std::isfinite(g.scale)) return invalid("scale must be finite");
  if (g.rows == 0 || g.heads == 0 || g.dim == 0) return KF_OK;
  if (g.q == nullptr || g.out == nullptr || g.cu_q == nullptr || g.cu_k == nullptr ||
      (g.keys > 0 && (g.k == nullptr || g.v == nullptr)))
    return invalid("null pointer");
  rc = check_output(g.q, g.out, g.rows, g.so_row, g.heads, g.so_head);
  if (rc != KF_OK) return rc;
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  AttnArgs a;
  a.dtype = static_cast<int>(g.dtype);
  a.q = g.q, a.sq_t = g.sq_row, a.sq_h = g.sq_head;
  a.k = g.k, a.sk_t = g.sk_row, a.sk_h = g.sk_head;
  a.v = g.v, a.sv_t = g.sv_row, a.sv_h = g.sv_head;
  a.out = g.out, a.so_t = g.so_row, a.so_h = g.so_head;
  a.lse = g.lse;
  a.cu_q = g.cu_q, a.cu_k = g.cu_k;
  a.seqs = g.seqs, a.rows = g.rows, a.keys = g.keys, a.heads = g.heads, a.kv_heads = g.kv_heads, a.dim = g.dim;
  a.scale_log2 = static_cast<float>(g.scale * LOG2_E);
  a.causal = g.causal != 0;
  if (attention_prefill_supported(a)) return launch_attention_prefill(a, *dev, static_cast<cudaStream_t>(stream));
  return launch_attention_block(a, *dev, static_cast<cudaStream_t>(stream));
}

int32_t kf_tree_attention(const kf_tree_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_tree_args& g = *args;
  int rc = check_heads(g.dtype, g.rows, g.seqs, g.heads, g.kv_heads, g.dim);
  if (rc != KF_OK) return rc;
  if (g.table_cols < 0 || g.pages < 0 || g.mask_words < 0) return invalid("negative size");
  if (g.pages > INT32_LIMIT || g.mask_words > INT32_LIMIT) return invalid("pages and mask words are counted in 32 bits");
  if (g.block_size < 1 || g.block_size > INT32_LIMIT) return invalid("block_size must be positive and fit 32 bits");
  if (!std::isfinite(g.scale)) return invalid("scale must be finite");
  if (g.rows == 0 || g.heads == 0 || g.dim == 0) return KF_OK;
  if (g.q == nullptr || g.out == nullptr || (g.seqs > 0 && g.context == nullptr) ||
      (g.seqs > 0 && g.table_cols > 0 && g.block_table == nullptr) ||
      (g.pages > 0 && (g.k_cache == nullptr || g.v_cache == nullptr)) || (g.mask_words > 0 && g.tree_mask == nullptr))
    return invalid("null pointer");
  if ((reinterpret_cast<uintptr_t>(g.workspace) & 255u) != 0)
    return set_error(KF_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  rc = check_output(g.q, g.out, g.rows, g.so_row, g.heads, g.so_head);
  if (rc != KF_OK) return rc;
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  AttnArgs a;
  a.dtype = static_cast<int>(g.dtype);
  a.q = g.q, a.sq_t = g.sq_row, a.sq_h = g.sq_head;
  a.k = g.k_cache, a.sk_p = g.sk_page, a.sk_h = g.sk_head, a.sk_t = g.sk_slot;
  a.v = g.v_cache, a.sv_p = g.sv_page, a.sv_h = g.sv_head, a.sv_t = g.sv_slot;
  a.out = g.out, a.so_t = g.so_row, a.so_h = g.so_head;
  a.lse = g.lse;
  a.cu_q = g.cu_q;
  a.paged = 1;
  a.table = g.block_table, a.table_stride = g.table_stride, a.table_cols = g.table_cols;
  a.pages = g.pages, a.block_size = g.block_size;
  a.context = g.context;
  a.mask = g.mask_words > 0 ? reinterpret_cast<const unsigned long long*>(g.tree_mask) : nullptr;
  a.mask_words = g.mask_words;
  a.seqs = g.seqs, a.rows = g.rows, a.heads = g.heads, a.kv_heads = g.kv_heads, a.dim = g.dim;
  a.scale_log2 = static_cast<float>(g.scale * LOG2_E);
  a.workspace = g.workspace, a.workspace_bytes = g.workspace_bytes;
  if (attention_tree_supported(a)) return launch_attention_tree(a, *dev, static_cast<cudaStream_t>(stream));
  return launch_attention_block(a, *dev, static_cast<cudaStream_t>(stream));
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

int32_t kf_rotary(const kf_rotary_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_rotary_args& g = *args;
  if (!known_dtype(g.dtype)) return invalid("unknown dtype code");
  if (g.tokens < 0 || g.heads < 0 || g.kv_heads < 0 || g.dim < 0 || g.table_rows < 0 || g.rot < 0 || g.pages < 0)
    return invalid("negative size");
  if (g.rot % 2 != 0 || g.rot > g.dim)
    return invalid("the turned part must be even and at most the head; got " + std::to_string(g.rot) + " of " +
                   std::to_string(g.dim));
  if (g.heads > INT32_LIMIT / 4 || g.kv_heads > INT32_LIMIT / 4 || g.dim > INT32_LIMIT / 4)
    return invalid("heads and their elements are counted in 32 bits");
  if (g.tokens == 0 || g.dim == 0 || g.heads + g.kv_heads == 0) return KF_OK;
  if ((g.heads > 0 && (g.q == nullptr || g.q_out == nullptr)) || (g.kv_heads > 0 && g.k == nullptr) ||
      (g.rot > 0 && (g.positions == nullptr || (g.table_rows > 0 && g.table == nullptr))))
    return invalid("null pointer");
  const bool cached = g.slots != nullptr && g.kv_heads > 0;
  if (g.kv_heads > 0 && g.k_out == nullptr && !cached) return invalid("k needs an output or a cache");
  if (cached && g.block_size < 1) return invalid("block_size must be positive");
  if (cached && (g.v == nullptr || (g.pages > 0 && (g.k_cache == nullptr || g.v_cache == nullptr))))
    return invalid("null pointer");
  RotaryArgs a;
  a.dtype = static_cast<int>(g.dtype);
  a.q = g.q, a.sq_t = g.sq_row, a.sq_h = g.sq_head;
  a.q_out = g.q_out, a.sqo_t = g.sqo_row, a.sqo_h = g.sqo_head;
  a.k = g.k, a.sk_t = g.sk_row, a.sk_h = g.sk_head;
  a.k_out = g.k_out, a.sko_t = g.sko_row, a.sko_h = g.sko_head;
  a.positions = g.positions, a.table = g.table, a.table_rows = g.table_rows, a.rot = g.rot;
  if (cached) {
    a.v = g.v, a.sv_t = g.sv_row, a.sv_h = g.sv_head;
    a.k_cache = g.k_cache, a.skc_p = g.skc_page, a.skc_h = g.skc_head, a.skc_s = g.skc_slot;
    a.v_cache = g.v_cache, a.svc_p = g.svc_page, a.svc_h = g.svc_head, a.svc_s = g.svc_slot;
    a.pages = g.pages, a.block_size = g.block_size;
    a.slots = g.slots;
  }
  a.tokens = g.tokens, a.heads = g.heads, a.kv_heads = g.kv_heads, a.dim = g.dim;
  a.interleaved = g.interleaved != 0, a.inverse = g.inverse != 0;
  DeviceInfo* dev = nullptr;
  const int rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  return launch_rotary(a, *dev, static_cast<cudaStream_t>(stream));
}

int32_t kf_build_slots(const kf_slots_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_slots_args& g = *args;
  if (g.seqs < 0 || g.table_cols < 0 || g.n_free < 0 || g.max_tokens < 0) return invalid("negative size");
  if (g.max_tokens > INT32_LIMIT) return invalid("tokens are counted in 32 bits");
  if (g.block_size < 1) return invalid("block_size must be positive");
  if (g.cu_new == nullptr || g.counts == nullptr || (g.seqs > 0 && (g.context == nullptr || g.added == nullptr)) ||
      (g.seqs > 0 && g.table_cols > 0 && g.block_table == nullptr) || (g.n_free > 0 && g.free_blocks == nullptr) ||
      (g.max_tokens > 0 && (g.positions == nullptr || g.slots == nullptr)))
    return invalid("null pointer");
  DeviceInfo* dev = nullptr;
  const int rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  return launch_slots(g, *dev, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
