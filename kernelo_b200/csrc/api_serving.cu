// extern "C" entry points of the serving operators: prompt attention, tree
// attention over a paged cache, rotary positions with the cache write, and
// block tables with slot maps. Argument checks here, kernels in their own files.
#include <cmath>
#include <limits>
#include <string>

#include "kf_common.cuh"
#include "kf_internal.h"
#include "overlap.h"

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
// Tokens of a vocabulary: a chunk beyond the last one, too. (Occurrences in a history are counted in 30 bits.)
constexpr int64_t LOGITS_LIMIT = 0x7fff0000ll;
constexpr int64_t LOGITS_BIASES = 16384;  // 32 of each thread of a block

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

// *nothing: no element to turn (the other fields are then not set).
int rotary_args(const kf_rotary_args& g, RotaryArgs* to, bool* nothing) {
  if (!known_dtype(g.dtype)) return invalid("unknown dtype code");
  if (g.tokens < 0 || g.heads < 0 || g.kv_heads < 0 || g.dim < 0 || g.table_rows < 0 || g.rot < 0 || g.pages < 0)
    return invalid("negative size");
  if (g.rot % 2 != 0 || g.rot > g.dim)
    return invalid("the turned part must be even and at most the head; got " + std::to_string(g.rot) + " of " +
                   std::to_string(g.dim));
  if (g.heads > INT32_LIMIT / 4 || g.kv_heads > INT32_LIMIT / 4 || g.dim > INT32_LIMIT / 4)
    return invalid("heads and their elements are counted in 32 bits");
  *nothing = g.tokens == 0 || g.dim == 0 || g.heads + g.kv_heads == 0;
  if (*nothing) return KF_OK;
  if ((g.heads > 0 && (g.q == nullptr || g.q_out == nullptr)) || (g.kv_heads > 0 && g.k == nullptr) ||
      (g.rot > 0 && (g.positions == nullptr || (g.table_rows > 0 && g.table == nullptr))))
    return invalid("null pointer");
  const bool cached = g.slots != nullptr && g.kv_heads > 0;
  if (g.kv_heads > 0 && g.k_out == nullptr && !cached) return invalid("k needs an output or a cache");
  if (cached && g.block_size < 1) return invalid("block_size must be positive");
  if (cached && (g.v == nullptr || (g.pages > 0 && (g.k_cache == nullptr || g.v_cache == nullptr))))
    return invalid("null pointer");
  RotaryArgs& a = *to;
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
  return KF_OK;
}

int shared(const Region& out, const Region& other) {
  return invalid(std::string(out.name) + " shares memory with " + other.name);
}
int self_shared(const Region& out) { return invalid(std::string(out.name) + " overlaps itself"); }

// Outputs are written while other heads' operands are still read: each has its own memory, or (q_out, k_out) its input's.
int check_norm_memory(const RotaryArgs& a, const NormArgs& n) {
  const int elem = a.dtype == KF_FP32 ? 4 : 2;
  const auto heads = [&](const char* name, const void* at, int64_t h, int64_t s_t, int64_t s_h) {
    return Region(name, h > 0 ? at : nullptr, elem, {{a.tokens, s_t}, {h, s_h}, {a.dim, 1}});
  };
  const auto cache = [&](const char* name, const void* at, int64_t s_p, int64_t s_h, int64_t s_s) {
    return Region(name, a.slots != nullptr ? at : nullptr, elem,
                  {{a.pages, s_p}, {a.kv_heads, s_h}, {a.block_size, s_s}, {a.dim, 1}});
  };
  const Region in[] = {heads("q", a.q, a.heads, a.sq_t, a.sq_h),
                       heads("k", a.k, a.kv_heads, a.sk_t, a.sk_h),
                       heads("v", a.v, a.kv_heads, a.sv_t, a.sv_h),
                       Region("q_weight", a.heads > 0 ? n.q_weight : nullptr, elem, {{a.dim, 1}}),
                       Region("k_weight", a.kv_heads > 0 ? n.k_weight : nullptr, elem, {{a.dim, 1}}),
                       Region("positions", a.rot > 0 ? a.positions : nullptr, 4, {{a.tokens, 1}}),
                       Region("table", a.table, 4, {{a.table_rows, a.rot}, {a.rot, 1}}),
                       Region("slots", a.slots, 8, {{a.tokens, 1}})};
  const Region out[] = {heads("q_out", a.q_out, a.heads, a.sqo_t, a.sqo_h),
                        heads("k_out", a.k_out, a.kv_heads, a.sko_t, a.sko_h),
                        cache("k_cache", a.k_cache, a.skc_p, a.skc_h, a.skc_s),
                        cache("v_cache", a.v_cache, a.svc_p, a.svc_h, a.svc_s)};
  for (int i = 0; i < 4; ++i) {
    if (out[i].overlaps_itself()) return self_shared(out[i]);
    for (int j = 0; j < 8; ++j)
      if (overlap(out[i], in[j]) && !(i < 2 && i == j && out[i].same_place(in[j]))) return shared(out[i], in[j]);
    for (int j = 0; j < i; ++j)
      if (overlap(out[i], out[j])) return shared(out[i], out[j]);
  }
  return KF_OK;
}

// A row's chunks read the row's lists while others write theirs.
int check_logits_memory(const kf_logits_args& g) {
  const int elem = g.dtype == KF_FP32 ? 4 : 2;
  const Region out("out", g.out, elem, {{g.rows, g.so_row}, {g.vocab, 1}});
  const Region logits("logits", g.logits, elem, {{g.rows, g.s_row}, {g.vocab, 1}});
  if (out.overlaps_itself()) return self_shared(out);
  if (overlap(out, logits) && !out.same_place(logits)) return shared(out, logits);
  const void* const tokens = g.tokens;  // without them nothing of a history is read
  const auto each = [&](const char* name, const void* at) { return Region(name, tokens != nullptr ? at : nullptr, 4, {{g.rows, 1}}); };
  const void* const biases = g.bias_tokens;
  const Region in[] = {Region("tokens", tokens, 4, {{g.rows, g.st_row}, {g.token_cols, 1}}),
                       each("token_lens", g.token_lens), each("prompt_lens", g.prompt_lens), each("repetition", g.repetition),
                       each("frequency", g.frequency), each("presence", g.presence),
                       Region("bias_tokens", biases, 4, {{g.rows, g.sb_row}, {g.bias_cols, 1}}),
                       Region("bias_values", biases != nullptr ? g.bias_values : nullptr, 4, {{g.rows, g.sv_row}, {g.bias_cols, 1}}),
                       Region("allowed", g.allowed, 4, {{g.masks, g.sa_row}, {ceil_div(g.vocab, 32), 1}}),
                       Region("allowed_rows", g.allowed != nullptr ? g.allowed_rows : nullptr, 4, {{g.rows, 1}})};
  for (const Region& other : in)
    if (overlap(out, other)) return shared(out, other);
  return KF_OK;
}

// Rows that one call's bits take 96 KB of shared memory for; and pages that a cluster's do 1 MB for.
constexpr int64_t TABLE_ROWS_LIMIT = 1 << 18;
constexpr int64_t COMPACT_PAGES_LIMIT = 1 << 22;

int check_table(int64_t rows, int64_t cols, const void* table, const void* context, int64_t pages, const void* holders) {
  if (rows < 0 || cols < 0) return invalid("negative size");
  if (rows > TABLE_ROWS_LIMIT) return invalid("block tables of at most " + std::to_string(TABLE_ROWS_LIMIT) + " rows");
  if (cols > COUNT_LIMIT || rows * cols > (1ll << 40)) return invalid("columns are counted in 32 bits");
  if ((rows > 0 && cols > 0 && table == nullptr) || (rows > 0 && context == nullptr) || (pages > 0 && holders == nullptr))
    return invalid("null pointer");
  return KF_OK;
}

int page_geometry(const kf_page_caches& c, PageGeometry* to) {
  if (!known_dtype(c.dtype)) return invalid("unknown dtype code");
  if (c.n_caches < 0 || c.pages < 0 || c.heads < 0 || c.dim < 0) return invalid("negative size");
  if (c.pages > COUNT_LIMIT) return invalid("pages are counted in 32 bits");
  if (c.block_size < 1) return invalid("block_size must be positive");
  if (c.block_size > INT32_LIMIT || c.heads > INT32_LIMIT || c.dim > INT32_LIMIT ||
      (c.heads > 0 && c.dim > 0 && c.block_size > INT32_LIMIT / 2 / c.heads / c.dim))
    return invalid("a page's elements are counted in 32 bits");
  if (c.n_caches > 0 && c.caches == nullptr) return invalid("null pointer");
  for (int64_t i = 0; i < c.n_caches; ++i)
    if (c.caches[i] == nullptr && c.pages * c.heads * c.dim > 0) return invalid("null pointer");
  to->elem = c.dtype == KF_FP32 ? 4 : 2;
  if (c.n_caches > 0 && Region("a cache", c.caches[0], to->elem, {{c.pages, c.s_page}, {c.heads, c.s_head},
                               {c.block_size, c.s_slot}, {c.dim, 1}}).overlaps_itself())
    return invalid("caches overlap themselves");
  to->s_page = c.s_page, to->s_head = c.s_head, to->s_slot = c.s_slot;
  to->pages = c.pages, to->heads = c.heads, to->block = c.block_size, to->dim = c.dim;
  return KF_OK;
}

PageCaches page_caches(const kf_page_caches& c, int64_t first) {
  PageCaches to{};
  const int64_t left = c.heads > 0 && c.dim > 0 ? c.n_caches - first : 0;  // empty pages have nothing to copy
  to.count = static_cast<int>(left < PAGE_CACHES ? left : PAGE_CACHES);
  for (int i = 0; i < to.count; ++i) to.at[i] = c.caches[first + i];
  return to;
}

int norm_args(int64_t dim, double eps, NormArgs* to) {
  if (dim > NORM_ROTARY_MAX_DIM)
    return set_error(KF_ERR_UNSUPPORTED, "norms of heads of at most " + std::to_string(NORM_ROTARY_MAX_DIM) +
                                             " elements; got " + std::to_string(dim));
  // Below the normal range squares as small as eps would lose their bits, and one rounded to zero makes NaN of zeros.
  if (!(eps >= std::numeric_limits<float>::min() && eps <= std::numeric_limits<float>::max()))
    return invalid("eps must be positive and in fp32's normal range");
  to->eps = static_cast<float>(eps);
  to->inv_dim = dim > 0 ? 1.0f / static_cast<float>(dim) : 0.0f;
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
  RotaryArgs a;
  bool nothing = false;
  int rc = rotary_args(*args, &a, &nothing);
  if (rc != KF_OK || nothing) return rc;
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  return launch_rotary(a, *dev, static_cast<cudaStream_t>(stream));
}

int32_t kf_norm_rotary(const kf_norm_rotary_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_norm_rotary_args& g = *args;
  RotaryArgs a;
  NormArgs n;
  bool nothing = false;
  int rc = norm_args(g.rotary.dim, g.eps, &n);
  if (rc == KF_OK) rc = rotary_args(g.rotary, &a, &nothing);
  if (rc != KF_OK) return rc;
  if (g.rotary.inverse != 0) return invalid("inverse: the gradient of norms and turn is kf_norm_rotary_grad");
  if (nothing) return KF_OK;
  if ((a.heads > 0 && g.q_weight == nullptr) || (a.kv_heads > 0 && g.k_weight == nullptr)) return invalid("null pointer");
  // Lanes of a warp beside its last head read a weight too, which may be of the kind that has no heads.
  n.q_weight = a.heads > 0 ? g.q_weight : g.k_weight;
  n.k_weight = a.kv_heads > 0 ? g.k_weight : g.q_weight;
  rc = check_norm_memory(a, n);
  if (rc != KF_OK) return rc;
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  return launch_norm_rotary(a, n, *dev, static_cast<cudaStream_t>(stream));
}

int32_t kf_norm_rotary_grad(const kf_norm_rotary_grad_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_norm_rotary_grad_args& g = *args;
  NormGradArgs a;
  bool nothing = false;
  int rc = norm_args(g.rotary.dim, g.eps, &a.norm);
  if (rc == KF_OK) rc = rotary_args(g.rotary, &a.rotary, &nothing);
  if (rc != KF_OK) return rc;
  if (g.rotary.inverse != 0) return invalid("inverse: the gradient is of the forward turn");
  if (g.rotary.slots != nullptr) return invalid("the gradient has no cache");
  if (g.rotary.dim == 0) return KF_OK;
  if (g.q_weight_grad == nullptr || g.k_weight_grad == nullptr) return invalid("null pointer");
  if (!nothing && ((g.rotary.heads > 0 && (g.dq == nullptr || g.q_weight == nullptr)) ||
                   (g.rotary.kv_heads > 0 && (g.dk == nullptr || g.k_weight == nullptr))))
    return invalid("null pointer");
  if (nothing) a.rotary.tokens = 0, a.rotary.dim = g.rotary.dim;
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  const RotaryArgs& r = a.rotary;
  if (g.workspace_bytes < norm_rotary_grad_workspace_bytes(r.tokens, r.heads, r.kv_heads, r.dim, *dev) ||
      (g.workspace == nullptr && g.workspace_bytes > 0))
    return set_error(KF_ERR_WORKSPACE, "workspace too small for the weights' partial sums");
  if ((reinterpret_cast<uintptr_t>(g.workspace) & 3u) != 0)
    return set_error(KF_ERR_WORKSPACE, "workspace must be 4-byte aligned");
  a.norm.q_weight = g.q_weight, a.norm.k_weight = g.k_weight;
  a.dq = g.dq, a.sdq_t = g.sdq_row, a.sdq_h = g.sdq_head;
  a.dk = g.dk, a.sdk_t = g.sdk_row, a.sdk_h = g.sdk_head;
  a.q_weight_grad = g.q_weight_grad, a.k_weight_grad = g.k_weight_grad;
  a.partial = static_cast<float*>(g.workspace);
  return launch_norm_rotary_grad(a, *dev, static_cast<cudaStream_t>(stream));
}

int64_t kf_norm_rotary_grad_workspace_bytes(int32_t device, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dim) {
  if (tokens < 0 || heads < 0 || kv_heads < 0 || dim < 0) return -invalid("negative size");
  if (heads > INT32_LIMIT / 4 || kv_heads > INT32_LIMIT / 4) return -invalid("heads are counted in 32 bits");
  DeviceInfo* dev = nullptr;
  const int rc = device_info(device, &dev);
  if (rc != KF_OK) return -rc;
  return norm_rotary_grad_workspace_bytes(tokens, heads, kv_heads, dim, *dev);
}

int32_t kf_fork(const kf_fork_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_fork_args& g = *args;
  PageGeometry geometry;
  int rc = page_geometry(g.caches, &geometry);
  if (rc == KF_OK) rc = check_table(g.rows, g.table_cols, g.block_table, g.context, g.caches.pages, g.holders);
  if (rc != KF_OK) return rc;
  if (g.pairs < 0 || g.n_free < 0) return invalid("negative size");
  if (g.pairs > TABLE_ROWS_LIMIT || g.n_free > COUNT_LIMIT) return invalid("too many pairs or free pages");
  if (g.counts == nullptr || (g.pairs > 0 && (g.parents == nullptr || g.children == nullptr)) ||
      (g.n_free > 0 && g.free_blocks == nullptr))
    return invalid("null pointer");
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (g.pairs == 0) {
    const cudaError_t err = cudaMemsetAsync(g.counts, 0, 2 * sizeof(int32_t), s);
    return err == cudaSuccess ? KF_OK : cuda_error(err, "memset(fork)");
  }
  kf_fork_args f = g;
  for (int64_t first = 0; first == 0 || first < g.caches.n_caches; first += PAGE_CACHES) {
    rc = launch_fork(page_caches(g.caches, first), geometry, f, *dev, s);
    if (rc != KF_OK) return rc;
    f.counts = nullptr;  // the books are kept; the other caches' pages are copied
  }
  return KF_OK;
}

int32_t kf_release(const kf_release_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_release_args& g = *args;
  if (g.pages < 0 || g.count < 0) return invalid("negative size");
  if (g.pages > COUNT_LIMIT) return invalid("pages are counted in 32 bits");
  int rc = check_table(g.rows, g.table_cols, g.block_table, g.context, g.pages, g.holders);
  if (rc != KF_OK) return rc;
  if (g.block_size < 1) return invalid("block_size must be positive");
  if (g.count > TABLE_ROWS_LIMIT || g.count * g.table_cols >= (1 << 30))
    return invalid("requests x columns of one call must be below 2^30");
  if (g.n_freed == nullptr || (g.count > 0 && (g.requests == nullptr || (g.table_cols > 0 && g.scratch == nullptr))) ||
      (g.count * g.table_cols > 0 && g.freed == nullptr))
    return invalid("null pointer");
  if ((reinterpret_cast<uintptr_t>(g.scratch) & 15u) != 0) return set_error(KF_ERR_WORKSPACE, "scratch must be 16-byte aligned");
  if (g.count * ceil_div(g.table_cols, 256) > 200000)
    return set_error(KF_ERR_UNSUPPORTED, "requests x columns / 256 of one call: at most 200000");
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  return launch_release(g, *dev, static_cast<cudaStream_t>(stream));
}

int32_t kf_compact(const kf_compact_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_compact_args& g = *args;
  PageGeometry geometry;
  int rc = page_geometry(g.caches, &geometry);
  if (rc == KF_OK) rc = check_table(g.rows, g.table_cols, g.block_table, g.context, g.caches.pages, g.holders);
  if (rc != KF_OK) return rc;
  if (g.caches.pages > COMPACT_PAGES_LIMIT)
    return set_error(KF_ERR_UNSUPPORTED, "compact takes at most " + std::to_string(COMPACT_PAGES_LIMIT) + " pages; got " +
                                             std::to_string(g.caches.pages));
  if (g.counts == nullptr || (g.caches.pages > 0 && g.renamed == nullptr) ||
      (g.caches.pages > 1 && (g.sources == nullptr || g.targets == nullptr)))
    return invalid("null pointer");
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = launch_compact_plan(g, geometry, *dev, s);
  for (int64_t first = 0; rc == KF_OK && first < g.caches.n_caches; first += PAGE_CACHES)
    rc = launch_move_pages(page_caches(g.caches, first), geometry, g, *dev, s);
  return rc;
}

int32_t kf_adjust_logits(const kf_logits_args* args, void* stream) {
  if (args == nullptr) return invalid("null arguments");
  const kf_logits_args& g = *args;
  if (!known_dtype(g.dtype)) return invalid("unknown dtype code");
  if (g.rows < 0 || g.vocab < 0 || g.token_cols < 0 || g.bias_cols < 0 || g.masks < 0) return invalid("negative size");
  if (g.rows > COUNT_LIMIT || g.vocab > LOGITS_LIMIT || g.token_cols >= (1 << 30))
    return invalid("rows, tokens and biases are counted in 32 bits");
  if (g.bias_cols > LOGITS_BIASES)
    return set_error(KF_ERR_UNSUPPORTED, "at most " + std::to_string(LOGITS_BIASES) + " biases a row; got " +
                                             std::to_string(g.bias_cols));
  if (g.rows == 0 || g.vocab == 0) return KF_OK;
  if (g.logits == nullptr || g.out == nullptr || (g.tokens != nullptr && g.token_lens == nullptr) ||
      (g.bias_tokens != nullptr && g.bias_values == nullptr))
    return invalid("null pointer");
  int rc = check_logits_memory(g);
  if (rc != KF_OK) return rc;
  DeviceInfo* dev = nullptr;
  rc = this_device(&dev);
  if (rc != KF_OK) return rc;
  return launch_logits(g, *dev, static_cast<cudaStream_t>(stream));
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
