// What the attention kernels share: the problem as the C ABI received it, the
// request a row belongs to, and where a request's keys are (packed rows, or
// pages of a cache).
//
// Requests are given by offsets on the device (cu_q, cu_k, context), which the
// host never reads. Every offset is clamped to the arrays it indexes, and every
// page number is checked, so a malformed plan gives wrong rows but no access
// out of bounds.
#pragma once

#include "kf_common.cuh"
#include "kf_internal.h"

namespace kf {

// Rows [begin, end) of request r. Rows past the last offset form one more
// request (r = seqs) that has no keys, so that they are written too.
__device__ __forceinline__ void request_rows(const AttnArgs& p, int r, int* begin, int* end) {
  const int rows = static_cast<int>(p.rows);
  if (p.cu_q == nullptr) {  // one row per request
    *begin = min(r, rows);
    *end = r < p.seqs ? min(r + 1, rows) : rows;
    return;
  }
  const int b = r == 0 ? 0 : min(max(__ldg(p.cu_q + r), 0), rows);
  *begin = b;
  *end = r < p.seqs ? min(max(__ldg(p.cu_q + r + 1), b), rows) : rows;
}

// Keys of request r: the first packed row (0 for a cache) and their number.
__device__ __forceinline__ void request_keys(const AttnArgs& p, int r, int nodes, long long* first, long long* length) {
  *first = 0;
  *length = 0;
  if (r >= p.seqs) return;
  if (p.paged) {
    const long long room = p.table_cols * p.block_size;
    const long long n = static_cast<long long>(max(__ldg(p.context + r), 0)) + nodes;
    // positions are counted in 31 bits
    *length = min(min(n, room), 0x7fffff00ll);
    return;
  }
  const int keys = static_cast<int>(p.keys);
  const int b = r == 0 ? 0 : min(max(__ldg(p.cu_k + r), 0), keys);
  *first = b;
  *length = min(max(__ldg(p.cu_k + r + 1), b), keys) - b;
}

// The request that holds row t: the last one whose first row is at most t
// (empty requests before it share its first row).
__device__ __forceinline__ int request_of(const AttnArgs& p, int t) {
  if (p.cu_q == nullptr) return min(t, static_cast<int>(p.seqs));
  int lo = 0, hi = static_cast<int>(p.seqs);  // first r with cu_q[r + 1] > t, or seqs
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.cu_q + mid + 1) > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}

// Element offset of key `pos` of request r for one head, or -1 where the block
// table names no page.
__device__ __forceinline__ long long key_offset(const AttnArgs& p, int r, long long first, long long pos,
                                                long long s_page, long long s_row) {
  if (!p.paged) return (first + pos) * s_row;
  const uint32_t at = static_cast<uint32_t>(pos), block = static_cast<uint32_t>(p.block_size), col = at / block;
  const int page = __ldg(p.table + r * p.table_stride + col);
  if (page < 0 || page >= p.pages) return -1;
  return page * s_page + (at - col * block) * s_row;
}

// A wait of a kernel whose rows may be computed again beside it (redo_begin).
__device__ __forceinline__ bool attn_wait(uint32_t bar, uint32_t parity, volatile int* flag, int* status, int site) {
  return mbar_wait<true>(bar, parity, flag, status, site);
}
// Around rows that a warp computes again, whose time goes by their keys: the other
// warps' waits do not run out meanwhile. `flag` is the CTA's abort flag.
__device__ __forceinline__ void redo_begin(volatile int* flag, int lane) {
  if (lane == 0) atomicAdd(const_cast<int*>(flag), 2);
  __syncwarp();
}
__device__ __forceinline__ void redo_end(volatile int* flag, int lane) {
  __syncwarp();
  if (lane == 0) atomicAdd(const_cast<int*>(flag), -2);
}

// What row t of the problem sees of its request's keys: all below `prefix`, then those
// that `mask` names (from `prefix` on; null: none), up to `last`.
struct RowKeys {
  int request;
  long long first, prefix, last, length;
  const unsigned long long* mask;

  __device__ __forceinline__ RowKeys(const AttnArgs& p, int t) {
    request = request_of(p, t);
    int row0, row1;
    request_rows(p, request, &row0, &row1);
    request_keys(p, request, row1 - row0, &first, &length);
    const int node = t - row0;
    mask = nullptr;
    if (!p.paged) {
      prefix = last = p.causal ? min(length, max(0ll, node + 1 + length - (row1 - row0))) : length;
      return;
    }
    prefix = min(length, static_cast<long long>(request < p.seqs ? max(__ldg(p.context + request), 0) : 0));
    last = length;
    if (p.mask == nullptr) prefix = last = min(length, prefix + node + 1);
    else mask = p.mask + t * p.mask_words;
  }
  __device__ __forceinline__ bool sees(const AttnArgs& p, long long pos) const {
    if (pos < prefix || mask == nullptr) return pos < prefix;
    const long long j = pos - prefix;
    return j < 64ll * p.mask_words && ((__ldg(mask + (j >> 6)) >> (j & 63)) & 1ull);
  }
};

constexpr int AT_ONCE = 8;  // keys whose loads a warp has in flight

// Elements lane + 32 i of AT_ONCE keys, zeros where `take` has no bit and past the head.
// Lane x < AT_ONCE has key x's offset.
template <typename T, int NE>
__device__ __forceinline__ void load_keys(const T* base, long long offset, uint32_t take, int dim, int lane,
                                          T (&raw)[AT_ONCE][NE]) {
#pragma unroll
  for (int x = 0; x < AT_ONCE; ++x) {
    const T* const at = base + __shfl_sync(0xffffffffu, offset, x) + lane;
#pragma unroll
    for (int i = 0; i < NE; ++i) raw[x][i] = ((take >> x) & 1u) && lane + 32 * i < dim ? at[32 * i] : from_f32<T>(0.0f);
  }
}

// The last of the keys [from, to) that row t does not see and whose value holds
// something not finite, -1 if none does. By one warp.
template <typename T, int NE>
__device__ __forceinline__ long long last_unseen_nonfinite(const AttnArgs& p, int t, int head, long long from, long long to,
                                                        int lane) {
  const RowKeys row(p, t);
  const int kv_head = head / static_cast<int>(p.heads / p.kv_heads), D = static_cast<int>(p.dim);
  const T* v = static_cast<const T*>(p.v) + kv_head * p.sv_h;
  to = min(to, row.length);
  for (long long end = to; end > from; end -= AT_ONCE) {
    const long long pos = end - AT_ONCE + lane;
    const long long vo = lane < AT_ONCE && pos >= from && !row.sees(p, pos)
                             ? key_offset(p, row.request, row.first, pos, p.sv_p, p.sv_t) : -1;
    const uint32_t take = __ballot_sync(0xffffffffu, vo >= 0);
    if (take == 0) continue;
    T raw[AT_ONCE][NE];
    load_keys<T, NE>(v, vo, take, D, lane, raw);
    uint32_t bad = 0;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (!(fabsf(to_f32(raw[x][i])) < INFINITY)) bad |= 1u << x;
    }
    bad = __reduce_or_sync(0xffffffffu, bad);
    if (bad != 0) return end - AT_ONCE + 31 - __clz(bad);
  }
  return -1;
}

// One row of attention by one warp, AT_ONCE keys at a time: for lane's elements
// e = lane + 32 i of the head, acc = sum_j p_j v_j with the running maximum m
// and sum l of the softmax in base 2 (q is read times scale * log2(e)). Keys that
// the row does not see are not read, so nothing in them reaches the result. About
// 0.4 us a key of 128 elements (one key at a time, and looked up in 64 bits, 2).
template <typename T, int NE>
__device__ __forceinline__ void attend_row(const AttnArgs& p, int t, int head, int lane, float (&acc)[NE], float* m_out,
                                           float* l_out) {
  const RowKeys row(p, t);
  const int kv_head = head / static_cast<int>(p.heads / p.kv_heads), D = static_cast<int>(p.dim);
  const T* q = static_cast<const T*>(p.q) + t * p.sq_t + head * p.sq_h;
  const T* k = static_cast<const T*>(p.k) + kv_head * p.sk_h;
  const T* v = static_cast<const T*>(p.v) + kv_head * p.sv_h;
  float qf[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = lane + 32 * i;
    qf[i] = e < D ? to_f32(q[e]) * p.scale_log2 : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  const int own = ((lane >> 4) & 1) * 4 + ((lane >> 3) & 1) * 2 + ((lane >> 2) & 1);  // the key whose score this lane gets
  for (long long pos0 = 0; pos0 < row.last; pos0 += AT_ONCE) {
    long long ko = -1, vo = 0;  // of key pos0 + lane
    const long long pos = pos0 + lane;
    if (lane < AT_ONCE && pos < row.last && row.sees(p, pos)) {
      ko = key_offset(p, row.request, row.first, pos, p.sk_p, p.sk_t);
      if (ko >= 0) vo = key_offset(p, row.request, row.first, pos, p.sv_p, p.sv_t);
    }
    const uint32_t seen = __ballot_sync(0xffffffffu, ko >= 0);
    if (seen == 0) continue;
    T raw[AT_ONCE][NE];
    load_keys<T, NE>(k, ko, seen, D, lane, raw);
    float s[AT_ONCE];
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      s[x] = 0.0f;
#pragma unroll
      for (int i = 0; i < NE; ++i) s[x] = fmaf(lane + 32 * i < D ? qf[i] : 0.0f, to_f32(raw[x][i]), s[x]);
    }
    // the lanes' shares of eight scores: halves are exchanged until a lane has one, four lanes the same
#pragma unroll
    for (int half = AT_ONCE / 2, o = 16; half > 0; half /= 2, o /= 2) {
#pragma unroll
      for (int x = 0; x < half; ++x) {
        const bool upper = lane & o;
        const float give = upper ? s[x] : s[x + half], keep = upper ? s[x + half] : s[x];
        s[x] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    }
    s[0] += __shfl_xor_sync(0xffffffffu, s[0], 2);
    s[0] += __shfl_xor_sync(0xffffffffu, s[0], 1);
    // weight zero at -infinity, also while m is still that
    const bool weighs = ((seen >> own) & 1u) && s[0] != -INFINITY;
    const uint32_t any = __ballot_sync(0xffffffffu, weighs);
    if (any == 0) continue;
    __syncwarp();  // the values are loaded behind the scores: with both in registers the callers spill
    load_keys<T, NE>(v, vo, seen, D, lane, raw);
    float m_new = weighs ? fmaxf(m, s[0]) : m;
#pragma unroll
    for (int o = 16; o > 2; o /= 2) m_new = fmaxf(m_new, __shfl_xor_sync(0xffffffffu, m_new, o));
    const float fix = ex2_ftz(m - m_new), w = weighs ? ex2_ftz(s[0] - m_new) : 0.0f;
    m = m_new;
    l = fmaf(l, fix, w);  // of this lane's key in each step
#pragma unroll
    for (int i = 0; i < NE; ++i) acc[i] *= fix;
#pragma unroll
    for (int x = 0; x < AT_ONCE; ++x) {
      const int from = (x & 4) * 4 + (x & 2) * 4 + (x & 1) * 4;
      const float weight = __shfl_sync(0xffffffffu, w, from);
#pragma unroll
      for (int i = 0; i < NE; ++i) acc[i] = (any >> from) & 1u ? fmaf(weight, to_f32(raw[x][i]), acc[i]) : acc[i];
    }
  }
#pragma unroll
  for (int o = 16; o > 2; o /= 2) l += __shfl_xor_sync(0xffffffffu, l, o);
  *m_out = m;
  *l_out = l;
}

// Whether a finished row may have to be computed again: something in it is not finite
// (`fine` false). A sum that is NaN comes from a score that the row sees, and stays.
// Otherwise a key that the row does not see may have done it (0 x infinity), which
// last_unseen_nonfinite tells; what else is not finite comes from what it sees.
__device__ __forceinline__ bool suspect(bool fine, float l) { return !fine && l == l; }

// Writes a row that attend_row left in `acc`: acc / l, zero where no key was seen.
template <typename T, int NE>
__device__ __forceinline__ void write_row(const AttnArgs& p, int t, int head, int lane, const float (&acc)[NE], float m,
                                          float l) {
  T* out = static_cast<T*>(p.out) + t * p.so_t + head * p.so_h;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int e = lane + 32 * i;
    if (e < p.dim) out[e] = from_f32<T>(l == 0.0f ? 0.0f : acc[i] / l);
  }
  if (p.lse != nullptr && lane == 0)
    p.lse[t * p.heads + head] = l == 0.0f ? -INFINITY : m * 0.69314718055994530942f + logf(l);
}

}  // namespace kf
