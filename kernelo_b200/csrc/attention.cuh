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
  const long long col = pos / p.block_size;
  const int page = __ldg(p.table + r * p.table_stride + col);
  if (page < 0 || page >= p.pages) return -1;
  return page * s_page + (pos - col * p.block_size) * s_row;
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

// One row of attention by one warp, key by key: for lane's elements
// e = lane + 32 i of the head, acc = sum_j p_j v_j with the running maximum m
// and sum l of the softmax in base 2 (q is read times scale * log2(e)). Keys that
// the row does not see are not read, so nothing in them reaches the result.
template <typename T, int NE>
__device__ __forceinline__ void attend_row(const AttnArgs& p, int t, int head, int lane, float (&acc)[NE], float* m_out,
                                           float* l_out) {
  const int r = request_of(p, t);
  int row0, row1;
  request_rows(p, r, &row0, &row1);
  long long first, length;
  request_keys(p, r, row1 - row0, &first, &length);
  const int kv_head = head / static_cast<int>(p.heads / p.kv_heads);
  const int D = static_cast<int>(p.dim);
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
  // all keys below `prefix`, then those the mask names
  const int node = t - row0;
  long long prefix, last = length;
  if (p.paged) {
    prefix = min(length, static_cast<long long>(r < p.seqs ? max(__ldg(p.context + r), 0) : 0));
    if (p.mask == nullptr) prefix = last = min(length, prefix + node + 1);
  } else {
    prefix = p.causal ? min(length, max(0ll, node + 1 + length - (row1 - row0))) : length;
    last = prefix;
  }
  const unsigned long long* mask = p.mask != nullptr ? p.mask + t * p.mask_words : nullptr;
  for (long long pos = 0; pos < last; ++pos) {
    if (pos >= prefix) {
      const long long j = pos - prefix;
      if (j >= 64ll * p.mask_words || !((__ldg(mask + (j >> 6)) >> (j & 63)) & 1ull)) continue;
    }
    const long long ko = key_offset(p, r, first, pos, p.sk_p, p.sk_t);
    if (ko < 0) continue;
    const long long vo = key_offset(p, r, first, pos, p.sv_p, p.sv_t);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = lane + 32 * i;
      if (e < D) s = fmaf(qf[i], to_f32(k[ko + e]), s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (s == -INFINITY) continue;  // weight zero, also while m is still -inf
    const float m_new = fmaxf(m, s);
    const float fix = ex2_ftz(m - m_new), w = ex2_ftz(s - m_new);
    m = m_new;
    l = fmaf(l, fix, w);
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int e = lane + 32 * i;
      acc[i] = fmaf(acc[i], fix, e < D ? w * to_f32(v[vo + e]) : 0.0f);
    }
  }
  *m_out = m;
  *l_out = l;
}

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
