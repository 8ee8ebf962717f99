// Block tables and slot maps of one serving step, from request lengths.
//
// Request r holds context[r] cached tokens in the first ceil(context / block)
// pages of its table row and adds added[r] tokens. With the exclusive sums
//
//   cu[r] = sum of added before r,   base[r] = sum of pages needed before r,
//
// its page `col` is table[r][col] where it is held already and
// free[base[r] + col - held] where it is new; token cu[r] + i has position
// context[r] + i and slot page(position / block) * block + position % block. A
// page beyond the free list or the table's row is -1 and its tokens' slots too:
// they count as dropped, as do tokens past the outputs' end. Outputs past the
// last token have position 0 and slot -1, so a captured step of a fixed size
// writes nothing for them.
//
// Each CTA sums all requests itself, a chunk of one per thread at a time, and
// writes its own slice of the tokens and of the new pages: one launch, no CTA
// reads what another writes, no atomics. The call is bound by its launch and the
// latency of the sums: 4.7 us for 64 requests of one token, 8.7 for 512 prompts.
#include <cuda.h>

#include "kf_common.cuh"
#include "kf_internal.h"

namespace kf {
namespace {

constexpr int SLOTS_THREADS = 512;
constexpr int SLOTS_WARPS = SLOTS_THREADS / 32;

struct Sums {
  long long tokens, pages;
};

// Exclusive sums over the block's threads; *total gets the block's sums.
__device__ __forceinline__ Sums block_exclusive(Sums v, Sums* total, Sums* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Sums in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, in.tokens, o), b = __shfl_up_sync(0xffffffffu, in.pages, o);
    if (lane >= o) {
      in.tokens += a;
      in.pages += b;
    }
  }
  if (lane == 31) scratch[warp] = in;
  __syncthreads();
  Sums before{0, 0};
  total->tokens = total->pages = 0;
#pragma unroll
  for (int w = 0; w < SLOTS_WARPS; ++w) {
    const Sums s = scratch[w];
    if (w < warp) {
      before.tokens += s.tokens;
      before.pages += s.pages;
    }
    total->tokens += s.tokens;
    total->pages += s.pages;
  }
  before.tokens += in.tokens - v.tokens;
  before.pages += in.pages - v.pages;
  return before;
}

__global__ void __launch_bounds__(SLOTS_THREADS) slots_kernel(const kf_slots_args p) {
  __shared__ Sums scratch[SLOTS_WARPS];
  __shared__ long long first_token[SLOTS_THREADS + 1];  // of the chunk's requests
  __shared__ long long first_page[SLOTS_THREADS + 1];   // index into the free list
  __shared__ int cached[SLOTS_THREADS];
  __shared__ unsigned long long lost;
  const int tid = threadIdx.x;
  const long long block = p.block_size;
  const long long share = (p.max_tokens + gridDim.x - 1) / gridDim.x;
  const long long lo = min(share * blockIdx.x, static_cast<long long>(p.max_tokens));
  const long long hi = min(lo + share, static_cast<long long>(p.max_tokens));
  const bool teller = blockIdx.x == 0;  // writes the offsets and the counts
  if (tid == 0) lost = 0;
  Sums carry{0, 0};
  for (long long r0 = 0; r0 < p.seqs; r0 += SLOTS_THREADS) {
    const long long r = r0 + tid;
    const int in_chunk = static_cast<int>(min(static_cast<long long>(SLOTS_THREADS), p.seqs - r0));
    long long have = 0, add = 0;
    if (r < p.seqs) {
      have = max(__ldg(p.context + r), 0);
      add = max(__ldg(p.added + r), 0);
    }
    const long long held = (have + block - 1) / block, after = (have + add + block - 1) / block;
    Sums total;
    __syncthreads();  // the previous chunk's arrays are done with
    const Sums before = block_exclusive({add, after - held}, &total, scratch);
    const long long my_token = carry.tokens + before.tokens, my_page = carry.pages + before.pages;
    if (tid < in_chunk) {
      first_token[tid] = my_token;
      first_page[tid] = my_page;
      cached[tid] = static_cast<int>(have);
    }
    if (tid == 0) {
      first_token[in_chunk] = carry.tokens + total.tokens;
      first_page[in_chunk] = carry.pages + total.pages;
    }
    __syncthreads();
    if (teller && r < p.seqs) {
      p.cu_new[r + 1] = static_cast<int>(my_token + add);
      // tokens that get a slot: those in the last held page, then those in new
      // pages up to the end of the free list and of the row
      const long long room = p.max_tokens - my_token;  // outputs left for this request
      const long long stop = have + min(add, max(room, 0ll));
      long long good = 0;
      if (have < held * block && held <= p.table_cols && p.block_table[r * p.table_stride + held - 1] >= 0)
        good += min(stop, held * block) - min(stop, have);
      const long long cols = min(min(after, static_cast<long long>(p.table_cols)),
                                 held + max(p.n_free - my_page, 0ll));
      good += max(min(stop, cols * block) - held * block, 0ll);
      if (good != add) atomicAdd(&lost, static_cast<unsigned long long>(add - good));
    }
    // this CTA's slice of the tokens, as far as they are this chunk's
    const long long t1 = min(hi, first_token[in_chunk]);
    for (long long t = max(lo, carry.tokens) + tid; t < t1; t += SLOTS_THREADS) {
      int a = 0, b = in_chunk - 1;  // the last request of the chunk that starts at or before t
      while (a < b) {
        const int mid = (a + b + 1) >> 1;
        if (first_token[mid] <= t) a = mid; else b = mid - 1;
      }
      const long long pos = cached[a] + (t - first_token[a]), col = pos / block;
      const long long mine = (cached[a] + block - 1) / block;
      int page = -1;
      if (col < p.table_cols) {
        if (col < mine) {
          page = p.block_table[(r0 + a) * p.table_stride + col];
        } else {
          const long long f = first_page[a] + col - mine;
          if (f < p.n_free) page = __ldg(p.free_blocks + f);
        }
      }
      p.positions[t] = static_cast<int>(pos);
      p.slots[t] = page < 0 ? -1 : page * block + (pos - col * block);
    }
    // and of the new pages, dealt out a thread block's worth at a time
    const long long f1 = first_page[in_chunk];
    for (long long f = carry.pages + static_cast<long long>(blockIdx.x) * SLOTS_THREADS + tid; f < f1;
         f += static_cast<long long>(gridDim.x) * SLOTS_THREADS) {
      int a = 0, b = in_chunk - 1;
      while (a < b) {
        const int mid = (a + b + 1) >> 1;
        if (first_page[mid] <= f) a = mid; else b = mid - 1;
      }
      const long long col = (cached[a] + block - 1) / block + (f - first_page[a]);
      if (col < p.table_cols) p.block_table[(r0 + a) * p.table_stride + col] = f < p.n_free ? __ldg(p.free_blocks + f) : -1;
    }
    carry.tokens += total.tokens;
    carry.pages += total.pages;
  }
  for (long long t = max(lo, carry.tokens) + tid; t < hi; t += SLOTS_THREADS) {
    p.positions[t] = 0;
    p.slots[t] = -1;
  }
  if (teller) {
    __syncthreads();
    if (tid == 0) {
      p.cu_new[0] = 0;
      p.counts[0] = static_cast<int>(carry.pages);
      p.counts[1] = static_cast<int>(lost);
    }
  }
}

}  // namespace

int launch_slots(const kf_slots_args& a, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t want = ceil_div(a.max_tokens, SLOTS_THREADS * 4);
  const int64_t grid = want < 1 ? 1 : want > dev.sm_count ? dev.sm_count : want;
  slots_kernel<<<static_cast<unsigned>(grid), SLOTS_THREADS, 0, stream>>>(a);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(slots)");
}

}  // namespace kf
