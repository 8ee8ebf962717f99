// The pages of a key/value cache when requests fork, end, and are moved together.
// Request r holds the first ceil(len / block) pages of its row of the block table;
// holders[p] counts the requests that hold page p besides the first (0 for a page of
// one request and for a free one).
//
// fork: child i gets the len / block whole pages of its parent, each with one holder
//   more, and for the len % block tokens behind them a page of its own, the
//   base[i]-th of the free list with base[i] = pages taken by the pairs before it,
//   into which those tokens are copied in every cache. One launch: each block
//   counts base[i] itself (as slots.cu does) and copies some caches of one child.
// release: a page goes back when its last holder ends. Counts go down by one for
//   each holder among the requests; a page left below zero is free, and listed where the
//   first of them has it, so that the list does not depend on the atomics' order.
// compact: with L live pages, the i-th live page behind the first L goes to
//   the i-th hole among them: a plan and the table's new numbers by one
//   cluster, then the copies by the whole GPU.
//
// Plans go in phases of a few dependent accesses per page, between the barriers of one
// CTA or cluster; releases of many go in a launch a phase over the whole GPU. Copies are bound
// by their bytes. Every number read from a table or a list is checked before it is used.
//
// On the GPU: 16 requests of up to 2048 tokens forked 4 ways in 32 caches 14.7 us (36 MB, 5.5 at a copy's rate: the books
// before the copies are a chain of dependent loads), one in 2 caches 5.0; one request of 256 pages released 9.2 us, of
// 2048 13.5, 16 of 2048 31 to 34, 192 of 2048 34 to 36; 1300 of 2600 pages of 16 caches moved in 158 us (1.03 GB, a copy's
// rate) behind a plan of 13.
#include <cuda.h>

#include "kf_common.cuh"
#include "kf_internal.h"

namespace kf {
namespace {

constexpr int COPY_THREADS = 256;
constexpr int COPY_BATCH = 4;  // vectors of a thread in flight
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_WARPS = PLAN_THREADS / 32;
constexpr int PLAN_CLUSTER = 8;

constexpr int TILE_WORDS = 8, TILE = 32 * TILE_WORDS;  // columns that a warp takes at a time

// Where a run of a page's elements lies, in vectors: `outer` runs (of heads, or of heads and slots).
struct CacheShape {
  long long s_page, s_head, s_slot;  // in vectors
  int heads, row;                    // vectors of a slot's head
};

// Sum over the block of v, and of the threads before this one; `scratch` holds PLAN_WARPS ints.
template <int WARPS>
__device__ __forceinline__ int block_sum(int v, int* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) sum += scratch[w];
  return sum;
}

__device__ __forceinline__ int pages_of(int len, long long block, long long cols) {
  const long long held = (max(len, 0) + block - 1) / block;
  return static_cast<int>(min(held, cols));
}

// ---------------------------------------------------------------- fork
struct ForkArgs {
  int* table;
  long long table_stride, cols, rows;
  int* context;
  int* holders;
  long long pages, block;
  const int* free_blocks;
  long long n_free;
  const int* parents;
  const int* children;
  int pairs;
  int* counts;  // pages taken, pairs without what they need; null: another launch has kept the books
};

// Bits of rows: named as a child, named so twice, named as a parent.
struct PairBits {
  uint32_t *child, *twice, *parent;
  __device__ __forceinline__ bool valid(const ForkArgs& a, int c, int p) const {
    if (c < 0 || c >= a.rows || p < 0 || p >= a.rows) return false;
    return ((twice[c >> 5] | parent[c >> 5]) >> (c & 31) & 1u) == 0;
  }
};

template <typename V>
__global__ void __launch_bounds__(COPY_THREADS)
    fork_kernel(const __grid_constant__ PageCaches caches, const __grid_constant__ ForkArgs a, const CacheShape shape, int slices) {
  extern __shared__ uint32_t words[];
  __shared__ int scratch[COPY_THREADS / 32];
  const int tid = threadIdx.x;
  const int pair = blockIdx.x / slices, slice = blockIdx.x % slices;
  const int bit_words = static_cast<int>((a.rows + 31) / 32);
  const PairBits bits{words, words + bit_words, words + 2 * bit_words};
  for (int i = tid; i < 3 * bit_words; i += COPY_THREADS) words[i] = 0;
  __syncthreads();
  for (int i = tid; i < a.pairs; i += COPY_THREADS) {
    const int c = __ldg(a.children + i), p = __ldg(a.parents + i);
    if (c >= 0 && c < a.rows && (atomicOr(bits.child + (c >> 5), 1u << (c & 31)) >> (c & 31) & 1u) != 0)
      atomicOr(bits.twice + (c >> 5), 1u << (c & 31));
    if (p >= 0 && p < a.rows) atomicOr(bits.parent + (p >> 5), 1u << (p & 31));
  }
  __syncthreads();
  // Pages that the pairs before this one take; the first block goes on to all of them.
  const bool teller = blockIdx.x == 0 && a.counts != nullptr;
  int before = 0, taken = 0, lost = 0;
  for (int i = tid; i < (teller ? a.pairs : pair); i += COPY_THREADS) {
    const int p = __ldg(a.parents + i);
    const bool valid = bits.valid(a, __ldg(a.children + i), p);
    const bool needs = valid && min(static_cast<long long>(max(a.context[p], 0)), a.cols * a.block) % a.block != 0;
    before += needs && i < pair;
    taken += needs;
    lost += !valid;
  }
  before = block_sum<COPY_THREADS / 32>(before, scratch);
  if (teller) {
    taken = block_sum<COPY_THREADS / 32>(taken, scratch);
    lost = block_sum<COPY_THREADS / 32>(lost, scratch);
    if (tid == 0) {
      a.counts[0] = taken;
      a.counts[1] = lost + static_cast<int>(max(taken - a.n_free, 0ll));
    }
  }
  const int parent = __ldg(a.parents + pair), child = __ldg(a.children + pair);
  if (!bits.valid(a, child, parent)) return;
  const int len = static_cast<int>(min(static_cast<long long>(max(a.context[parent], 0)), a.cols * a.block));
  const int full = static_cast<int>(len / a.block), tail = static_cast<int>(len - full * a.block);
  const int target = tail > 0 && before < a.n_free ? __ldg(a.free_blocks + before) : -1;
  const int* const from = a.table + parent * a.table_stride;
  if (slice == 0 && a.counts != nullptr) {
    int* const to = a.table + child * a.table_stride;
    for (int col = tid; col < a.cols; col += COPY_THREADS) {
      int page = -1;
      if (col < full) {
        page = from[col];
        if (page >= 0 && page < a.pages) atomicAdd(a.holders + page, 1);
      } else if (col == full) {
        page = target;
      }
      to[col] = page;
    }
    if (tid == 0) a.context[child] = len;
  }
  if (target < 0 || target >= a.pages) return;
  const int source = from[full];
  if (source < 0 || source >= a.pages || source == target) return;
  // Every slices-th cache, its heads' first `tail` slots.
  const uint32_t row = shape.row, per_head = tail * row, per_cache = shape.heads * per_head;
  const uint32_t mine = slice < caches.count ? (caches.count - slice + slices - 1) / slices : 0;
  const long long s = source * shape.s_page, t = target * shape.s_page;
  for (uint32_t c = 0; c < mine; ++c) {
    V* const cache = static_cast<V*>(caches.at[slice + c * slices]);
    for (uint32_t first = tid; first < per_cache; first += COPY_BATCH * COPY_THREADS) {
      V v[COPY_BATCH];
      long long at[COPY_BATCH];
#pragma unroll
      for (int k = 0; k < COPY_BATCH; ++k) {
        const uint32_t i = first + k * COPY_THREADS;
        if (i >= per_cache) continue;
        const uint32_t head = i / per_head, in = i - head * per_head, slot = in / row;
        at[k] = head * shape.s_head + slot * shape.s_slot + (in - slot * row);
        v[k] = cache[s + at[k]];
      }
#pragma unroll
      for (int k = 0; k < COPY_BATCH; ++k)
        if (first + k * COPY_THREADS < per_cache) cache[t + at[k]] = v[k];
    }
  }
}

// ---------------------------------------------------------------- release
struct ReleaseArgs {
  int* table;
  long long table_stride, cols, rows;
  int* context;
  int* holders;
  long long pages, block;
  const int* requests;
  int count;        // of requests
  int tiles;        // of a row
  uint32_t* votes;  // [count x tiles][TILE_WORDS]: entries whose page goes back
  int* held;        // [count x tiles]: pages of the tile's request, -1 where it is skipped
  int* freed;       // [count x cols]
  int* n_freed;     // one word
};

// A free page's count says which of its places in the rows is the first: below every count that is one.
constexpr int MARK = -(1 << 30);

// Entries (request, column) go by tiles of a row, dealt out to the warps in turn (rows end early, and a run of them for
// each warp would leave most warps with nothing). The four phases, 0 to 3, are one launch of a cluster for few
// entries (PHASE -1), and otherwise a launch each over the whole GPU: an entry costs five scattered accesses, and
// a cluster's 8 SMs take 98 us for 192 of 256 requests of up to 2048 pages, the launches 34.
template <int PHASE>
__global__ void __launch_bounds__(PLAN_THREADS) release_kernel(const __grid_constant__ ReleaseArgs a) {
  __shared__ int scratch[PLAN_WARPS];
  extern __shared__ int places[];  // of the tiles that this CTA's warps have: where the first of their pages goes
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(blockIdx.x), ctas = static_cast<int>(gridDim.x);
  const int warps = ctas * PLAN_WARPS, my_warp = rank * PLAN_WARPS + warp;
  const int cols = static_cast<int>(a.cols), entries = a.count * cols, tiles = a.count * a.tiles;  // below 2^30
  if constexpr (PHASE >= 0 && PHASE < 3) griddep_launch_dependents();  // the next phase's blocks wait for this one's end
  if constexpr (PHASE > 0) griddep_wait();
  // f(tile, its number among this CTA's, request, row, first column, pages from there on) for tiles that are not skipped.
  const auto each_tile = [&](const auto& f) {
    for (int t = my_warp, n = warp; t < tiles; t += warps, n += PLAN_WARPS) {
      const int i = t / a.tiles, col = (t - i * a.tiles) * TILE, held = a.held[t];
      if (held >= 0) f(t, n, i, __ldg(a.requests + i), col, held - col);
    }
  };
  // A lane's pages of a tile, -1 where there is none.
  const auto load_pages = [&](int row, int col, int left, int (&page)[TILE_WORDS]) {
    const int* const at = a.table + row * a.table_stride + col;
#pragma unroll
    for (int k = 0; k < TILE_WORDS; ++k) {
      page[k] = lane + 32 * k < left ? at[lane + 32 * k] : -1;
      if (page[k] >= a.pages) page[k] = -1;
    }
  };
  if constexpr (PHASE <= 0) {
    // Skipped are requests whose row is none, or named by an earlier one too.
    for (int t = my_warp; t < tiles; t += warps) {
      const int i = t / a.tiles, row = __ldg(a.requests + i);
      bool skip = row < 0 || row >= a.rows;
      for (int j = lane; j < i; j += 32) skip |= __ldg(a.requests + j) == row;
      skip = __any_sync(0xffffffffu, skip);
      if (lane == 0) a.held[t] = skip ? -1 : pages_of(a.context[row], a.block, a.cols);
    }
    __syncwarp();
    each_tile([&](int, int, int, int row, int col, int left) {
      if (left <= 0) return;
      int page[TILE_WORDS];
      load_pages(row, col, left, page);
#pragma unroll
      for (int k = 0; k < TILE_WORDS; ++k)
        if (page[k] >= 0) atomicSub(a.holders + page[k], 1);
    });
  }
  if constexpr (PHASE < 0) cluster_sync_all();
  if constexpr (PHASE < 0 || PHASE == 1) {
    each_tile([&](int, int, int i, int row, int col, int left) {
      if (left <= 0) return;
      int page[TILE_WORDS], holds[TILE_WORDS];
      load_pages(row, col, left, page);
#pragma unroll
      for (int k = 0; k < TILE_WORDS; ++k) holds[k] = page[k] >= 0 ? __ldcg(a.holders + page[k]) : 0;
#pragma unroll
      for (int k = 0; k < TILE_WORDS; ++k)
        if (holds[k] < 0) atomicMin(a.holders + page[k], MARK - (entries - (i * cols + col + lane + 32 * k)));
    });
  }
  if constexpr (PHASE < 0) cluster_sync_all();
  if constexpr (PHASE < 0 || PHASE == 2) {
    for (int t = my_warp; t < tiles; t += warps) {
      const int i = t / a.tiles, col = (t - i * a.tiles) * TILE, left = a.held[t] - col;
      uint32_t mine = 0;
      if (left > 0) {
        int page[TILE_WORDS], holds[TILE_WORDS];
        load_pages(__ldg(a.requests + i), col, left, page);
#pragma unroll
        for (int k = 0; k < TILE_WORDS; ++k) holds[k] = page[k] >= 0 ? __ldcg(a.holders + page[k]) : 0;
#pragma unroll
        for (int k = 0; k < TILE_WORDS; ++k) {
          const uint32_t vote = __ballot_sync(
              0xffffffffu, page[k] >= 0 && holds[k] == MARK - (entries - (i * cols + col + lane + 32 * k)));
          if (lane == k) mine = vote;
        }
      }
      if (lane < TILE_WORDS) a.votes[t * TILE_WORDS + lane] = mine;
    }
  }
  if constexpr (PHASE < 0) cluster_sync_all();
  if constexpr (PHASE < 0 || PHASE == 3) {
    // Each CTA counts all tiles' votes itself, a run of tiles to each thread, and keeps the places of its own tiles.
    const int run = (tiles + PLAN_THREADS - 1) / PLAN_THREADS;
    const int t0 = min(tid * run, tiles), t1 = min(t0 + run, tiles);
    const auto votes_of = [&](int t) {
      int n = 0;
#pragma unroll
      for (int k = 0; k < TILE_WORDS; k += 4) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4*>(a.votes + t * TILE_WORDS + k));
        n += __popc(v.x) + __popc(v.y) + __popc(v.z) + __popc(v.w);
      }
      return n;
    };
    int mine = 0;
    for (int t = t0; t < t1; ++t) mine += votes_of(t);
    int in = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += up;
    }
    if (lane == 31) scratch[warp] = in;
    __syncthreads();
    int place = in - mine, all = 0;
    for (int w = 0; w < PLAN_WARPS; ++w) {
      place += w < warp ? scratch[w] : 0;
      all += scratch[w];
    }
    for (int t = t0; t < t1; ++t) {
      if (t % warps / PLAN_WARPS == rank) places[t / warps * PLAN_WARPS + t % PLAN_WARPS] = place;
      place += votes_of(t);
    }
    __syncthreads();
    each_tile([&](int t, int n, int, int row, int col, int) {
      int* const at = a.table + row * a.table_stride + col;
      const uint32_t votes = lane < TILE_WORDS ? __ldcg(a.votes + t * TILE_WORDS + lane) : 0;
      int to = places[n];
#pragma unroll
      for (int k = 0; k < TILE_WORDS; ++k) {
        const uint32_t vote = __shfl_sync(0xffffffffu, votes, k);
        if ((vote >> lane & 1u) != 0) {
          const int page = at[lane + 32 * k];
          a.freed[to + __popc(vote & ((1u << lane) - 1))] = page;
          a.holders[page] = 0;
        }
        to += __popc(vote);
        if (col + lane + 32 * k < cols) at[lane + 32 * k] = -1;
      }
    });
    for (int e = all + rank * PLAN_THREADS + tid; e < entries; e += ctas * PLAN_THREADS) a.freed[e] = -1;
    if (rank == 0 && tid == 0) *a.n_freed = all;
    for (int i = rank * PLAN_THREADS + tid; i < a.count; i += ctas * PLAN_THREADS) {
      const int row = __ldg(a.requests + i);
      if (row >= 0 && row < a.rows) a.context[row] = 0;
    }
  }
}

// ---------------------------------------------------------------- compact
struct CompactArgs {
  int* table;
  long long table_stride, cols, rows;
  const int* context;
  int* holders;
  long long pages, block;
  int* renamed;  // [pages]
  int* sources;  // [pages / 2]: pages that move, in order
  int* targets;  // [pages / 2]: where to
  int* counts;   // live pages, moves
};

__device__ __forceinline__ uint32_t cluster_load(const void* mine, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(mine), rank)) : "memory");
  return v;
}

// live: one bit a page, `own` words in each CTA; before: live pages of the CTA in front of each word.
__global__ void __launch_bounds__(PLAN_THREADS) compact_plan_kernel(const __grid_constant__ CompactArgs a, int own) {
  extern __shared__ uint32_t words[];
  __shared__ int scratch[PLAN_WARPS];
  __shared__ int cta_total, cta_rank_of_live;
  uint32_t* const live = words;
  uint32_t* const before = words + own;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(cluster_ctarank()), ctas = gridDim.x;
  const int all_threads = ctas * PLAN_THREADS, me = rank * PLAN_THREADS + tid;
  for (int i = tid; i < own; i += PLAN_THREADS) live[i] = 0;
  cluster_sync_all();
  // A warp takes pieces of a row, 32 x BATCH columns each.
  const int warps = ctas * PLAN_WARPS, my_warp = rank * PLAN_WARPS + warp;
  constexpr int BATCH = 4;
  const long long per_row = max((a.cols + 32 * BATCH - 1) / (32 * BATCH), 1ll);
  for (long long piece = my_warp;; piece += warps) {
    const long long r = piece / per_row;
    if (r >= a.rows) break;
    const int held = pages_of(__ldg(a.context + r), a.block, a.cols);
    const int col = static_cast<int>(piece - r * per_row) * 32 * BATCH + lane;
    int page[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) page[k] = col + 32 * k < held ? a.table[r * a.table_stride + col + 32 * k] : -1;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      if (page[k] < 0 || page[k] >= a.pages) continue;
      const int word = page[k] >> 5, owner = word / own;
      asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(
                       mapa_shared(smem_u32(live + (word - owner * own)), owner)),
                   "r"(1u << (page[k] & 31))
                   : "memory");
    }
  }
  cluster_sync_all();
  // Each thread counts a run of words; then the runs in front of it.
  const int run = (own + PLAN_THREADS - 1) / PLAN_THREADS;
  const int w0 = min(tid * run, own), w1 = min(w0 + run, own);
  int mine = 0;
  for (int w = w0; w < w1; ++w) mine += __popc(live[w]);
  int in = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += up;
  }
  if (lane == 31) scratch[warp] = in;
  __syncthreads();
  int front = in - mine, total = 0;
  for (int w = 0; w < PLAN_WARPS; ++w) {
    front += w < warp ? scratch[w] : 0;
    total += scratch[w];
  }
  if (tid == 0) cta_total = total;
  for (int w = w0; w < w1; ++w) {
    before[w] = front;
    front += __popc(live[w]);
  }
  cluster_sync_all();
  int base = 0, count = 0;  // live pages of the CTAs in front, and of all
  for (int r = 0; r < ctas; ++r) {
    const int theirs = static_cast<int>(cluster_load(&cta_total, r));
    base += r < rank ? theirs : 0;
    count += theirs;
  }
  // Live pages among the first `count`: those that stay.
  const int first_word = rank * own;
  if (tid == 0) cta_rank_of_live = 0;
  __syncthreads();
  const int edge = (count >> 5) - first_word;  // word that holds page `count`
  if (tid == 0 && edge >= 0 && edge < own)
    cta_rank_of_live = base + static_cast<int>(before[edge]) + __popc(live[edge] & ((1u << (count & 31)) - 1));
  cluster_sync_all();
  int stay = 0;
  for (int r = 0; r < ctas; ++r) stay += static_cast<int>(cluster_load(&cta_rank_of_live, r));
  if (count >= a.pages) stay = count;  // a full pool: page `count` has no word
  // Pages by their bit: a warp a word.
  for (int w = warp; w < own; w += PLAN_WARPS) {
    const long long page = static_cast<long long>(first_word + w) * 32 + lane;
    if (page >= a.pages) continue;
    const uint32_t bits = live[w];
    const int at = base + static_cast<int>(before[w]) + __popc(bits & ((1u << lane) - 1));  // live pages in front
    const bool is_live = (bits >> lane & 1u) != 0;
    const int p = static_cast<int>(page);
    if (is_live && p < count) a.renamed[p] = p;
    if (is_live && p >= count) a.sources[at - stay] = p;
    if (!is_live) {
      a.renamed[p] = -1;
      a.holders[p] = 0;
      if (p < count) a.targets[p - at] = p;
    }
  }
  if (me == 0) {
    a.counts[0] = count;
    a.counts[1] = count - stay;
  }
  cluster_sync_all();
  for (int i = me; i < count - stay; i += all_threads) {
    const int from = a.sources[i], to = a.targets[i];
    a.renamed[from] = to;
    a.holders[to] = a.holders[from];
    a.holders[from] = 0;
  }
  cluster_sync_all();
  for (long long piece = my_warp;; piece += warps) {
    const long long r = piece / per_row;
    if (r >= a.rows) break;
    const int held = pages_of(__ldg(a.context + r), a.block, a.cols);
    const int col = static_cast<int>(piece - r * per_row) * 32 * BATCH + lane;
    int* const at = a.table + r * a.table_stride + col;
    int page[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) page[k] = col + 32 * k < held ? at[32 * k] : -1;
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
      if (page[k] >= count && page[k] < a.pages) at[32 * k] = a.renamed[page[k]];
  }
}

// Whole pages, `outer` x `inner` runs of `run` vectors each; a block takes (move, cache) pairs in turn.
struct MoveShape {
  long long s_page, s_outer, s_inner;
  uint32_t outer, inner, run;
};

template <typename V>
__global__ void __launch_bounds__(COPY_THREADS)
    move_pages_kernel(const __grid_constant__ PageCaches caches, const MoveShape shape, const int* sources, const int* targets,
                      const int* counts) {
  const long long units = static_cast<long long>(counts[1]) * caches.count;
  const uint32_t per_outer = shape.inner * shape.run, total = shape.outer * per_outer;
  for (long long unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int move = static_cast<int>(unit / caches.count);
    V* const cache = static_cast<V*>(caches.at[unit - static_cast<long long>(move) * caches.count]);
    const V* const from = cache + __ldg(sources + move) * shape.s_page;
    V* const to = cache + __ldg(targets + move) * shape.s_page;
    for (uint32_t first = threadIdx.x; first < total; first += COPY_BATCH * COPY_THREADS) {
      V v[COPY_BATCH];
      long long at[COPY_BATCH];
#pragma unroll
      for (int k = 0; k < COPY_BATCH; ++k) {
        const uint32_t i = first + k * COPY_THREADS;
        if (i >= total) continue;
        const uint32_t o = i / per_outer, rest = i - o * per_outer, n = rest / shape.run;
        at[k] = o * shape.s_outer + n * shape.s_inner + (rest - n * shape.run);
        v[k] = from[at[k]];
      }
#pragma unroll
      for (int k = 0; k < COPY_BATCH; ++k)
        if (first + k * COPY_THREADS < total) to[at[k]] = v[k];
    }
  }
}

// Bytes of the widest vectors that heads, strides and addresses hold whole.
int vector_bytes(const PageCaches& caches, const PageGeometry& g) {
  for (int bytes = 16; bytes > g.elem; bytes /= 2) {
    const int64_t n = bytes / g.elem;
    bool fits = g.dim % n == 0 && g.s_page % n == 0 && g.s_head % n == 0 && g.s_slot % n == 0;
    for (int c = 0; c < caches.count && fits; ++c) fits = reinterpret_cast<uintptr_t>(caches.at[c]) % bytes == 0;
    if (fits) return bytes;
  }
  return g.elem;
}

// Calls f with a vector's type of that many bytes.
template <typename F>
int with_vector(int bytes, const F& f) {
  switch (bytes) {
    case 16: return f(uint4{});
    case 8: return f(uint2{});
    case 4: return f(uint32_t{});
    default: return f(uint16_t{});
  }
}

int launched(const char* what) {
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, what);
}

template <typename Kernel, typename... Args>
int launch_plan(Kernel kernel, int ctas, int smem, const cudaLaunchAttribute* attribute, cudaStream_t stream, const char* what,
                const Args&... args) {
  if (smem > 48 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return cuda_error(err, what);
  }
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(ctas));
  config.blockDim = dim3(PLAN_THREADS);
  config.dynamicSmemBytes = static_cast<size_t>(smem);
  config.stream = stream;
  cudaLaunchAttribute copy{};
  if (attribute != nullptr) copy = *attribute;
  config.attrs = &copy;
  config.numAttrs = attribute != nullptr ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, args...);
  return err == cudaSuccess ? KF_OK : cuda_error(err, what);
}

template <typename Kernel, typename... Args>
int launch_cluster(Kernel kernel, int ctas, int smem, cudaStream_t stream, const char* what, const Args&... args) {
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = static_cast<unsigned>(ctas);
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  return launch_plan(kernel, ctas, smem, &cluster, stream, what, args...);
}

// A launch behind another of this call starts while that one ends, and waits for it where it needs its results.
template <typename Kernel, typename... Args>
int launch_behind(Kernel kernel, int ctas, int smem, cudaStream_t stream, const char* what, const Args&... args) {
  cudaLaunchAttribute behind{};
  behind.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  behind.val.programmaticStreamSerializationAllowed = 1;
  return launch_plan(kernel, ctas, smem, &behind, stream, what, args...);
}

// One CTA where it does the work in a few rounds: its barriers are cheaper than a cluster's.
int plan_ctas(int64_t entries) { return entries <= 8 * PLAN_THREADS ? 1 : PLAN_CLUSTER; }

}  // namespace

int launch_fork(const PageCaches& all, const PageGeometry& g, const kf_fork_args& f, const DeviceInfo& dev,
                cudaStream_t stream) {
  ForkArgs a{f.block_table, f.table_stride, f.table_cols, f.rows, f.context, f.holders, g.pages, g.block, f.free_blocks,
             f.n_free, f.parents, f.children, static_cast<int>(f.pairs), f.counts};
  const int64_t smem = 3 * ceil_div(f.rows, 32) * 4;
  const int bytes = vector_bytes(all, g);
  const int64_t n = bytes / g.elem;
  const CacheShape shape{g.s_page / n, g.s_head / n, g.s_slot / n, static_cast<int>(g.heads), static_cast<int>(g.dim / n)};
  // Enough blocks to fill the GPU, as far as there are caches.
  int64_t slices = ceil_div(6 * dev.sm_count, f.pairs);
  if (slices > all.count) slices = all.count;
  if (slices < 1) slices = 1;
  return with_vector(bytes, [&](auto v) {
    const auto kernel = fork_kernel<decltype(v)>;
    if (smem > 48 * 1024) {
      const cudaError_t err =
          cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
      if (err != cudaSuccess) return cuda_error(err, "attributes(fork)");
    }
    kernel<<<static_cast<unsigned>(f.pairs * slices), COPY_THREADS, static_cast<size_t>(smem), stream>>>(
        all, a, shape, static_cast<int>(slices));
    return launched("launch(fork)");
  });
}

int launch_release(const kf_release_args& r, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t parts = ceil_div(r.table_cols, TILE), tiles = r.count * parts;
  const ReleaseArgs a{r.block_table, r.table_stride, r.table_cols, r.rows, r.context, r.holders, r.pages, r.block_size,
                      r.requests, static_cast<int>(r.count), static_cast<int>(parts),
                      reinterpret_cast<uint32_t*>(r.scratch), r.scratch + tiles * TILE_WORDS, r.freed, r.n_freed};
  const auto smem = [&](int ctas) { return static_cast<int>(ceil_div(tiles, ctas * PLAN_WARPS) * PLAN_WARPS * 4); };
  // One CTA takes 9 us and 4 more by 2048 pages; a cluster 28 to 32 us for 8192 pages and 31 to 34 for 32768, where the
  // four launches take 33 to 34, and 34 to 36 for 393216.
  if (tiles * TILE <= 32768) {
    const int ctas = plan_ctas(tiles * TILE);
    return launch_cluster(release_kernel<-1>, ctas, smem(ctas), stream, "launch(release)", a);
  }
  const int64_t want = ceil_div(tiles, PLAN_WARPS);
  const int ctas = static_cast<int>(want < dev.sm_count ? want : dev.sm_count);
  int rc = launch_plan(release_kernel<0>, ctas, 0, nullptr, stream, "launch(release)", a);
  if (rc == KF_OK) rc = launch_behind(release_kernel<1>, ctas, 0, stream, "launch(release marks)", a);
  if (rc == KF_OK) rc = launch_behind(release_kernel<2>, ctas, 0, stream, "launch(release votes)", a);
  if (rc == KF_OK) rc = launch_behind(release_kernel<3>, ctas, smem(ctas), stream, "launch(release list)", a);
  return rc;
}

int launch_compact_plan(const kf_compact_args& c, const PageGeometry& g, const DeviceInfo& dev, cudaStream_t stream) {
  const CompactArgs a{c.block_table, c.table_stride, c.table_cols, c.rows, c.context, c.holders,
                      g.pages,       g.block,        c.renamed,    c.sources, c.targets, c.counts};
  const int64_t entries = c.rows * c.table_cols > g.pages ? c.rows * c.table_cols : g.pages;
  const int ctas = plan_ctas(entries);
  const int64_t own = ceil_div(ceil_div(g.pages, 32) > 0 ? ceil_div(g.pages, 32) : 1, ctas);
  return launch_cluster(compact_plan_kernel, ctas, static_cast<int>(own * 8), stream, "launch(compact plan)", a,
                        static_cast<int>(own));
}

int launch_move_pages(const PageCaches& caches, const PageGeometry& g, const kf_compact_args& c, const DeviceInfo& dev,
                      cudaStream_t stream) {
  const int bytes = vector_bytes(caches, g);
  const int64_t n = bytes / g.elem;
  // Runs as long as the strides make them: whole pages, heads, or single slots.
  MoveShape shape{g.s_page / n, g.s_head / n, g.s_slot / n, static_cast<uint32_t>(g.heads), static_cast<uint32_t>(g.block),
                  static_cast<uint32_t>(g.dim / n)};
  if (g.s_slot == g.dim || g.block == 1) shape.run *= shape.inner, shape.inner = 1;
  if (shape.inner == 1 && (g.s_head == g.block * g.dim || g.heads == 1)) shape.run *= shape.outer, shape.outer = 1;
  // Ten times as many blocks as run at once, so that SMs that are ahead take more: 1.03 GB 158 us; 8 blocks to an SM 180.
  const int64_t most = (g.pages / 2) * caches.count, enough = 64ll * dev.sm_count;
  const int64_t blocks = most < enough ? most : enough;
  if (blocks < 1) return KF_OK;
  return with_vector(bytes, [&](auto v) {
    move_pages_kernel<decltype(v)><<<static_cast<unsigned>(blocks), COPY_THREADS, 0, stream>>>(caches, shape, c.sources,
                                                                                              c.targets, c.counts);
    return launched("launch(move pages)");
  });
}

}  // namespace kf
