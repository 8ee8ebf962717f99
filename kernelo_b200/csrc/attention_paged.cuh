// What the paged-cache attention kernels share: how the work of all requests is
// cut into equal runs of key blocks, where keys lie, and how items cut between
// CTAs are joined.
//
// An item is a row tile of one request and key head with all of its key blocks.
// Items follow one another request by request, key head by key head; the list of
// all their blocks is cut into runs of one length, one per CTA. An item takes
// ITEM_COST positions more than it has blocks, for its queries and its results,
// so that runs over many short items are no longer than those along one cache.
#pragma once

#include "attention.cuh"
#include "attention_softmax.cuh"

namespace kf {

// Workspace: arrival counters of items cut between CTAs, one per CTA, at a fixed
// place and zero between calls; then two partial results per CTA.
constexpr int64_t TREE_COUNTER_BYTES = 64 * 1024;

// The block that a CTA works on: request, key head, row tile, block of keys.
struct Cursor {
  int left;  // positions of the CTA's run from this block on
  int r, head, tile, blk;
  int row0, nodes, tiles, blocks;
  int context, length;
};

// A CTA's run: its first position and their number (0: none), and all CTAs' share.
struct Run {
  long long first, per;
  int count;
};

template <int KEYS, int ITEM_COST>
struct Walk {
  // A row tile: heads of the group that it holds (all, or an even share of
  // more than it has rows), nodes of the request, and tiles for the group.
  int tile_heads, tile_nodes, head_tiles;

  __device__ __forceinline__ Walk(const AttnArgs& p, int m) {
    const int group = static_cast<int>(p.heads / p.kv_heads);
    head_tiles = (group + m - 1) / m;
    tile_heads = (group + head_tiles - 1) / head_tiles;
    tile_nodes = m / tile_heads;
  }

  __device__ __forceinline__ void request(const AttnArgs& p, Cursor& c) const {
    int begin, end;
    request_rows(p, c.r, &begin, &end);
    long long first, length;
    request_keys(p, c.r, end - begin, &first, &length);
    c.length = static_cast<int>(length);
    c.row0 = begin;
    c.nodes = end - begin;
    c.context = c.r < p.seqs ? max(__ldg(p.context + c.r), 0) : 0;
    c.tiles = (c.nodes + tile_nodes - 1) / tile_nodes * head_tiles;
    c.blocks = max(1, (c.length + KEYS - 1) / KEYS);
  }

  __device__ __forceinline__ long long positions(const AttnArgs& p, const Cursor& c) const {
    return static_cast<long long>(c.tiles) * p.kv_heads * (c.blocks + ITEM_COST);
  }

  // From the item's last block to the next item.
  __device__ __forceinline__ void next_item(const AttnArgs& p, Cursor& c) const {
    c.left -= c.blocks + ITEM_COST - c.blk;
    c.blk = 0;
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.head < p.kv_heads) return;
    c.head = 0;
    do {
      if (++c.r > p.seqs) {
        c.left = 0;
        return;
      }
      request(p, c);
    } while (c.tiles == 0);
  }

  __device__ __forceinline__ bool item_ends(const Cursor& c) const { return c.left == 1 || c.blk + 1 == c.blocks; }

  __device__ __forceinline__ void advance(const AttnArgs& p, Cursor& c) const {
    if (c.blk + 1 < c.blocks) {
      ++c.blk;
      --c.left;
    } else {
      next_item(p, c);
    }
  }

  // Where this CTA's run begins. Positions are summed over the requests, a
  // contiguous share of them per thread, and the thread whose share holds the
  // first one finds it. Called by all threads; `at` is set where run.count > 0.
  template <int THREADS>
  __device__ __forceinline__ Run find(const AttnArgs& p, int min_run, Cursor& at) const {
    constexpr int WARPS = THREADS / 32;
    __shared__ long long scan[WARPS];
    __shared__ long long rest_of;
    __shared__ int request_of;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int share = static_cast<int>((p.seqs + 1 + THREADS - 1) / THREADS);
    const int r0 = min(static_cast<int>(p.seqs) + 1, tid * share), r1 = min(static_cast<int>(p.seqs) + 1, r0 + share);
    long long sum = 0;
    Cursor c;
    for (c.r = r0; c.r < r1; ++c.r) {
      request(p, c);
      sum += positions(p, c);
    }
    long long upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    long long before = upto - sum, total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    Run run;
    run.per = max((total + gridDim.x - 1) / gridDim.x, static_cast<long long>(min_run));
    run.first = run.per * blockIdx.x;
    run.count = static_cast<int>(max(0ll, min(run.per, total - run.first)));
    if (run.count > 0 && run.first >= before && run.first < before + sum) {
      long long rest = run.first - before;
      for (c.r = r0; c.r < r1; ++c.r) {
        request(p, c);
        const long long n = positions(p, c);
        if (rest < n) break;
        rest -= n;
      }
      request_of = c.r;
      rest_of = rest;
    }
    __syncthreads();
    if (run.count == 0) return run;
    at.r = request_of;
    request(p, at);
    const long long rest = rest_of;
    const int item = static_cast<int>(rest / (at.blocks + ITEM_COST));
    at.blk = static_cast<int>(rest - static_cast<long long>(item) * (at.blocks + ITEM_COST));
    at.head = item / at.tiles;
    at.tile = item - at.head * at.tiles;
    at.left = run.count;
    if (at.blk >= at.blocks) next_item(p, at);  // between two items
    if (at.left <= 0) run.count = 0;
    return run;
  }
};

// The rows of a tile: row i is head head0 + i % width of node node0 + i / width.
struct TileRows {
  int node0, nodes, head0, heads, width;

  template <typename W>
  __device__ __forceinline__ TileRows(const AttnArgs& p, const W& walk, const Cursor& c) {
    const int group = static_cast<int>(p.heads / p.kv_heads), part = c.tile % walk.head_tiles;
    node0 = c.tile / walk.head_tiles * walk.tile_nodes;
    nodes = min(walk.tile_nodes, c.nodes - node0);
    width = walk.tile_heads;
    head0 = c.head * group + part * width;
    heads = min(width, group - part * width);
  }
  __device__ __forceinline__ int rows() const { return nodes * width; }
  // The node (of the request) and head of row i; false if there is none.
  __device__ __forceinline__ bool find(int i, int* node, int* head) const {
    const int n = i / width, h = i - n * width;
    *node = node0 + n;
    *head = head0 + h;
    return n < nodes && h < heads;
  }
};

// n / d = n * mul >> shift for n below 2^31: with 2^s >= d, mul = ceil(2^(31 + s) / d)
// exceeds 2^(31 + s) / d by less than one, too little to reach the next quotient.
struct Divisor {
  uint32_t mul;
  int shift;
  __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
    return static_cast<uint32_t>(static_cast<uint64_t>(n) * mul >> shift);
  }
};
inline Divisor divisor(int64_t d) {
  int s = 0;
  while ((1ull << s) < static_cast<uint64_t>(d)) ++s;
  return Divisor{static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), 31 + s};
}

// Page of position `pos` of request r and its slot in it; -1 past the request's
// end and where the table names none.
__device__ __forceinline__ int page_of(const AttnArgs& p, const Divisor& by_page, const Cursor& c, int pos, int* slot) {
  *slot = 0;
  if (pos >= c.length) return -1;
  const uint32_t col = by_page(static_cast<uint32_t>(pos));
  *slot = static_cast<int>(static_cast<uint32_t>(pos) - col * static_cast<uint32_t>(p.block_size));
  const int page = __ldg(p.table + c.r * p.table_stride + col);
  return page >= 0 && page < p.pages ? page : -1;
}

// Which of the 32 keys from node j on (j may be negative: cached tokens, seen by
// all) row `node` of the request at row0 sees.
__device__ __forceinline__ uint32_t nodes_seen(const AttnArgs& p, const Cursor& c, int node, int j) {
  if (j <= -32) return 0xffffffffu;
  if (p.mask == nullptr) {
    const int n = node - j + 1;  // a chain
    return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
  }
  if (node >= c.nodes) return 0u;
  const unsigned long long* words = p.mask + static_cast<long long>(c.row0 + node) * p.mask_words;
  if (j < 0) {
    const uint32_t cached = (1u << -j) - 1u;
    return cached | (p.mask_words > 0 ? static_cast<uint32_t>(__ldg(words)) << -j : 0u);
  }
  const int w = j >> 6, b = j & 63;
  unsigned long long v = w < p.mask_words ? __ldg(words + w) >> b : 0ull;
  if (b > 32 && w + 1 < p.mask_words) v |= __ldg(words + w + 1) << (64 - b);
  return static_cast<uint32_t>(v);
}

template <typename T, int NE>
__device__ __noinline__ void redo_row(const AttnArgs& p, int t, int head, int lane) {
  // cached tokens are seen by all nodes, so only nodes can have done it
  const RowKeys keys(p, t);
  if (last_unseen_nonfinite<T, NE>(p, t, head, keys.prefix, keys.length, lane) < 0) return;
  float acc[NE], m, l;
  attend_row<T, NE>(p, t, head, lane, acc, &m, &l);
  write_row<T, NE>(p, t, head, lane, acc, m, l);
}

// A partial result in the workspace: M rows of DP sums, then maxima, then weights' sums.
template <int M, int DP>
struct Partial {
  static constexpr int64_t FLOATS = M * DP + 2 * M;
  float* at;
  __device__ __forceinline__ Partial(const AttnArgs& p, long long cta, bool second)
      : at(reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + TREE_COUNTER_BYTES) + (2 * cta + second) * FLOATS) {}
  __device__ __forceinline__ float* row(int r) const { return at + r * DP; }
  __device__ __forceinline__ float* top(int r) const { return at + M * DP + r; }
  __device__ __forceinline__ float* sum(int r) const { return at + M * DP + M + r; }
};

// Writes 8 elements of a finished row, o / l, at column `col`; true if the row has to be
// computed again, if a key that it does not see did it.
template <typename T>
__device__ __forceinline__ bool store_8(const AttnArgs& p, int t, int head, int col, const float (&o)[8], float l,
                                        int vector_out) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  float v[8], zero = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = l == 0.0f ? 0.0f : o[i] * inv;  // a row that sees nothing may hold anything
    zero = fmaf(v[i], 0.0f, zero);
  }
  T* out = static_cast<T*>(p.out) + static_cast<long long>(t) * p.so_t + head * p.so_h + col;
  if (vector_out) {
    *reinterpret_cast<uint4*>(out) = make_uint4(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]),
                                                pack_pair<T>(v[4], v[5]), pack_pair<T>(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = from_f32<T>(v[i]);
  }
  return suspect(zero == 0.0f, l);
}

__device__ __forceinline__ void store_lse(const AttnArgs& p, int t, int head, float m, float l) {
  if (p.lse != nullptr)
    p.lse[static_cast<long long>(t) * p.heads + head] = l == 0.0f ? -INFINITY : m * 0.69314718055994530942f + logf(l);
}

// Rows that may have to be computed again: `bad` and the row of each lane.
template <typename T, int NE>
__device__ __forceinline__ void redo_rows(const AttnArgs& p, bool bad, int t, int head, int lane, volatile int* flag) {
  uint32_t again = __ballot_sync(0xffffffffu, bad);
  if (again != 0) redo_begin(flag, lane);
  while (again != 0) {
    const int src = __ffs(again) - 1;
    const int row = __shfl_sync(0xffffffffu, t, src), h = __shfl_sync(0xffffffffu, head, src);
    redo_row<T, NE>(p, row, h, lane);
    again &= ~__ballot_sync(0xffffffffu, t == row && head == h);
    if (again == 0) redo_end(flag, lane);
  }
}

// A running (maximum, sum, 8 columns), and another one added to it.
struct Sums8 {
  float m = -INFINITY, l = 0.0f, o[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};

  __device__ __forceinline__ void raise(float top) {
    const float old = m == -INFINITY ? 0.0f : ex2_ftz(m - top);
    l *= old;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= old;
    m = top;
  }
  // pm <= m. A part that weighs nothing is added like any other: its sums are NaN
  // where its scores or values are (with all scores NaN its maximum is -infinity).
  __device__ __forceinline__ void add(float pm, float pl, const float (&e)[8]) {
    const float fix = pm == -INFINITY ? 0.0f : ex2_ftz(pm - m);
    l = fmaf(pl, fix, l);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fmaf(e[i], fix, o[i]);
  }
};

// Joins the partial results of CTAs [owner, last], by THREADS threads that each
// take 8 columns of a row: the owner holds the item's first blocks in its second
// slot, the others theirs in their first. With few rows several threads share a
// row's CTAs and add up through `scratch` (10 floats a thread, or null). The order
// of the sums goes by the numbers alone.
template <typename T, int M, int DP, int THREADS, typename Barrier>
__device__ __forceinline__ void join_partials(const AttnArgs& p, const Cursor& c, const TileRows& tile, int owner, int last,
                                              int tid, int vector_out, float* scratch, volatile int* flag, Barrier barrier) {
  constexpr int LANES = DP / 8, PASS = THREADS / LANES;
  const int col = (tid % LANES) * 8;
  int share = 1;  // threads to a row's CTAs
  if (scratch != nullptr)
    while (2 * share * tile.rows() <= PASS && share < 8) share *= 2;
  const int pass = PASS / share, part = tid / LANES / pass;
#pragma unroll 1
  for (int row0 = 0; row0 < tile.rows(); row0 += pass) {
    const int row = row0 + tid / LANES % pass;
    int t, head;
    const bool mine = tile.find(row, &t, &head);
    t += c.row0;
    bool bad = false;
    Sums8 sums;
    if (mine) {
#pragma unroll 1
      for (int b0 = owner + part; b0 <= last; b0 += 4 * share) {
        float pm[4], pl[4];
        float4 w[4][2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int b = b0 + x * share;
          pm[x] = -INFINITY;
          pl[x] = 0.0f;
          w[x][0] = w[x][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (b <= last) {
            const Partial<M, DP> from(p, b, b == owner);
            pm[x] = __ldcg(from.top(row));
            pl[x] = __ldcg(from.sum(row));
            w[x][0] = __ldcg(reinterpret_cast<const float4*>(from.row(row) + col));
            w[x][1] = __ldcg(reinterpret_cast<const float4*>(from.row(row) + col + 4));
          }
        }
        sums.raise(fmaxf(fmaxf(sums.m, fmaxf(pm[0], pm[1])), fmaxf(pm[2], pm[3])));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float e[8] = {w[x][0].x, w[x][0].y, w[x][0].z, w[x][0].w, w[x][1].x, w[x][1].y, w[x][1].z, w[x][1].w};
          sums.add(pm[x], pl[x], e);
        }
      }
    }
    if (share > 1) {
      float* mine_at = scratch + 10 * (tid - LANES * pass);
      if (part > 0) {
        mine_at[0] = sums.m;
        mine_at[1] = sums.l;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine_at[2 + i] = sums.o[i];
      }
      barrier();
      if (part == 0) {
        for (int x = 1; x < share; ++x) {
          const float* other = scratch + 10 * (tid + (x - 1) * LANES * pass);
          float e[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] = other[2 + i];
          sums.raise(fmaxf(sums.m, other[0]));
          sums.add(other[0], other[1], e);
        }
      }
      barrier();
    }
    if (mine && part == 0) {
      if (col < p.dim) bad = store_8<T>(p, t, head, col, sums.o, sums.l, vector_out);
      if (col == 0) store_lse(p, t, head, sums.m, sums.l);
    }
    redo_rows<T, DP / 32>(p, bad, t, head, threadIdx.x & 31, flag);
  }
}

}  // namespace kf
