// Attention of many drafted tokens over a paged cache (more than 16 rows to a key
// head: nodes x heads of the group), fp16/bf16, heads of up to 128 elements.
//
// The list of key blocks, its runs and the joining of items cut between CTAs are
// those of attention_paged.cuh; a row tile is 128 rows on the 5th-generation
// tensor cores, so up to 128 rows cost one pass over the cache:
//
//   warp 4     loads: queries of the next item, then K and V blocks of 128 keys
//              through a ring, a TMA box per run of keys that is whole in any page.
//   warp 5     issues the MMAs. S = Q K^T of the next block runs while the softmax
//              warps work on this one (two S buffers); O alternates between two
//              buffers item by item, so an item starts while the last is written.
//   warps 0-3  softmax and results, a thread per row: S from TMEM, P (16 bit) back
//              over its columns, O += P V by the tensor cores; m is raised and O
//              rescaled only when a row's maximum grew by more than 2^8.
//
// 128 keys of one head are 64 KB: 1.5 us of this SM's share of the HBM's rate, in
// which the two products take 0.55 us and 128 x 128 exponentials 0.55 us, so the
// cache's bytes bound the call; with mma.sync tiles of 64 rows the products did
// (1.2 us per 64 keys). 16 trees of up to 16 nodes over up to 8192 keys, 32 heads to 8 of 128 elements: 84 us,
// 276 MB at 3.3 TB/s (102 on mma.sync tiles); what is left are the latencies between
// a block's two products and its softmax, since 64 rows of a tile's 128 are real.
#include <cuda.h>

#include <mutex>
#include <numeric>
#include <string>

#include "attention_paged.cuh"

namespace kf {
namespace {

constexpr int M = 128;
constexpr int KEYS = 128;
constexpr int SOFTMAX_WARPS = 4;
constexpr int LOAD_WARP = 4, MMA_WARP = 5;
constexpr int THREADS = 6 * 32;
constexpr int MIN_RUN = 2;
constexpr int ITEM_COST = 2;
constexpr int INFO = 16;  // blocks whose `present` bits are kept: more than the loads run ahead
constexpr uint32_t TMEM_COLS = 512;  // S0 | S1 | O0 | O1, 128 each
constexpr uint64_t DRAIN_NS = 100000000ull;

template <int DP_>
struct Shape {
  static constexpr int DP = DP_;
  static constexpr int HALVES = DP / 64;
  static constexpr int TILE = KEYS * DP * 2;        // bytes of a Q, K or V tile
  static constexpr int STAGES = DP == 128 ? 5 : 8;  // K and V tiles in flight
  static constexpr int BARS = 4 + 2 * STAGES + INFO + 4 + 2 + 2 + 1;
  static constexpr int SMEM = 1024 + (2 + STAGES) * TILE + 8 * BARS + 16 * INFO;
};

template <typename T, int DP>
__global__ void __launch_bounds__(THREADS, 1)
    tree_wide_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnArgs p, const Divisor by_page,
                     int box_rows, int vector_out, int* status) {
  using S = Shape<DP>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* q_tiles = smem;
  uint8_t* ring = smem + 2 * S::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + STAGES * S::TILE);
  volatile uint32_t* present = reinterpret_cast<volatile uint32_t*>(bars + S::BARS);  // 4 words per block
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, last_one;
  volatile int* abort_flag = &abort_word;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t q_full = smem_u32(bars), q_empty = q_full + 16, full = q_empty + 16, empty = full + 8 * STAGES,
                 info = empty + 8 * STAGES, s_full = info + 8 * INFO, p_full = s_full + 16, o_done = p_full + 16,
                 o_free = o_done + 16, drain = o_free + 16;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, SOFTMAX_WARPS);
      mbar_init(o_done + 8 * i, 1);
      mbar_init(o_free + 8 * i, SOFTMAX_WARPS);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int i = 0; i < INFO; ++i) mbar_init(info + 8 * i, 1);
    mbar_init(drain, 1);
    abort_word = 0;
    mbar_init_fence();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == MMA_WARP) {
    tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  const Walk<KEYS, ITEM_COST> walk(p, M);
  Cursor at;
  const Run run = walk.template find<THREADS>(p, MIN_RUN, at);  // ends in a barrier of the CTA
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // A wait that gives up records its status and all warps go on together: the
  // results are lost, the barriers between the warps are not.
  if (run.count == 0) {
    // nothing of the list; only the TMEM to give back
  } else if (warp == LOAD_WARP) {
    int issued = 0, items = 0, unit = 0;
    bool fresh = true;
    // V of a block follows K of the next: its pages are kept
    int v_page = -1, v_slot = 0, v_head = 0;
    const bool mine = lane * box_rows < KEYS;
    auto load = [&](const CUtensorMap* map, int page, int slot_in_page, int head) {
      const int slot = issued % STAGES;
      attn_wait(empty + 8 * slot, ((issued / STAGES) & 1) ^ 1, abort_flag, status, SITE_ATTN_LOAD);
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(full + 8 * slot, S::TILE);
      __syncwarp();
      if (mine) {
#pragma unroll
        for (int x = 0; x < S::HALVES; ++x)
          tma_load_4d(smem_u32(ring + slot * S::TILE) + x * KEYS * 128 + lane * box_rows * 128, map, full + 8 * slot, 64 * x,
                      slot_in_page, head, page >= 0 ? page : static_cast<int>(p.pages));
      }
      __syncwarp();
      ++issued;
    };
    while (at.left > 0) {
      if (fresh) {
        const int buf = items & 1;
        attn_wait(q_empty + 8 * buf, ((items >> 1) & 1) ^ 1, abort_flag, status, SITE_ATTN_LOAD);
        __syncwarp();
        if (lane == 0) {
          const TileRows tile(p, walk, at);
          mbar_arrive_expect_tx(q_full + 8 * buf, walk.tile_heads * walk.tile_nodes * 128 * S::HALVES);
#pragma unroll
          for (int x = 0; x < S::HALVES; ++x)
            tma_load_3d(smem_u32(q_tiles + buf * S::TILE) + x * M * 128, &tm_q, q_full + 8 * buf, 64 * x, tile.head0,
                        at.row0 + tile.node0);
        }
        __syncwarp();
        ++items;
      }
      const int pos = at.blk * KEYS + lane * box_rows;
      int slot = 0;
      const int page = mine ? page_of(p, by_page, at, pos, &slot) : -1;
      // a bit per key that is there
      const int rows = page >= 0 ? min(box_rows, at.length - pos) : 0;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int from = lane * box_rows - 32 * w;  // the run's first key in this word
        uint32_t b = 0u;
        if (rows > 0 && from < 32 && from + rows > 0) {
          const int lo = max(from, 0), hi = min(from + rows, 32);
          b = (hi == 32 ? 0xffffffffu : (1u << hi) - 1u) & ~((1u << lo) - 1u);
        }
        b = __reduce_or_sync(0xffffffffu, b);
        if (lane == 0) present[4 * (unit % INFO) + w] = b;
      }
      if (lane == 0) mbar_arrive(info + 8 * (unit % INFO));
      load(&tm_k, page, slot, at.head);
      if (unit > 0) load(&tm_v, v_page, v_slot, v_head);
      v_page = page;
      v_slot = slot;
      v_head = at.head;
      ++unit;
      fresh = walk.item_ends(at);
      walk.advance(p, at);
    }
    load(&tm_v, v_page, v_slot, v_head);
    if (*abort_flag & 1) {  // let the copies in flight land before the shared memory goes away
      for (int i = 0; i < 2 && i < items; ++i)
        mbar_wait(q_full + 8 * i, ((items - 1 - i) >> 1) & 1, nullptr, status, SITE_DRAIN, DRAIN_NS);
      for (int s = 0; s < STAGES && s < issued; ++s)
        mbar_wait(full + 8 * s, ((issued - 1 - s) / STAGES) & 1, nullptr, status, SITE_DRAIN, DRAIN_NS);
    }
  } else if (warp == MMA_WARP) {
    const uint32_t fmt = DType<T>::code == KF_BF16 ? 1u : 0u;
    const uint32_t idesc_s = instr_desc_f16(fmt, 0, 0, M, KEYS), idesc_o = instr_desc_f16(fmt, 0, 1, M, DP);
    int taken = 0, items = 0, unit = 0;
    auto wait = [&](uint32_t bar, int parity) {
      attn_wait(bar, parity, abort_flag, status, SITE_ATTN_MMA);
      __syncwarp();
      tc_fence_after();
    };
    auto wait_tile = [&]() {
      const int slot = taken % STAGES;
      wait(full + 8 * slot, (taken / STAGES) & 1);
      ++taken;
      return slot;
    };
    // S of block `u`, the first of its item if `first`, the last of it if `last`
    auto scores = [&](int u, bool first, bool last) {
      if (first) {
        wait(q_full + 8 * (items & 1), (items >> 1) & 1);
        ++items;
      }
      const int buf = (items - 1) & 1, slot = wait_tile();
      if (lane == 0) {
        const uint64_t a = smem_desc_sw128(smem_u32(q_tiles + buf * S::TILE), 16, 1024);
        const uint64_t b = smem_desc_sw128(smem_u32(ring + slot * S::TILE), 16, 1024);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint64_t step = static_cast<uint64_t>((k / 4) * (KEYS * 128 / 16) + (k % 4) * 2);
          tc_mma_f16(tmem + (u & 1) * KEYS, a + step, b + step, idesc_s, k > 0);
        }
        tc_commit(s_full + 8 * (u & 1));
        tc_commit(empty + 8 * slot);
        if (last) tc_commit(q_empty + 8 * buf);
      }
      __syncwarp();
    };
    int done_items = 0;
    bool first = true;
    scores(0, true, walk.item_ends(at));
    while (at.left > 0) {
      Cursor next = at;
      walk.advance(p, next);
      const bool last = walk.item_ends(at);
      if (next.left > 0) scores(unit + 1, last, walk.item_ends(next));
      const int slot = wait_tile();
      const int held = at.length - at.blk * KEYS;  // keys of the request in this block
      if (held < KEYS) {
        const int from = max(held, 0);
        for (int i = lane; i < (KEYS - from) * S::HALVES * 8; i += 32) {
          const int h = i / ((KEYS - from) * 8), rest = i - h * (KEYS - from) * 8;
          *reinterpret_cast<uint4*>(ring + slot * S::TILE + h * KEYS * 128 + from * 128 + rest * 16) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
      }
      const int buf = done_items & 1;
      if (first) wait(o_free + 8 * buf, ((done_items >> 1) & 1) ^ 1);
      const uint64_t b = smem_desc_sw128(smem_u32(ring + slot * S::TILE), KEYS * 128, 1024);
      auto products = [&](int k0, int k1) {
#pragma unroll
        for (int k = k0; k < k1; ++k)
          tc_mma_f16_ta(tmem + 2 * KEYS + buf * 128, tmem + (unit & 1) * KEYS + 8 * k, b + static_cast<uint64_t>(k * 128),
                        idesc_o, !first || k > 0);
      };
      wait(p_full + 8 * (unit & 1), (unit >> 1) & 1);
      if (lane == 0) {
        products(0, KEYS / 16);
        tc_commit(o_done + 8 * (unit & 1));
        tc_commit(empty + 8 * slot);
      }
      __syncwarp();
      first = last;
      done_items += last;
      ++unit;
      at = next;
    }
    if (lane == 0) {  // the last products are done before the TMEM goes back
      tc_commit(drain);
      mbar_wait(drain, 0, nullptr, status, SITE_DRAIN, DRAIN_NS);
    }
    __syncwarp();
  } else {
    const int row = warp * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const float c = p.scale_log2;
    const auto join = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * SOFTMAX_WARPS) : "memory"); };
    float m = -INFINITY, l = 0.0f;
    int items = 0, node = 0, head = 0;
    bool first = true, real = false;
    for (int unit = 0; at.left > 0; ++unit) {
      const uint32_t s_addr = lanes + (unit & 1) * KEYS, o_addr = lanes + 2 * KEYS + (items & 1) * 128;
      if (first) {
        m = -INFINITY;
        l = 0.0f;
        real = TileRows(p, walk, at).find(row, &node, &head);
      }
      attn_wait(info + 8 * (unit % INFO), (unit / INFO) & 1, abort_flag, status, SITE_ATTN_SOFTMAX);
      attn_wait(s_full + 8 * (unit & 1), (unit >> 1) & 1, abort_flag, status, SITE_ATTN_SOFTMAX);
      // A parity says "done" of the phase before the last one too, so no phase of
      // o_done may be skipped; S of this block was issued behind those products.
      if (unit >= 2) attn_wait(o_done + 8 * (unit & 1), ((unit >> 1) - 1) & 1, abort_flag, status, SITE_ATTN_SOFTMAX);
      __syncwarp();
      tc_fence_after();
      float s[KEYS];
#pragma unroll
      for (int x = 0; x < KEYS; x += 32) tmem_ld_32(s_addr + x, reinterpret_cast<uint32_t*>(s + x));
      tmem_ld_wait();
      const int key0 = at.blk * KEYS;
      uint32_t seen[4], both = 0xffffffffu;
#pragma unroll
      for (int w = 0; w < 4; ++w) both &= seen[w] = present[4 * (unit % INFO) + w];
      // a block of cached tokens, all there, needs no look at its keys
      const bool all_seen = key0 + KEYS <= at.context && both == 0xffffffffu;
      if (!all_seen) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          seen[w] &= nodes_seen(p, at, node, key0 + 32 * w - at.context);
#pragma unroll
          for (int x = 0; x < 32; ++x)
            if (!((seen[w] >> x) & 1u)) s[32 * w + x] = -INFINITY;
        }
      }
      __syncwarp();
      const float m_new = row_max(s, m);
      if (first) {
        m = m_new;
      } else if (__any_sync(0xffffffffu, (m_new - m) * c > RAISE_LOG2)) {
        attn_wait(o_done + 8 * ((unit - 1) & 1), ((unit - 1) >> 1) & 1, abort_flag, status, SITE_ATTN_SOFTMAX);
        __syncwarp();
        tc_fence_after();
        const float fix = m_new > m ? ex2_ftz((m - m_new) * c) : 1.0f;
        l *= fix;
        m = m_new;
#pragma unroll 1
        for (int x = 0; x < DP; x += 32) {
          uint32_t o[32];
          tmem_ld_32(o_addr + x, o);
          tmem_ld_wait();
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * fix);
          tmem_st_32(o_addr + x, o);
        }
      }
      const float cm = m == -INFINITY ? 0.0f : fmaf(m, c, WEIGHT_SHIFT<T>);
      l += row_weights<T, false>(s, c, cm, s_addr, 0, p_full + 8 * (unit & 1), lane);
      first = walk.item_ends(at);
      if (!first) {
        walk.advance(p, at);
        continue;
      }

      // The item's last block of this run: its result, or its partial one.
      attn_wait(o_done + 8 * (unit & 1), (unit >> 1) & 1, abort_flag, status, SITE_ATTN_SOFTMAX);
      __syncwarp();
      tc_fence_after();
      const int item = run.count - at.left - at.blk;
      const bool whole = item >= 0 && at.blk + 1 == at.blocks;
      const Partial<M, DP> part(p, blockIdx.x, item >= 0);
      const int t = at.row0 + node;
      const float top2 = m == -INFINITY ? -INFINITY : fmaf(m, c, WEIGHT_SHIFT<T>);  // base 2, as the partial results keep it
      bool bad = false;
#pragma unroll 1
      for (int x = 0; x < DP; x += 32) {
        uint32_t o[32];
        tmem_ld_32(o_addr + x, o);
        tmem_ld_wait();
        if (real) {
#pragma unroll
          for (int y = 0; y < 32; y += 8) {
            const float v[8] = {__uint_as_float(o[y]),     __uint_as_float(o[y + 1]), __uint_as_float(o[y + 2]),
                                __uint_as_float(o[y + 3]), __uint_as_float(o[y + 4]), __uint_as_float(o[y + 5]),
                                __uint_as_float(o[y + 6]), __uint_as_float(o[y + 7])};
            if (whole) {
              if (x + y < p.dim) bad = store_8<T>(p, t, head, x + y, v, l, vector_out) || bad;
            } else {
              __stcg(reinterpret_cast<float4*>(part.row(row) + x + y), make_float4(v[0], v[1], v[2], v[3]));
              __stcg(reinterpret_cast<float4*>(part.row(row) + x + y + 4), make_float4(v[4], v[5], v[6], v[7]));
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free + 8 * (items & 1));
      ++items;
      if (whole) {
        if (real) store_lse(p, t, head, top2, l);
        redo_rows<T, DP / 32>(p, bad, t, head, lane, abort_flag);
      } else {
        if (real) {
          __stcg(part.top(row), top2);
          __stcg(part.sum(row), l);
        }
        int* counters = static_cast<int*>(p.workspace);
        const int owner = static_cast<int>((run.first + item) / run.per);
        const int last = static_cast<int>((run.first + item + at.blocks - 1) / run.per);
        __threadfence();
        join();
        if (tid == 0) last_one = atomicAdd(counters + owner, 1) == last - owner;
        join();
        if (last_one) {
          __threadfence();
          join_partials<T, M, DP, 32 * SOFTMAX_WARPS>(p, at, TileRows(p, walk, at), owner, last, tid, vector_out, nullptr, abort_flag, join);
          if (tid == 0) counters[owner] = 0;
        }
        join();
      }
      walk.advance(p, at);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(tmem, TMEM_COLS);
}

int box_rows_of(const AttnArgs& a) { return static_cast<int>(std::gcd(a.block_size, static_cast<int64_t>(KEYS))); }

// The host's copy of Walk's row tile.
void tile_of(const AttnArgs& a, int* heads, int* nodes) {
  const int64_t group = a.heads / a.kv_heads, parts = ceil_div(group, M);
  *heads = static_cast<int>(ceil_div(group, parts));
  *nodes = M / *heads;
}

template <typename T, int DP>
int launch_typed(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  static std::once_flag once;
  static cudaError_t attr = cudaSuccess;
  std::call_once(once, [] {
    attr = cudaFuncSetAttribute(tree_wide_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DP>::SMEM);
  });
  if (attr != cudaSuccess) return cuda_error(attr, "wide tree attention attributes");
  int tile_heads, tile_nodes;
  tile_of(a, &tile_heads, &tile_nodes);
  CUtensorMap q, k, v;
  const int box_rows = box_rows_of(a);
  const int rc = encode_heads(&q, a.dtype, a.q, a.rows, a.heads, a.dim, a.sq_t, a.sq_h, tile_heads, tile_nodes);
  if (rc != KF_OK) return rc;
  if (!encode_pages(&k, a, a.k, a.sk_p, a.sk_h, a.sk_t, box_rows, 64) ||
      !encode_pages(&v, a, a.v, a.sv_p, a.sv_h, a.sv_t, box_rows, 64))
    return set_error(KF_ERR_UNALIGNED, "wide tree attention: no tensor map describes the cache");
  const int vector_out = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.so_t % 8 == 0 && a.so_h % 8 == 0;
  tree_wide_kernel<T, DP><<<dev.sm_count, THREADS, Shape<DP>::SMEM, stream>>>(q, k, v, a, divisor(a.block_size), box_rows,
                                                                             vector_out, dev.status);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(wide tree attention)");
}

bool fits(int64_t s, int64_t n) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); }

}  // namespace

bool attention_tree_wide_supported(const AttnArgs& a) {
  // the softmax takes its maximum over q k, so the scale has to keep its order
  return a.scale_log2 > 0.0f && box_rows_of(a) >= 8 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(a.k) % 16 == 0 && reinterpret_cast<uintptr_t>(a.v) % 16 == 0 &&
         fits(a.sq_t, a.rows) && fits(a.sq_h, a.heads) && fits(a.sk_t, a.block_size) && fits(a.sk_h, a.kv_heads) &&
         fits(a.sk_p, a.pages) && fits(a.sv_t, a.block_size) && fits(a.sv_h, a.kv_heads) && fits(a.sv_p, a.pages);
}

int64_t attention_tree_wide_workspace_bytes(const AttnArgs& a, const DeviceInfo& dev) {
  return TREE_COUNTER_BYTES + 4ll * 2 * dev.sm_count * M * ((a.dim <= 64 ? 64 : 128) + 2);
}

int launch_attention_tree_wide(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  if (a.dtype == KF_FP16)
    return a.dim <= 64 ? launch_typed<__half, 64>(a, dev, stream) : launch_typed<__half, 128>(a, dev, stream);
  return a.dim <= 64 ? launch_typed<__nv_bfloat16, 64>(a, dev, stream) : launch_typed<__nv_bfloat16, 128>(a, dev, stream);
}

}  // namespace kf
