// Prompt attention on the 5th-generation tensor cores: causal or not, grouped
// heads, requests of any lengths packed without padding.
//
// One CTA stays on each SM and takes items in turn: 256 rows of one request and
// head, as two tiles of 128. It walks an item's keys 128 at a time, with the
// softmax's running maximum and sum:
//
//   S = Q K^T                      tcgen05, fp32 in TMEM, 128 x 128 per tile
//   m' = max(m, max S),  P = 2^(c S - c m'),  l = l 2^(c m - c m') + sum P
//   O = O 2^(c m - c m') + P V     tcgen05, P read from TMEM        (c = scale log2 e)
//
//   warps 0-3, 4-7   softmax of tile 0 and 1, a thread per row: S from TMEM into
//                    registers, P (16 bit) back over the same columns.
//   warp 8           TMA: Q once, then K and V blocks through a ring.
//   warp 9           issues the MMAs. While one tile's warps compute their
//                    weights the tensor cores work for the other tile; the second
//                    product starts when half of a block's weights are there.
//   warp 10          zeroes what the last V block holds of the next request.
//   warp 11          finds the CTA's next item while this one is computed, so that
//                    its loads and first products start behind this one's results.
//
// m is raised, and O (in TMEM) rescaled, only when a row's maximum grew by more
// than 2^8: until then the weights are at most 256 (bf16: one, see WEIGHT_SHIFT), which 16
// bits and the fp32 sums hold as well. P is rounded to the operands' type for the second product; l sums
// the unrounded weights.
//
// Keys of the next request in a request's last block have weight zero, and
// their V rows are zeroed in shared memory (0 x inf is NaN); a row that still
// comes out non-finite, with later tokens of its own in the block that hold
// infinities, is computed again from the keys that it sees.
//
// The tensor cores bound it from below and the softmax's chain (maximum,
// exponentials, sums, conversions, ~1800 cycles for 128 x 128 scores a warp group)
// from above. One prompt of 8192 tokens, 32 heads to 8 of 128 elements, bf16: 449 us,
// 1.22 PFLOP/s in a burst (75% of a plain product's rate), 511 to 525 us, 1.05 to 1.08
// PFLOP/s, under the power cap (77%). Nine ragged prompts (53 GFLOP) 104 us, 0.51 PFLOP/s:
// an SM has five items of two to eleven blocks, whose beginnings and ends nothing hides. 11.1 us for four prompts of up to 160.
#include <cuda.h>

#include <mutex>

#include "attention.cuh"
#include "attention_softmax.cuh"

namespace kf {
namespace {

constexpr int BLK = 128;       // rows of a tile, keys of a block
constexpr int PAIR = 2 * BLK;  // rows of a CTA
constexpr int SOFTMAX_WARPS = 8;
constexpr int TMA_WARP = 8, MMA_WARP = 9, CLEAN_WARP = 10, PLAN_WARP = 11;
// Three warpgroups; the last (loads, products) hands registers to the softmax:
// 3 x 168 a thread become 2 x 208 and 88.
constexpr int THREADS = 3 * 128;
constexpr int LAUNCH_REGISTERS = 168;
constexpr uint32_t TMEM_COLS = 512;  // S0 | S1 | O0 | O1, 128 each
constexpr uint64_t DRAIN_NS = 100000000ull;

template <int DH>
struct Shape {
  static constexpr int HALVES = DH / 64;            // 128-byte swizzle atoms of a row
  static constexpr int TILE = BLK * DH * 2;         // bytes of a Q, K or V tile
  static constexpr int STAGES = DH == 128 ? 5 : 8;  // K and V tiles in flight
  static constexpr int SMEM = 1024 + 2 * TILE + STAGES * TILE + 320;
};

struct Item {
  int row0;       // first row of q
  int rows;       // of the request from row0 on, at most PAIR; 0: there is no item
  int node0;      // row0's place in its request
  int first_key;  // first row of k and v
  int keys;
  int shift;      // keys - rows of the request: row i sees i + 1 + shift keys
  int head;
  int blocks[2];  // key blocks of each tile: those that its last row sees some of
};

// The tile pair with number `g`, counted through the requests, the last rows of
// a request (which see the most keys) first. Called by a whole warp.
__device__ __forceinline__ bool find_item(const AttnArgs& p, int g, int lane, Item* out) {
  for (int r0 = 0; r0 <= p.seqs; r0 += 32) {
    const int r = r0 + lane;
    int begin = 0, end = 0;
    if (r <= p.seqs) request_rows(p, r, &begin, &end);
    const int tiles = (end - begin + PAIR - 1) / PAIR;
    int upto = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const int total = __shfl_sync(0xffffffffu, upto, 31);
    if (g < total) {
      if (upto > g && upto - tiles <= g) {
        const int tile = upto - 1 - g;
        long long first, length;
        request_keys(p, r, end - begin, &first, &length);
        out->node0 = tile * PAIR;
        out->row0 = begin + out->node0;
        out->rows = min(PAIR, end - out->row0);
        out->first_key = static_cast<int>(first);
        out->keys = static_cast<int>(length);
        out->shift = static_cast<int>(length) - (end - begin);
      }
      return true;
    }
    g -= total;
  }
  return false;
}

// The same items, the ones with most key blocks first, where a lane can keep a
// request (the rows behind the last one counted as one more).
constexpr int ORDERED = 32;
struct Order {
  int begin, rows, keys, first;
  int level;  // the key blocks of the item found last

  __device__ __forceinline__ void load(const AttnArgs& p, int lane) {
    int end = 0;
    long long from = 0, length = 0;
    begin = 0;
    if (lane <= p.seqs) {
      request_rows(p, lane, &begin, &end);
      request_keys(p, lane, end - begin, &from, &length);
    }
    rows = end - begin;
    keys = static_cast<int>(length);
    first = static_cast<int>(from);
    level = __reduce_max_sync(0xffffffffu, keys) / BLK + 1;
  }
  // Tile pairs of this lane's request with `blocks` key blocks or more: its last ones.
  __device__ __forceinline__ int tiles(int causal, int blocks) const {
    const int all = (rows + PAIR - 1) / PAIR, before = (blocks - 1) * BLK;  // they see a key behind `before`
    if (all == 0 || blocks <= 0) return all;
    if (!causal) return keys > before ? all : 0;
    const int row = before - (keys - rows);  // a tile pair of them ends behind this row
    if (rows <= row) return 0;
    return all - (row < 0 ? 0 : min(row / PAIR, all - 1));
  }
  __device__ __forceinline__ int count(int causal, int blocks) const {
    return __reduce_add_sync(0xffffffffu, tiles(causal, blocks));
  }
  // Tile pair `g` in that order; called with g that do not fall.
  __device__ __forceinline__ bool find(const AttnArgs& p, int g, int lane, Item* out) {
    if (g >= count(p.causal, 0)) return false;
    // the largest number of blocks that more than g tile pairs reach
    int lo = 0;
    while (lo < level) {
      const int mid = (lo + level + 1) >> 1;
      if (count(p.causal, mid) > g) lo = mid; else level = mid - 1;
    }
    const int above = tiles(p.causal, level + 1), here = tiles(p.causal, level) - above;
    g -= __reduce_add_sync(0xffffffffu, above);
    int upto = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    if (g < upto && g >= upto - here) {
      const int all = (rows + PAIR - 1) / PAIR;
      out->node0 = (all - 1 - above - (g - (upto - here))) * PAIR;
      out->row0 = begin + out->node0;
      out->rows = min(PAIR, rows - out->node0);
      out->first_key = first;
      out->keys = keys;
      out->shift = keys - rows;
    }
    return true;
  }
};

// Keys that row i (of the item) sees.
__device__ __forceinline__ int visible(const AttnArgs& p, const Item& it, int i) {
  if (!p.causal) return it.keys;
  return min(it.keys, max(0, it.node0 + i + 1 + it.shift));
}

template <typename T, int DH>
__device__ __noinline__ long long last_unseen(const AttnArgs& p, int t, int head, long long from, long long to, int lane) {
  return last_unseen_nonfinite<T, DH / 32>(p, t, head, from, to, lane);
}
template <typename T, int DH>
__device__ __noinline__ void redo_row(const AttnArgs& p, int t, int head, int lane) {
  float acc[DH / 32], m, l;
  attend_row<T, DH / 32>(p, t, head, lane, acc, &m, &l);
  write_row<T, DH / 32>(p, t, head, lane, acc, m, l);
}

template <typename T, int DH>
__global__ void __launch_bounds__(THREADS, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ AttnArgs p, int vector_out, int* status) {
  using S = Shape<DH>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* q_tiles = smem;
  uint8_t* ring = smem + 2 * S::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + STAGES * S::TILE);
  // bars: item[2] | item_free[2] | q[2] | q_free[2] | full[STAGES] | empty[STAGES] | s_full[2] | p_half[2] |
  //       p_full[2] | o_full[2] | dirty | clean
  __shared__ Item items[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t item_bar = smem_u32(bars), item_free = item_bar + 16, q_bar = item_free + 16, q_free = q_bar + 16,
                 full = q_free + 16, empty = full + 8 * STAGES, s_full = empty + 8 * STAGES, p_half = s_full + 16,
                 p_full = p_half + 16, o_full = p_full + 16, dirty = o_full + 16, clean = dirty + 8;

  if (warp == TMA_WARP && lane == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(item_bar + 8 * i, 1);
      mbar_init(item_free + 8 * i, SOFTMAX_WARPS + 3);  // softmax, loads, products, cleaning
      mbar_init(q_bar + 8 * i, 1);
      mbar_init(q_free + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_half + 8 * i, SOFTMAX_WARPS / 2);
      mbar_init(p_full + 8 * i, SOFTMAX_WARPS / 2);
      mbar_init(o_full + 8 * i, 1);
    }
    for (int i = 0; i < 2 * STAGES; ++i) mbar_init(full + 8 * i, 1);
    mbar_init(dirty, 1);
    mbar_init(clean, 1);
    abort_word = 0;
    mbar_init_fence();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  } else if (warp == MMA_WARP) {
    tmem_alloc(smem_u32(&tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // The n-th item of this CTA, for each role in turn; rows 0 when there are no
  // more, or a wait gave up. All roles go through the same items in order, and
  // every barrier below is waited for phase by phase.
  auto next_item = [&](int n, int site) {
    Item it;
    const bool ok = __all_sync(0xffffffffu, attn_wait(item_bar + 8 * (n & 1), (n >> 1) & 1, abort_flag, status, site));
    it = items[n & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(item_free + 8 * (n & 1));
    if (!ok) it.rows = 0;
    return it;
  };

  if (warp >= SOFTMAX_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == PLAN_WARP) {
      // Items: tile pairs x heads, dealt out to the CTAs in turn, forwards and
      // backwards, so that each gets large and small ones alike.
      const int heads = static_cast<int>(p.heads), ctas = static_cast<int>(gridDim.x), me = static_cast<int>(blockIdx.x);
      // In the order of their lengths where a CTA has a few items. 9 ragged prompts, 32 heads (6 items at
      // most on average): 121 us, as they come 135; 7 prompts, 8 heads (2): 70 and 79; 27 shorter ones,
      // 32 heads (12): 103 and 95.
      const long long most = (p.rows / PAIR + p.seqs + 1) * p.heads;
      const bool ordered = p.seqs < ORDERED && most > ctas && most <= 8ll * ctas;
      Order order;
      if (ordered) order.load(p, lane);
      for (int n = 0;; ++n) {
        const long long i = static_cast<long long>(n) * ctas + (n & 1 ? ctas - 1 - me : me);
        const bool ok = __all_sync(
            0xffffffffu, attn_wait(item_free + 8 * (n & 1), ((n >> 1) & 1) ^ 1, abort_flag, status, SITE_ATTN_LOAD));
        Item* it = &items[n & 1];
        const int g = static_cast<int>(i / heads);
        const bool found = ok && (ordered ? order.find(p, g, lane, it) : find_item(p, g, lane, it));
        __syncwarp();
        if (lane == 0) {
          if (found) {
            it->head = static_cast<int>(i % heads);
            for (int t = 0; t < 2; ++t)
              it->blocks[t] =
                  it->rows > t * BLK ? (visible(p, *it, min(it->rows, (t + 1) * BLK) - 1) + BLK - 1) / BLK : 0;
          } else {
            it->rows = 0;
          }
          mbar_arrive(item_bar + 8 * (n & 1));
        }
        __syncwarp();
        if (!found) break;
      }
    } else if (warp == TMA_WARP) {
      bool ok = true;
      int issued = 0, loaded = 0;  // K and V tiles, and items with any
      auto load = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int h, int row) {
        mbar_arrive_expect_tx(bar, S::TILE);
#pragma unroll
        for (int x = 0; x < S::HALVES; ++x) tma_load_3d(dst + x * BLK * 128, map, bar, 64 * x, h, row);
      };
      for (int n = 0;; ++n) {
        const Item it = next_item(n, SITE_ATTN_LOAD);
        if (it.rows == 0) break;
        const int most = max(it.blocks[0], it.blocks[1]);
        if (most == 0) continue;
        if (lane == 0) {
          const int kv_head = it.head / static_cast<int>(p.heads / p.kv_heads);
          auto next = [&](const CUtensorMap* map, int block) {
            const int slot = issued % STAGES;
            if (!attn_wait(empty + 8 * slot, ((issued / STAGES) & 1) ^ 1, abort_flag, status, SITE_ATTN_LOAD)) return false;
            load(smem_u32(ring + slot * S::TILE), map, full + 8 * slot, kv_head, it.first_key + block * BLK);
            ++issued;
            return true;
          };
          auto query = [&](int t) {
            if (!attn_wait(q_free + 8 * t, (loaded & 1) ^ 1, abort_flag, status, SITE_ATTN_LOAD)) return false;
            load(smem_u32(q_tiles + t * S::TILE), &tm_q, q_bar + 8 * t, it.head, it.row0 + t * BLK);
            return true;
          };
          ok = query(0) && next(&tm_k, 0) && query(1);
          for (int j = 0; ok && j < most; ++j) {
            ok = next(&tm_v, j);
            if (ok && j + 1 < most) ok = next(&tm_k, j + 1);
          }
        }
        ++loaded;
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      if (!ok && lane == 0) {  // let the copies in flight land before the shared memory goes away
        for (int t = 0; t < 2; ++t) mbar_wait(q_bar + 8 * t, (loaded - 1) & 1, nullptr, status, SITE_DRAIN, DRAIN_NS);
        for (int s = 0; s < STAGES && s < issued; ++s)
          mbar_wait(full + 8 * s, ((issued - 1 - s) / STAGES) & 1, nullptr, status, SITE_DRAIN, DRAIN_NS);
      } else if (lane == 0) {  // the products' last arrivals here come behind those that the results wait for
        for (int s = 0; s < STAGES && s < issued; ++s)
          attn_wait(empty + 8 * ((issued - 1 - s) % STAGES), ((issued - 1 - s) / STAGES) & 1, abort_flag, status,
                    SITE_ATTN_LOAD);
        for (int t = 0; t < 2 && loaded > 0; ++t)
          attn_wait(q_free + 8 * t, (loaded - 1) & 1, abort_flag, status, SITE_ATTN_LOAD);
      }
    } else if (warp == CLEAN_WARP) {
      // The last block of a request: its V rows past the request's keys, when the
      // warp of the products has seen them land
      int tiles = 0, cleaned = 0;  // K and V tiles before the item's
      for (int n = 0;; ++n) {
        const Item it = next_item(n, SITE_ATTN_LOAD);
        if (it.rows == 0) break;
        const int most = max(it.blocks[0], it.blocks[1]);
        if (most == 0) continue;
        tiles += 2 * most;
        const int held = it.keys - (most - 1) * BLK, slot = (tiles - 1) % STAGES;
        if (held >= BLK) continue;
        if (!__all_sync(0xffffffffu, attn_wait(dirty, cleaned & 1, abort_flag, status, SITE_ATTN_LOAD))) break;
        for (int i = lane; i < (BLK - held) * S::HALVES * 8; i += 32) {
          const int h = i / ((BLK - held) * 8), rest = i - h * (BLK - held) * 8;
          *reinterpret_cast<uint4*>(ring + slot * S::TILE + h * BLK * 128 + held * 128 + rest * 16) =
              make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(clean);
        ++cleaned;
      }
    } else {
      // MMA_WARP. The warp runs together on uniform values and one elected lane
      // issues: a few instructions a product, where a branch for one lane takes
      // about 20 and the tensor cores run dry behind them. (A warp for each tile
      // measured slower: two tiles' products in turn finish later than one tile's,
      // then the other's.)
      const uint32_t lead = elect_lane();
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t q_at = __shfl_sync(0xffffffffu, smem_u32(q_tiles), 0), ring_at = __shfl_sync(0xffffffffu, smem_u32(ring), 0);
      constexpr uint32_t fmt = DType<T>::code == KF_BF16 ? 1u : 0u;
      constexpr uint32_t idesc_s = instr_desc_f16(fmt, 0, 0, BLK, BLK), idesc_o = instr_desc_f16(fmt, 0, 1, BLK, DH);
      const uint64_t q_desc = smem_desc_sw128(q_at, 16, 1024);
      const uint64_t k_desc = smem_desc_sw128(ring_at, 16, 1024), v_desc = smem_desc_sw128(ring_at, BLK * 128, 1024);
      int slot = 0, phase = 0;  // of the ring's next tile
      int done[2] = {0, 0};     // blocks of each tile, over all items
      int loaded = 0, cleaned = 0;
      bool ok = true;
      auto wait = [&](uint32_t bar, int parity) {
        if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity)))
          ok = __all_sync(0xffffffffu, attn_wait(bar, parity, abort_flag, status, SITE_ATTN_MMA)) && ok;
        tc_fence_after();
      };
      auto wait_tile = [&]() {
        const int at = slot;
        wait(full + 8 * at, phase);
        if (++slot == STAGES) {
          slot = 0;
          phase ^= 1;
        }
        return at;
      };
      auto scores = [&](int t, int at, bool last) {  // S_t = Q_t K^T
        const uint64_t a = q_desc + static_cast<uint64_t>(t * S::TILE / 16), b = k_desc + static_cast<uint64_t>(at * (S::TILE / 16));
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) {
          const uint64_t step = static_cast<uint64_t>((k / 4) * (BLK * 128 / 16) + (k % 4) * 2);
          tc_mma_f16_by(lead, tm + t * BLK, a + step, b + step, idesc_s, k > 0);
        }
        tc_commit_by(lead, s_full + 8 * t);  // with it all products before are done, O_t's too
        if (last) tc_commit_by(lead, q_free + 8 * t);
      };
      auto products = [&](int t, int at, bool accumulate, int k0, int k1) {  // O_t += P_t V
        const uint64_t b = v_desc + static_cast<uint64_t>(at * (S::TILE / 16));
#pragma unroll
        for (int k = k0; k < k1; ++k)
          tc_mma_f16_ta_by(lead, tm + 2 * BLK + t * BLK, tm + t * BLK + 8 * k, b + static_cast<uint64_t>(k * 128), idesc_o,
                           accumulate || k > 0);
      };
      for (int n = 0; ok; ++n) {
        const Item it = next_item(n, SITE_ATTN_MMA);
        if (__shfl_sync(0xffffffffu, it.rows, 0) == 0) break;
        const int count[2] = {__shfl_sync(0xffffffffu, it.blocks[0], 0), __shfl_sync(0xffffffffu, it.blocks[1], 0)};
        const int all = max(count[0], count[1]);
        const bool partial = __shfl_sync(0xffffffffu, it.keys, 0) - (all - 1) * BLK < BLK;
        if (all == 0) continue;
        wait(q_bar, loaded & 1);
        int k_at = wait_tile();
        if (count[0] > 0) {
          if (ok) scores(0, k_at, count[0] == 1);
        } else {
          tc_commit_by(lead, q_free);
        }
        wait(q_bar + 8, loaded & 1);
        if (count[1] > 0) {
          if (ok) scores(1, k_at, count[1] == 1);
        } else {
          tc_commit_by(lead, q_free + 8);
        }
        ++loaded;
        tc_commit_by(lead, empty + 8 * k_at);
        for (int j = 0; ok && j < all; ++j) {
          const int v_at = wait_tile();
          if (j + 1 < all) {
            k_at = wait_tile();
          } else if (partial) {
            if (lead) mbar_arrive(dirty);
            wait(clean, cleaned & 1);
            ++cleaned;
          }
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >= count[t]) continue;
            const int parity = (done[t] + j) & 1;
            wait(p_half + 8 * t, parity);
            if (ok) products(t, v_at, j > 0, 0, 4);
            wait(p_full + 8 * t, parity);
            if (ok) products(t, v_at, true, 4, 8);
            if (j + 1 < count[t]) {
              if (ok) scores(t, k_at, j + 2 == count[t]);
            } else {
              tc_commit_by(lead, o_full + 8 * t);
            }
          }
          tc_commit_by(lead, empty + 8 * v_at);
          if (j + 1 < all) tc_commit_by(lead, empty + 8 * k_at);
        }
        done[0] += count[0];
        done[1] += count[1];
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;  // of the tile
    const int i = t * BLK + row;             // of the item
    const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_addr = lanes + t * BLK, o_addr = lanes + 2 * BLK + t * BLK;
    const float c = p.scale_log2;
    int done = 0, results = 0;  // blocks of this tile, and items with any, before this item
    bool ok = true;
    for (int n = 0; ok; ++n) {
      const Item it = next_item(n, SITE_ATTN_SOFTMAX);
      if (it.rows == 0) break;
      const int blocks = t == 0 ? it.blocks[0] : it.blocks[1];
      const bool valid = i < it.rows;
      const int limit = valid ? visible(p, it, i) : 0;
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < blocks; ++j) {
        ok = attn_wait(s_full + 8 * t, (done + j) & 1, abort_flag, status, SITE_ATTN_SOFTMAX);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        float s[BLK];
#pragma unroll
        for (int x = 0; x < BLK; x += 32) tmem_ld_32(s_addr + x, reinterpret_cast<uint32_t*>(s + x));
        tmem_ld_wait();
        const int left = limit - j * BLK;
        if (left < BLK) {
#pragma unroll
          for (int x = 0; x < BLK; ++x)
            if (x >= left) s[x] = -INFINITY;
        }
        __syncwarp();
        const float m_new = row_max(s, m);
        if (j == 0) {
          m = m_new;
        } else if (__any_sync(0xffffffffu, (m_new - m) * c > RAISE_LOG2)) {
          // S of this block came with the end of all products before it: O rests
          const float fix = m_new > m ? ex2_ftz((m - m_new) * c) : 1.0f;
          l *= fix;
          m = m_new;
#pragma unroll 1
          for (int x = 0; x < DH; x += 32) {
            uint32_t o[32];
            tmem_ld_32(o_addr + x, o);
            tmem_ld_wait();
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * fix);
            tmem_st_32(o_addr + x, o);
          }
        }
        const float cm = m == -INFINITY ? 0.0f : fmaf(m, c, WEIGHT_SHIFT<T>);
        // NaN among the row's scores, or infinity: the row is NaN (`m` need not have been raised, and
        // the polynomial takes NaN for zero)
        if (!(m_new * c < INFINITY)) l = NAN;
        l += row_weights<T, true>(s, c, cm, s_addr, p_half + 8 * t, p_full + 8 * t, lane);
      }
      done += blocks;
      if (ok && blocks > 0) {
        ok = attn_wait(o_full + 8 * t, results & 1, abort_flag, status, SITE_ATTN_SOFTMAX);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        ++results;
      }
      if (!ok || it.rows <= t * BLK) continue;
      const int q_row = it.row0 + i;
      T* out = static_cast<T*>(p.out) + static_cast<long long>(q_row) * p.so_t + it.head * p.so_h;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      float bad = 0.0f;  // NaN if anything in the row is not finite
#pragma unroll 1
      for (int x = 0; x < DH; x += 32) {
        uint32_t o[32];
        if (blocks > 0) {
          tmem_ld_32(o_addr + x, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int y = 0; y < 32; ++y) o[y] = 0u;
        }
        uint32_t w[16];
#pragma unroll
        for (int y = 0; y < 32; y += 2) {
          // a row that sees nothing may hold anything in O: its result is zero
          const float a = l == 0.0f ? 0.0f : __uint_as_float(o[y]) * inv;
          const float b = l == 0.0f ? 0.0f : __uint_as_float(o[y + 1]) * inv;
          bad = fmaf(a, 0.0f, fmaf(b, 0.0f, bad));
          w[y / 2] = pack_pair<T>(a, b);
        }
        if (valid) {
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            if (x + 8 * y >= p.dim) break;
            if (vector_out) {
              *reinterpret_cast<uint4*>(out + x + 8 * y) = make_uint4(w[4 * y], w[4 * y + 1], w[4 * y + 2], w[4 * y + 3]);
            } else {
              const T* e = reinterpret_cast<const T*>(w + 4 * y);
#pragma unroll
              for (int z = 0; z < 8; ++z) out[x + 8 * y + z] = e[z];
            }
          }
        }
        __syncwarp();
      }
      if (p.lse != nullptr && valid)
        p.lse[static_cast<long long>(q_row) * p.heads + it.head] =
            l == 0.0f ? -INFINITY : fmaf(m, c, WEIGHT_SHIFT<T>) * 0.69314718055994530942f + logf(l);
      uint32_t again = __ballot_sync(0xffffffffu, valid && suspect(bad == 0.0f, l));
      if (again != 0) {
        redo_begin(abort_flag, lane);
        // the first of them sees the fewest keys, the others more of the same
        const int src = __ffs(again) - 1;
        const long long last = last_unseen<T, DH>(p, __shfl_sync(0xffffffffu, q_row, src), it.head,
                                                  __shfl_sync(0xffffffffu, limit, src), blocks * BLK, lane);
        again = __ballot_sync(0xffffffffu, ((again >> lane) & 1u) && limit <= last);
        while (again != 0) {
          redo_row<T, DH>(p, __shfl_sync(0xffffffffu, q_row, __ffs(again) - 1), it.head, lane);
          again &= again - 1;
        }
        redo_end(abort_flag, lane);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == MMA_WARP) tmem_dealloc(tmem, TMEM_COLS);
}

bool on_grid(const void* ptr, int64_t s_row, int64_t rows, int64_t s_head, int64_t heads) {
  const auto fits = [](int64_t s, int64_t n) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
  return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && fits(s_row, rows) && fits(s_head, heads);
}

template <typename T, int DH>
int launch_typed(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  CUtensorMap q, k, v;
  int rc = encode_heads(&q, a.dtype, a.q, a.rows, a.heads, a.dim, a.sq_t, a.sq_h, 1, BLK);
  if (rc == KF_OK) rc = encode_heads(&k, a.dtype, a.k, a.keys, a.kv_heads, a.dim, a.sk_t, a.sk_h, 1, BLK);
  if (rc == KF_OK) rc = encode_heads(&v, a.dtype, a.v, a.keys, a.kv_heads, a.dim, a.sv_t, a.sv_h, 1, BLK);
  if (rc != KF_OK) return rc;
  static std::once_flag once;
  static cudaError_t attr = cudaSuccess;
  static int registers = 0;
  std::call_once(once, [] {
    attr = cudaFuncSetAttribute(prefill_kernel<T, DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<DH>::SMEM);
    cudaFuncAttributes f{};
    if (attr == cudaSuccess) attr = cudaFuncGetAttributes(&f, prefill_kernel<T, DH>);
    registers = f.numRegs;
  });
  if (attr != cudaSuccess) return cuda_error(attr, "prefill attributes");
  if (registers < LAUNCH_REGISTERS)  // the warpgroups' shares must not exceed what the block is launched with
    return set_error(KF_ERR_UNSUPPORTED, "prompt attention: built with too few registers to split");
  const int64_t most = (a.rows / PAIR + a.seqs + 1) * a.heads;  // items
  const int64_t blocks = most < dev.sm_count ? most : dev.sm_count;
  const int vector_out = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.so_t % 8 == 0 && a.so_h % 8 == 0;
  prefill_kernel<T, DH><<<static_cast<unsigned>(blocks), THREADS, Shape<DH>::SMEM, stream>>>(q, k, v, a, vector_out,
                                                                                            dev.status);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(prompt attention)");
}

}  // namespace

bool attention_prefill_supported(const AttnArgs& a) {
  return (a.dtype == KF_FP16 || a.dtype == KF_BF16) && a.dim <= 128 && a.dim % 8 == 0 && a.keys > 0 &&
         a.scale_log2 > 0.0f && on_grid(a.q, a.sq_t, a.rows, a.sq_h, a.heads) &&
         on_grid(a.k, a.sk_t, a.keys, a.sk_h, a.kv_heads) && on_grid(a.v, a.sv_t, a.keys, a.sv_h, a.kv_heads) &&
         (a.rows / PAIR + a.seqs + 1) * a.heads <= 0x7fffffffll;
}

int launch_attention_prefill(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  if (a.dtype == KF_FP16)
    return a.dim <= 64 ? launch_typed<__half, 64>(a, dev, stream) : launch_typed<__half, 128>(a, dev, stream);
  return a.dim <= 64 ? launch_typed<__nv_bfloat16, 64>(a, dev, stream) : launch_typed<__nv_bfloat16, 128>(a, dev, stream);
}

}  // namespace kf
