// Attention of new tokens (one, a chain or a tree of drafts per request) over a
// paged cache, fp16/bf16, heads of up to 128 elements.
//
// All query rows of a request that share a key head -- its nodes times the
// heads of the group -- form tiles of 16 rows against the request's keys, so the
// cache is read once for all of them. The work of all requests, key heads and
// tiles is one list of key blocks, cut into equal runs, one per CTA
// (attention_paged.cuh): a long cache is spread over the GPU and short ones share
// a CTA, whatever the lengths, which only the device knows. An item cut between
// CTAs leaves partial sums (m, l, O) in the workspace, and whichever CTA arrives
// last adds them in the order of the keys, so results do not depend on timing and
// nobody waits for another CTA.
//
// In a CTA each of four warps holds the 16 rows and takes 16 keys of each block
// of 64, with its own running maximum and sum:
//
//   s = scale log2(e) q k^T,  m' = max(m, max s),  p = 2^(s - m'),
//   l = l 2^(m - m') + sum p,  O = O 2^(m - m') + p v       (mma.sync, fp32 sums)
//
// One more warp loads: it reads the block table ahead, brings each item's queries
// while the one before is computed, and fills a ring of K and V blocks, with one TMA box per run of keys that is whole in any page (gcd of
// page and block, 8 keys at least), or where pages are not multiples of 8 keys
// with 16-byte cp.async. Pages a table does not name are read as zeros (a box
// past the last page); V rows past the request's end are zeroed in shared memory
// (0 x NaN is NaN); weights of keys that a row does not see are zero. A row that
// comes out non-finite (a node it does not see holds infinities) is computed again from
// the keys that it sees.
//
// With one new token and G heads to a key head, G of the 16 rows are real: the
// products are free beside the cache's bytes, which bound the call. 64 requests of up
// to 4096 keys, 32 heads to 8 of 128 elements, bf16: 98 us, 540 MB at 5.5 TB/s (84%
// of a copy's rate); one of 131072 keys 98 us, 537 MB at 5.5 TB/s; one of 100 keys
// 9.0 us. What is left: the chain of products, maxima and exponentials of a block is
// longer than its bytes take to come, and each item's joining is in nobody's shadow.
#include <cuda.h>

#include <initializer_list>
#include <mutex>
#include <numeric>
#include <string>

#include "attention_paged.cuh"

namespace kf {
namespace {

constexpr int M = 16;         // rows of a tile
constexpr int KEYS = 64;      // of a block
constexpr int WARPS = 4;      // of products
constexpr int KW = KEYS / WARPS;
constexpr int LOAD_WARP = WARPS, FINISH_WARP = WARPS + 1;
constexpr int THREADS = 32 * (WARPS + 2);
constexpr int MIN_RUN = 4;  // positions of a run: fewer blocks cost more to join than to read (8: 14.5 us for 12.2, one request of 100 keys, calls back to back)
// Blocks that an item's queries and results are worth. 64 requests of up to 4096 keys: 98.5 us
// (104.6 with none, 97.4 with 2, 99.8 with 6); 128 of up to 1000: 57.9 (76.5, 59.5, 61.7); one of
// 131072: 98 to 100 with any.
constexpr int ITEM_COST = 3;
constexpr uint64_t DRAIN_NS = 100000000ull;

template <int DP_, int STAGES_>
struct Shape {
  static constexpr int DP = DP_, STAGES = STAGES_;
  static constexpr int HALVES = DP == 128 ? 2 : 1;  // boxes of at most 128 bytes a row
  static constexpr int TILE = KEYS * DP * 2;        // bytes of a K or V block in the ring
  static constexpr int Q_TILE = M * DP * 2;
  static constexpr int PITCH = DP + 8;              // floats of a row of the joined result
  // ring | queries | joined result | maxima, sums | barriers | present
  static constexpr int SMEM =
      1024 + STAGES * 2 * TILE + Q_TILE + M * PITCH * 4 + 2 * M * WARPS * 4 + 8 * (2 * STAGES + 3) + 8 * STAGES;
};

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool present) {
  // nothing is read where the row is absent: 16 bytes of zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(present ? 16 : 0) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// Where ldmatrix finds 16 x 16 elements of a tile in the swizzle of chunk_at: this
// lane's row and half of a pair of chunks give `first` (of a tile on a 1 KB
// boundary), and pair k of the row is one XOR and a constant away.
template <int DP, int ROWS>
__device__ __forceinline__ uint32_t first_pair(int row, int half) {
  if constexpr (DP >= 64) {
    return static_cast<uint32_t>(row * 128 + ((half ^ (row & 7)) << 4));
  } else {
    return static_cast<uint32_t>(row * 64 + ((half ^ ((row >> 1) & 3)) << 4));
  }
}
template <int ROWS>
__device__ __forceinline__ uint32_t pair_at(uint32_t first, int k) {
  return (first ^ static_cast<uint32_t>((k & 3) << 5)) + static_cast<uint32_t>((k >> 2) * (ROWS * 128));
}

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile, as TMA's swizzles
// place it: rows of 128 bytes (64 elements, a second half behind the first) or of
// 64 bytes, chunks XORed so that eight rows of one column meet eight bank groups.
template <int DP, int ROWS>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
  if constexpr (DP >= 64) {
    return static_cast<uint32_t>((chunk >> 3) * (ROWS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
  } else {
    return static_cast<uint32_t>(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
  }
}

template <typename T, typename S, bool BULK>
__global__ void __launch_bounds__(THREADS, 2)
    tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ AttnArgs p, const Divisor by_page, int box_rows, int vector_out, int* status) {
  constexpr int DP = S::DP, STAGES = S::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* q_tile = smem + STAGES * 2 * S::TILE;
  float* joined = reinterpret_cast<float*>(q_tile + S::Q_TILE);
  float* part_m = joined + M * S::PITCH;
  float* part_l = part_m + M * WARPS;
  uint64_t* bars = reinterpret_cast<uint64_t*>(part_l + M * WARPS);
  volatile uint32_t* present = reinterpret_cast<volatile uint32_t*>(bars + 2 * STAGES + 3);  // a bit per key of each stage
  static_assert(S::TILE % 1024 == 0 && S::Q_TILE % 1024 == 0 && S::PITCH % 4 == 0 && Partial<M, DP>::FLOATS % 4 == 0,
                "vectors of 16 bytes");
  __shared__ int last_one, abort_word;
  __shared__ Cursor first_item;
  __shared__ int first_is_last;
  volatile int* abort_flag = &abort_word;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring = smem_u32(smem), full = smem_u32(bars), empty = full + 8 * STAGES, q_full = empty + 8 * STAGES,
                 q_empty = q_full + 8, finished = q_empty + 8;

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + 8 * s, BULK ? 1 : 33);
      mbar_init(empty + 8 * s, WARPS);
    }
    mbar_init(q_full, 32);
    mbar_init(q_empty, WARPS);
    mbar_init(finished, 1);
    abort_word = 0;
    mbar_init_fence();
  }
  if (p.dim < DP) {  // columns past the head stay zero where no box fills them
    const int from = BULK ? STAGES * 2 * S::TILE / 16 : 0, to = (STAGES * 2 * S::TILE + S::Q_TILE) / 16;
    for (int i = from + tid; i < to; i += THREADS) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  const Walk<KEYS, ITEM_COST> walk(p, M);
  Cursor at;
  const Run run = walk.template find<THREADS>(p, MIN_RUN, at);
  if (run.count == 0) return;
  // The run begins inside an item and goes on behind it: the item's arrival (a
  // fence and an atomic, a few microseconds when the memory is busy) is left to a
  // warp of its own, and its joining, if it falls to this CTA, to the end.
  const bool defer = at.blk > 0 && at.left > at.blocks + ITEM_COST - at.blk;
  const int first_owner = static_cast<int>((run.first - at.blk) / run.per);
  const int first_last = static_cast<int>((run.first - at.blk + at.blocks - 1) / run.per);

  if (warp == FINISH_WARP) {
    if (!defer) return;
    if (lane == 0) first_item = at;
    asm volatile("bar.sync 2, %0;" ::"n"(32 * (WARPS + 1)) : "memory");  // the partial result is written
    __threadfence();
    if (lane == 0) {
      first_is_last = atomicAdd(static_cast<int*>(p.workspace) + first_owner, 1) == first_last - first_owner;
      mbar_arrive(finished);
    }
    return;
  }
  if (warp == LOAD_WARP) {
    // ------------------------------------------------------------ loads
    constexpr int OPS = 2 * S::HALVES;  // boxes of one run of keys
    const int chunks = static_cast<int>(p.dim) / 8;
    int slot = 0, phase = 1, items = 0, blocks = 0;
    bool fresh = true;
    while (at.left > 0) {
      if (fresh) {  // the item's queries
        attn_wait(q_empty, (items & 1) ^ 1, abort_flag, status, SITE_ATTN_LOAD);
        __syncwarp();
        const TileRows tile(p, walk, at);
        const uint32_t dst = smem_u32(q_tile);
        for (int i = lane; i < M * chunks; i += 32) {
          const int row = i / chunks, c = i - row * chunks;
          int node, head;
          const bool real = tile.find(row, &node, &head);
          const T* q = static_cast<const T*>(p.q);
          if (real) q += static_cast<long long>(at.row0 + node) * p.sq_t + head * p.sq_h + 8 * c;
          cp_async_16(dst + chunk_at<DP, M>(row, c), q, real);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(q_full) : "memory");
        ++items;
      }
      const int pos0 = at.blk * KEYS;
      uint32_t bits[2] = {0u, 0u};
      if constexpr (BULK) {
        const int part = lane / OPS, op = lane % OPS;
        const bool mine = part * box_rows < KEYS;
        const int pos = pos0 + part * box_rows;
        int in_page = 0;
        const int page = mine ? page_of(p, by_page, at, pos, &in_page) : -1;
        if (page >= 0) {
          const int rows = min(box_rows, at.length - pos);
          const unsigned long long b = (~0ull >> (64 - rows)) << (part * box_rows);
          bits[0] = static_cast<uint32_t>(b);
          bits[1] = static_cast<uint32_t>(b >> 32);
        }
        bits[0] = __reduce_or_sync(0xffffffffu, bits[0]);
        bits[1] = __reduce_or_sync(0xffffffffu, bits[1]);
        attn_wait(empty + 8 * slot, phase, abort_flag, status, SITE_ATTN_LOAD);
        __syncwarp();
        if (lane == 0) {
          present[2 * slot] = bits[0];
          present[2 * slot + 1] = bits[1];
          mbar_arrive_expect_tx(full + 8 * slot, 2 * S::TILE);
        }
        __syncwarp();
        if (mine) {
          const int half = op >> 1;
          const uint32_t dst = ring + (2 * slot + (op & 1)) * S::TILE + half * (KEYS * 128) +
                               part * box_rows * (DP >= 64 ? 128 : 64);
          tma_load_4d(dst, (op & 1) ? &tm_v : &tm_k, full + 8 * slot, 64 * half, in_page, at.head,
                      page >= 0 ? page : static_cast<int>(p.pages));
        }
        __syncwarp();
      } else {
        // a lane copies two rows of keys
        int page[2], in_page[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          page[i] = page_of(p, by_page, at, pos0 + lane + 32 * i, &in_page[i]);
          bits[i] = __ballot_sync(0xffffffffu, page[i] >= 0);
        }
        attn_wait(empty + 8 * slot, phase, abort_flag, status, SITE_ATTN_LOAD);
        __syncwarp();
        if (lane < 2) present[2 * slot + lane] = bits[lane];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const long long pg = max(page[i], 0);
          const T* k = static_cast<const T*>(p.k) + at.head * p.sk_h + pg * p.sk_p + in_page[i] * p.sk_t;
          const T* v = static_cast<const T*>(p.v) + at.head * p.sv_h + pg * p.sv_p + in_page[i] * p.sv_t;
          const uint32_t dst = ring + 2 * slot * S::TILE;
          for (int c = 0; c < chunks; ++c) {
            cp_async_16(dst + chunk_at<DP, KEYS>(lane + 32 * i, c), k + 8 * c, page[i] >= 0);
            cp_async_16(dst + S::TILE + chunk_at<DP, KEYS>(lane + 32 * i, c), v + 8 * c, page[i] >= 0);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(full + 8 * slot);  // for `present`; and each lane once its copies have landed
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full + 8 * slot) : "memory");
      }
      ++blocks;
      if (++slot == STAGES) {
        slot = 0;
        phase ^= 1;
      }
      fresh = walk.item_ends(at);
      walk.advance(p, at);
    }
    if (*abort_flag & 1) {
      // a wait gave up: let the copies in flight land before the shared memory goes away
      asm volatile("cp.async.wait_all;" ::: "memory");
      for (int s = 0; s < STAGES && s < blocks; ++s)
        mbar_wait(full + 8 * s, ((blocks - 1 - s) / STAGES) & 1, nullptr, status, SITE_DRAIN, DRAIN_NS);
    }
    return;
  }

  // -------------------------------------------------------------- products
  // A wait that gives up records its status and the warps go on together (the
  // results are lost, the barriers between them are not).
  const auto join = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory"); };
  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];
  int stage = 0, phase = 0, items = 0;
  const uint32_t k_first = first_pair<DP, KEYS>(warp * KW + ((lane >> 4) << 3) + (lane & 7), (lane >> 3) & 1);
  const uint32_t v_first = S::TILE + first_pair<DP, KEYS>(warp * KW + (((lane >> 3) & 1) << 3) + (lane & 7), lane >> 4);
  while (at.left > 0) {  // items; what a block needs is dead between them
    attn_wait(q_full, items & 1, abort_flag, status, SITE_ATTN_SOFTMAX);
    __syncwarp();
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
      ldmatrix_x4(qf[k], pair_at<M>(smem_u32(q_tile) + first_pair<DP, M>((((lane >> 3) & 1) << 3) + (lane & 7), lane >> 4), k));
    __syncwarp();
    if (lane == 0) mbar_arrive(q_empty);
    ++items;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    for (;;) {
      attn_wait(full + 8 * stage, phase, abort_flag, status, SITE_ATTN_SOFTMAX);
      __syncwarp();
      const uint32_t tile_at = ring + stage * 2 * S::TILE;
      // two sums for each half of the head: their products wait less for one another
      float s[KW / 8][4], s2[KW / 8][4];
#pragma unroll
      for (int n = 0; n < KW / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = s2[n][0] = s2[n][1] = s2[n][2] = s2[n][3] = 0.0f;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        uint32_t b[4];
        ldmatrix_x4(b, pair_at<KEYS>(tile_at + k_first, k));
        auto& to = k % 2 ? s2 : s;
        mma16816<T>(to[0], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[0], b[1]);
        mma16816<T>(to[1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[2], b[3]);
      }
#pragma unroll
      for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s[n][x] += s2[n][x];
      }
      // base-2 scores, -inf where a row sees nothing
      const int key0 = at.blk * KEYS + warp * KW;
      const uint32_t mine = (present[2 * stage + warp / 2] >> (warp % 2 * KW)) & 0xffffu;  // this warp's keys, from bit 0
      if (key0 + KW <= at.context && mine == 0xffffu) {
#pragma unroll
        for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
          for (int x = 0; x < 4; ++x) s[n][x] *= p.scale_log2;
        }
      } else {
        const TileRows tile(p, walk, at);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int node, head;
          tile.find((lane >> 2) + 8 * h, &node, &head);
          const uint32_t seen = mine & nodes_seen(p, at, node, key0 - at.context);
#pragma unroll
          for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
              s[n][2 * h + x] = (seen >> (n * 8 + 2 * (lane & 3) + x)) & 1u ? s[n][2 * h + x] * p.scale_log2 : -INFINITY;
          }
        }
        if (BULK && key0 + KW > at.length) {  // rows past the request's end hold anything
          const int from = max(at.length - key0, 0);
          for (int i = from * (DP / 8) + lane; i < KW * (DP / 8); i += 32)
            *reinterpret_cast<uint4*>(smem + (2 * stage + 1) * S::TILE +
                                      chunk_at<DP, KEYS>(warp * KW + i / (DP / 8), i % (DP / 8))) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();  // before the next box lands here
        }
        __syncwarp();
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float top = m[h];
#pragma unroll
        for (int n = 0; n < KW / 8; ++n) top = fmaxf(top, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (__any_sync(0xffffffffu, top > m[h])) {
          const float fix = top > m[h] ? ex2_ftz(m[h] - top) : 1.0f;
          l[h] *= fix;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n) {
            o[n][2 * h] *= fix;
            o[n][2 * h + 1] *= fix;
          }
          m[h] = top;
        }
        const float base = m[h] == -INFINITY ? 0.0f : m[h];
#pragma unroll
        for (int n = 0; n < KW / 8; ++n) {
          s[n][2 * h] = ex2_ftz(s[n][2 * h] - base);
          s[n][2 * h + 1] = ex2_ftz(s[n][2 * h + 1] - base);
          l[h] += s[n][2 * h] + s[n][2 * h + 1];
        }
      }
      {
        const uint32_t a0 = pack_pair<T>(s[0][0], s[0][1]), a1 = pack_pair<T>(s[0][2], s[0][3]);
        const uint32_t a2 = pack_pair<T>(s[1][0], s[1][1]), a3 = pack_pair<T>(s[1][2], s[1][3]);
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          uint32_t b[4];
          ldmatrix_x4_trans(b, pair_at<KEYS>(tile_at + v_first, n));
          mma16816<T>(o[2 * n], a0, a1, a2, a3, b[0], b[1]);
          mma16816<T>(o[2 * n + 1], a0, a1, a2, a3, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * stage);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
      if (walk.item_ends(at)) break;
      walk.advance(p, at);
    }

    // The item's last block of this run: join the warps' sums.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if ((lane & 3) == 0) {
        part_m[((lane >> 2) + 8 * h) * WARPS + warp] = m[h];
        part_l[((lane >> 2) + 8 * h) * WARPS + warp] = l[h];
      }
    }
    join();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 tops = *reinterpret_cast<const float4*>(part_m + ((lane >> 2) + 8 * h) * WARPS);
      const float top = fmaxf(fmaxf(tops.x, tops.y), fmaxf(tops.z, tops.w));
      const float fix = m[h] == -INFINITY ? 0.0f : ex2_ftz(m[h] - top);
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        o[n][2 * h] *= fix;
        o[n][2 * h + 1] *= fix;
      }
    }
#pragma unroll 1
    for (int c = 0; c < WARPS; ++c) {
      if (c == warp) {
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float2* to = reinterpret_cast<float2*>(joined + ((lane >> 2) + 8 * h) * S::PITCH + n * 8 + 2 * (lane & 3));
            float2 v = make_float2(o[n][2 * h], o[n][2 * h + 1]);
            if (c > 0) {
              const float2 w = *to;
              v.x += w.x;
              v.y += w.y;
            }
            *to = v;
          }
        }
      }
      join();
    }
    const TileRows tile(p, walk, at);
    const int item = run.count - at.left - at.blk;  // the item's first position, counted from the run's
    const bool whole = item >= 0 && at.blk + 1 == at.blocks;
    const Partial<M, DP> part(p, blockIdx.x, item >= 0);
    constexpr int LANES = DP / 8, PASS = 32 * WARPS / LANES;
    const int col = (tid % LANES) * 8;
#pragma unroll 1
    for (int row0 = 0; row0 < tile.rows(); row0 += PASS) {
      const int row = row0 + tid / LANES;
      int t, head;
      const bool real = tile.find(row, &t, &head);
      t += at.row0;
      bool bad = false;
      if (real) {
        const float4 tops = *reinterpret_cast<const float4*>(part_m + row * WARPS);
        const float4 sums = *reinterpret_cast<const float4*>(part_l + row * WARPS);
        const float top = fmaxf(fmaxf(tops.x, tops.y), fmaxf(tops.z, tops.w)), base = top == -INFINITY ? 0.0f : top;
        const float sum = fmaf(sums.x, ex2_ftz(tops.x - base), sums.y * ex2_ftz(tops.y - base)) +
                          fmaf(sums.z, ex2_ftz(tops.z - base), sums.w * ex2_ftz(tops.w - base));
        const float4 a = *reinterpret_cast<const float4*>(joined + row * S::PITCH + col);
        const float4 b = *reinterpret_cast<const float4*>(joined + row * S::PITCH + col + 4);
        if (whole) {
          const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
          if (col < p.dim) bad = store_8<T>(p, t, head, col, v, sum, vector_out);
          if (col == 0) store_lse(p, t, head, top, sum);
        } else {
          __stcg(reinterpret_cast<float4*>(part.row(row) + col), a);
          __stcg(reinterpret_cast<float4*>(part.row(row) + col + 4), b);
          if (col == 0) {
            __stcg(part.top(row), top);
            __stcg(part.sum(row), sum);
          }
        }
      }
      redo_rows<T, DP / 32>(p, bad, t, head, lane, abort_flag);
    }
    if (!whole && defer && item < 0) {
      asm volatile("bar.arrive 2, %0;" ::"n"(32 * (WARPS + 1)) : "memory");
    } else if (!whole) {
      int* counters = static_cast<int*>(p.workspace);
      const int owner = static_cast<int>((run.first + item) / run.per);
      const int last = static_cast<int>((run.first + item + at.blocks - 1) / run.per);
      __threadfence();
      join();
      if (tid == 0) last_one = atomicAdd(counters + owner, 1) == last - owner;
      join();
      if (last_one) {
        __threadfence();
        join_partials<T, M, DP, 32 * WARPS>(p, at, tile, owner, last, tid, vector_out, DP >= 64 ? joined : nullptr, abort_flag, join);
        if (tid == 0) counters[owner] = 0;
      }
    }
    join();  // `joined` and the maxima may be written again
    walk.advance(p, at);
  }
  if (defer) {
    // one thread looks: the warps take one way even where the wait gave up
    const bool there = attn_wait(finished, 0, abort_flag, status, SITE_ATTN_SOFTMAX);
    if (tid == 0) last_one = there && first_is_last;
    join();
    if (last_one) {
      __threadfence();
      const Cursor c = first_item;
      join_partials<T, M, DP, 32 * WARPS>(p, c, TileRows(p, walk, c), first_owner, first_last, tid, vector_out,
                                          DP >= 64 ? joined : nullptr, abort_flag, join);
      if (tid == 0) static_cast<int*>(p.workspace)[first_owner] = 0;
    }
  }
}

template <typename T, typename S>
int launch_shape(const AttnArgs& a, const DeviceInfo& dev, int ctas, cudaStream_t stream) {
  static std::once_flag once;
  static cudaError_t attr = cudaSuccess;
  std::call_once(once, [] {
    attr = cudaFuncSetAttribute(tree_kernel<T, S, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (attr == cudaSuccess)
      attr = cudaFuncSetAttribute(tree_kernel<T, S, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  });
  if (attr != cudaSuccess) return cuda_error(attr, "tree attention attributes");
  const int vector_out = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.so_t % 8 == 0 && a.so_h % 8 == 0;
  // Keys that lie in one page wherever a block starts; boxes of 8 or more keep
  // whole swizzle patterns. A cache that no tensor map describes (a stride of
  // zero or beyond its range) is copied row by row.
  CUtensorMap k{}, v{};
  const int box_rows = static_cast<int>(std::gcd(a.block_size, static_cast<int64_t>(KEYS)));
  const int width = S::DP < 64 ? 32 : 64;
  const bool bulk = box_rows >= 8 && encode_pages(&k, a, a.k, a.sk_p, a.sk_h, a.sk_t, box_rows, width) &&
                    encode_pages(&v, a, a.v, a.sv_p, a.sv_h, a.sv_t, box_rows, width);
  const auto kernel = bulk ? tree_kernel<T, S, true> : tree_kernel<T, S, false>;
  kernel<<<static_cast<unsigned>(ctas), THREADS, S::SMEM, stream>>>(k, v, a, divisor(a.block_size), box_rows, vector_out,
                                                                   dev.status);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(tree attention)");
}

int padded_dim(const AttnArgs& a) { return a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128; }

template <typename T>
int launch_typed(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  // two CTAs an SM, and no more than a table of full rows could give work
  const int64_t group = a.heads / a.kv_heads;
  const int64_t tiles = (a.rows * ceil_div(group, M) + a.seqs + 1) * a.kv_heads;
  const int64_t blocks = ceil_div(a.table_cols * a.block_size, KEYS) + ITEM_COST;
  int ctas = 2 * dev.sm_count;
  if (tiles < ctas && blocks < ctas && ceil_div(tiles * blocks, MIN_RUN) < ctas)
    ctas = static_cast<int>(ceil_div(tiles * blocks, MIN_RUN));
  switch (padded_dim(a)) {
    case 32: return launch_shape<T, Shape<32, 8>>(a, dev, ctas, stream);
    case 64: return launch_shape<T, Shape<64, 5>>(a, dev, ctas, stream);
    default: return launch_shape<T, Shape<128, 3>>(a, dev, ctas, stream);
  }
}

bool on_grid(const void* ptr, int64_t vec, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(ptr) % (2 * vec) != 0) return false;
  for (int64_t s : strides)
    if (s % vec != 0) return false;
  return true;
}

}  // namespace

bool attention_tree_supported(const AttnArgs& a) {
  return (a.dtype == KF_FP16 || a.dtype == KF_BF16) && a.dim <= 128 && a.dim % 8 == 0 && a.seqs > 0 && a.pages > 0 &&
         on_grid(a.k, 8, {a.sk_p, a.sk_h, a.sk_t}) && on_grid(a.v, 8, {a.sv_p, a.sv_h, a.sv_t}) &&
         on_grid(a.q, 8, {a.sq_t, a.sq_h});
}

// Rows that a request has for a key head on average: above 16 the products of
// mma.sync tiles take longer than the cache's bytes. 16 trees over 8192 keys, 32 heads to 8,
// by their nodes, here and on tcgen05 tiles: 4 99 us and 106, 5 174 and 107, 9 253 and 110,
// 16 330 and 114; 64 requests of one token 98 and 150. (With up to 8 nodes over up to 8192
// keys 75 and 83: trees far apart in size are taken for their mean.)
static bool many_rows(const AttnArgs& a) {
  return ceil_div(a.rows, a.seqs > 0 ? a.seqs : 1) * (a.heads / a.kv_heads) > M;
}

int64_t attention_tree_workspace_bytes(const AttnArgs& a, const DeviceInfo& dev) {
  const int64_t narrow = TREE_COUNTER_BYTES + 4ll * 2 * (2 * dev.sm_count) * M * (padded_dim(a) + 2);
  const int64_t wide = many_rows(a) ? attention_tree_wide_workspace_bytes(a, dev) : 0;
  return narrow > wide ? narrow : wide;
}

int launch_attention_tree(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t need = attention_tree_workspace_bytes(a, dev);
  if (a.workspace == nullptr || a.workspace_bytes < need)
    return set_error(KF_ERR_WORKSPACE, "tree attention needs " + std::to_string(need) + " bytes of workspace; got " +
                                           std::to_string(a.workspace == nullptr ? 0 : a.workspace_bytes));
  if (2 * dev.sm_count > TREE_COUNTER_BYTES / 4) return set_error(KF_ERR_UNSUPPORTED, "tree attention: too many SMs");
  if (many_rows(a) && attention_tree_wide_supported(a)) return launch_attention_tree_wide(a, dev, stream);
  return a.dtype == KF_FP16 ? launch_typed<__half>(a, dev, stream) : launch_typed<__nv_bfloat16>(a, dev, stream);
}

}  // namespace kf
