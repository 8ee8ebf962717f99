// Attention of new tokens (one, a chain or a tree of drafts per request) over a
// paged cache, fp16/bf16, heads of up to 128 elements.
//
// All query rows of a request that share a key head -- its nodes times the
// heads of the group -- form tiles of M rows against the request's keys, so the
// cache is read once for all of them. The work of all requests, key heads and
// tiles is one list of (item, block of 64 keys) units, cut into equal runs, one per
// CTA: a long cache is spread over the GPU and short ones share a CTA, whatever
// the lengths, which only the device knows. An item cut between CTAs leaves
// partial sums (m, l, O) in the workspace, and whichever CTA arrives last adds
// them in the order of the keys, so results do not depend on timing and nobody
// waits for another CTA.
//
// In a CTA, R x C warps: warp (r, c) holds 16 rows and takes the keys
// [c 64/C, (c+1) 64/C) of each block, with its own running maximum and sum:
//
//   s = scale log2(e) q k^T,  m' = max(m, max s),  p = 2^(s - m'),
//   l = l 2^(m - m') + sum p,  O = O 2^(m - m') + p v       (mma.sync, fp32 sums)
//
// One more warp loads: it reads the block table ahead and fills a ring of K and
// V blocks, with one TMA box per run of keys that is whole in any page (gcd of
// page and block, 8 keys at least), or where pages are not multiples of 8 keys
// with 16-byte cp.async. Pages a table does not name are read as zeros (a box
// past the last page); V rows past the request's end are zeroed in shared memory
// (0 x NaN is NaN); weights of keys that a row does not see are zero. A row that
// comes out non-finite (a node it does not see holds infinities) is recomputed key by key.
//
// With one new token and G heads to a key head, G of the 16 rows are real: the
// products are free beside the cache's bytes, which bound the call until
// nodes x G passes about 64.
#include <cudaTypedefs.h>

#include <initializer_list>
#include <mutex>
#include <numeric>
#include <string>

#include "attention.cuh"

namespace kf {
namespace {

constexpr int KEYS = 64;      // of a block
constexpr int MIN_BLOCKS = 4; // a CTA's run: fewer blocks cost more to join than to read

template <int DP_, int R_, int C_, int STAGES_>
struct Shape {
  static constexpr int DP = DP_, R = R_, C = C_, STAGES = STAGES_;
  // With 8 warps of products the loading warp gets a warpgroup of its own, whose
  // registers go to them: 3 x 168 a thread become 2 x 224 and 56.
  static constexpr int M = 16 * R, WARPS = R * C, LOADERS = WARPS == 8 ? 4 : 1, THREADS = 32 * (WARPS + LOADERS);
  static constexpr int HALVES = DP == 128 ? 2 : 1;  // boxes of at most 128 bytes a row
  static constexpr int TILE = KEYS * DP * 2;        // bytes of a K or V block in the ring
  static constexpr int PITCH = DP + 8;              // floats of a row of the joined result
  static constexpr int SMEM = 1024 + STAGES * 2 * TILE + M * PITCH * 4 + 2 * M * C * 4 + STAGES * 24;
  static constexpr int64_t PARTIAL = M * DP + 2 * M;  // floats of a partial result
};

// Workspace: arrival counters of items cut between CTAs, one per CTA, at a fixed
// place and zero between calls; then two partial results per CTA.
constexpr uint64_t DRAIN_NS = 100000000ull;
constexpr int64_t COUNTER_BYTES = 64 * 1024;

struct Run {
  long long per, total;  // units of a CTA and of all
};

// The block that a CTA works on: request, key head, row tile, block of keys.
struct Cursor {
  int left;  // units of the CTA's run from this one on
  int r, head, tile, blk;
  int row0, nodes, tiles, blocks;
  int context, length;
};

__device__ __forceinline__ void load_request(const AttnArgs& p, Cursor& c, int group, int m) {
  int begin, end;
  request_rows(p, c.r, &begin, &end);
  long long first, length;
  request_keys(p, c.r, end - begin, &first, &length);
  c.length = static_cast<int>(length);
  c.row0 = begin;
  c.nodes = end - begin;
  c.context = c.r < p.seqs ? max(__ldg(p.context + c.r), 0) : 0;
  c.tiles = static_cast<int>((static_cast<long long>(c.nodes) * group + m - 1) / m);
  c.blocks = max(1, (c.length + KEYS - 1) / KEYS);
}

__device__ __forceinline__ void advance(const AttnArgs& p, Cursor& c, int group, int m) {
  --c.left;
  if (++c.blk < c.blocks) return;
  c.blk = 0;
  if (++c.tile < c.tiles) return;
  c.tile = 0;
  if (++c.head < p.kv_heads) return;
  c.head = 0;
  do {
    if (++c.r > p.seqs) return;
    load_request(p, c, group, m);
  } while (c.tiles == 0);
}

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

// Byte offset of 16-byte chunk `chunk` of row `row` in a tile, as TMA's swizzles
// place it: rows of 128 bytes (64 elements, a second half behind the first) or of
// 64 bytes, chunks XORed so that eight rows of one column meet eight bank groups.
template <int DP>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
  if constexpr (DP >= 64) {
    return static_cast<uint32_t>((chunk >> 3) * (KEYS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
  } else {
    return static_cast<uint32_t>(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  uint32_t r;
  if constexpr (DType<T>::code == KF_BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  }
  return r;
}

template <typename T, int NE>
__device__ __noinline__ void redo_row(const AttnArgs& p, int t, int head, int lane) {
  float acc[NE], m, l;
  attend_row<T, NE>(p, t, head, lane, acc, &m, &l);
  write_row<T, NE>(p, t, head, lane, acc, m, l);
}

// Writes one finished row, 4 elements a lane: acc / l.
template <typename T, int DP>
__device__ __forceinline__ void store_row(const AttnArgs& p, int t, int head, int lane, float4 o, float m, float l,
                                          int vector_out) {
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  const bool mine = 4 * lane < p.dim;
  const float v[4] = {l > 0.0f ? o.x * inv : 0.0f, l > 0.0f ? o.y * inv : 0.0f, l > 0.0f ? o.z * inv : 0.0f,
                      l > 0.0f ? o.w * inv : 0.0f};
  bool bad = !(l >= 0.0f && l < INFINITY);
  if (mine) {
    T* out = static_cast<T*>(p.out) + static_cast<long long>(t) * p.so_t + head * p.so_h + 4 * lane;
    const uint2 w = make_uint2(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]));
    if (vector_out) {
      *reinterpret_cast<uint2*>(out) = w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = from_f32<T>(v[i]);
    }
    float zero = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) zero = fmaf(v[i], 0.0f, zero);
    bad = bad || !(zero == 0.0f);
  }
  if (p.lse != nullptr && lane == 0)
    p.lse[static_cast<long long>(t) * p.heads + head] = l > 0.0f ? m * 0.69314718055994530942f + logf(l) : -INFINITY;
  if (__any_sync(0xffffffffu, bad)) redo_row<T, DP / 32>(p, t, head, lane);
}

// n / d = n * mul >> shift for n below 2^31: with 2^s >= d, mul = ceil(2^(31 + s) / d)
// exceeds 2^(31 + s) / d by less than one, too little to reach the next quotient.
struct Divisor {
  uint32_t mul;
  int shift;
};

template <typename T, typename S, bool BULK>
__global__ void __launch_bounds__(S::THREADS, S::WARPS == 4 ? 2 : 1)
    tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ AttnArgs p, const Divisor by_page, int box_rows, int vector_out, int* status) {
  constexpr int DP = S::DP, C = S::C, M = S::M, STAGES = S::STAGES, THREADS = S::THREADS;
  constexpr int KW = KEYS / C;  // keys of a warp
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // ring | joined | maxima and sums (16-byte vectors up to here) | barriers | present
  float* joined = reinterpret_cast<float*>(smem + STAGES * 2 * S::TILE);
  float* part_m = joined + M * S::PITCH;
  float* part_l = part_m + M * C;
  uint64_t* bars = reinterpret_cast<uint64_t*>(part_l + M * C);
  volatile uint32_t* present = reinterpret_cast<volatile uint32_t*>(bars + 2 * STAGES);  // a bit per key of each stage
  static_assert(S::TILE % 1024 == 0 && (M * S::PITCH) % 4 == 0 && S::PITCH % 4 == 0 && (M * C) % 2 == 0 && S::PARTIAL % 4 == 0,
                "vectors of 16 bytes and barriers of 8");
  __shared__ long long scan[S::WARPS + S::LOADERS];
  __shared__ long long found_rest;
  __shared__ int found_r, last_one, abort_word;
  volatile int* abort_flag = &abort_word;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int group = static_cast<int>(p.heads / p.kv_heads);
  const uint32_t ring = smem_u32(smem), full = smem_u32(bars), empty = full + 8 * STAGES;
  float* partials = reinterpret_cast<float*>(static_cast<uint8_t*>(p.workspace) + COUNTER_BYTES);
  int* counters = static_cast<int*>(p.workspace);

  if (tid == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + 8 * s, BULK ? 1 : 33);
      mbar_init(empty + 8 * s, S::WARPS);
    }
    abort_word = 0;
    mbar_init_fence();
  }
  if (!BULK && p.dim < DP)  // columns past the head stay zero
    for (int i = tid; i < STAGES * 2 * S::TILE / 16; i += THREADS)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0u, 0u, 0u, 0u);

  // Where this CTA's run begins: units are summed over the requests, a
  // contiguous share of them per thread, and the thread whose share holds the
  // first unit finds it.
  Run run;
  {
    const int share = static_cast<int>((p.seqs + 1 + THREADS - 1) / THREADS);
    const int r0 = tid * share, r1 = min(static_cast<int>(p.seqs) + 1, r0 + share);
    long long sum = 0;
    Cursor c;
    for (c.r = r0; c.r < r1; ++c.r) {
      load_request(p, c, group, M);
      sum += static_cast<long long>(c.tiles) * p.kv_heads * c.blocks;
    }
    long long upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    long long before = 0;
    run.total = 0;
#pragma unroll
    for (int w = 0; w < S::WARPS + S::LOADERS; ++w) {
      if (w < warp) before += scan[w];
      run.total += scan[w];
    }
    before += upto - sum;
    run.per = max((run.total + gridDim.x - 1) / gridDim.x, static_cast<long long>(MIN_BLOCKS));
    const long long start = run.per * blockIdx.x;
    if (start >= before && start < before + sum) {
      long long rest = start - before;
      for (c.r = r0; c.r < r1; ++c.r) {
        load_request(p, c, group, M);
        const long long units = static_cast<long long>(c.tiles) * p.kv_heads * c.blocks;
        if (rest < units) break;
        rest -= units;
      }
      found_r = c.r;
      found_rest = rest;
    }
    __syncthreads();
  }
  const long long first = run.per * blockIdx.x, stop = min(first + run.per, run.total);
  if (first >= stop) return;
  const int units = static_cast<int>(stop - first);
  Cursor at;
  at.r = found_r;
  load_request(p, at, group, M);
  {
    const long long rest = found_rest;
    const int tile = static_cast<int>(rest / at.blocks);
    at.blk = static_cast<int>(rest - static_cast<long long>(tile) * at.blocks);
    at.head = tile / at.tiles;
    at.tile = tile - at.head * at.tiles;
    at.left = units;
  }

  if (warp >= S::WARPS) {
    // ------------------------------------------------------------ loads
    if constexpr (S::LOADERS == 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp > S::WARPS) return;
    constexpr int OPS = 2 * S::HALVES;  // boxes of one run of keys
    int slot = 0, phase = 1;
    for (; at.left > 0; advance(p, at, group, M)) {
      const int pos0 = at.blk * KEYS;
      uint32_t bits[2] = {0u, 0u};
      if constexpr (BULK) {
        const int part = lane / OPS, op = lane % OPS;
        const bool mine = part * box_rows < KEYS;
        const int pos = pos0 + part * box_rows;
        int page = -1, in_page = 0;
        if (mine && pos < at.length) {
          const uint32_t n = static_cast<uint32_t>(pos);
          const uint32_t col = static_cast<uint32_t>(static_cast<uint64_t>(n) * by_page.mul >> by_page.shift);
          in_page = static_cast<int>(n - col * static_cast<uint32_t>(p.block_size));
          page = __ldg(p.table + at.r * p.table_stride + col);
          if (page < 0 || page >= p.pages) page = -1;
        }
        if (page >= 0) {
          const int rows = min(box_rows, at.length - pos);
          const unsigned long long b = (~0ull >> (64 - rows)) << (part * box_rows);
          bits[0] = static_cast<uint32_t>(b);
          bits[1] = static_cast<uint32_t>(b >> 32);
        }
        bits[0] = __reduce_or_sync(0xffffffffu, bits[0]);
        bits[1] = __reduce_or_sync(0xffffffffu, bits[1]);
        mbar_wait(empty + 8 * slot, phase, abort_flag, status, SITE_ATTN_LOAD);
        __syncwarp();
        if (lane == 0) {
          present[2 * slot] = bits[0];
          present[2 * slot + 1] = bits[1];
          mbar_arrive_expect_tx(full + 8 * slot, 2 * S::TILE);
        }
        __syncwarp();
        if (mine) {
          const int half = op >> 1;
          const uint32_t dst = ring + (2 * slot + (op & 1)) * S::TILE + half * (KEYS * 128) + part * box_rows * (DP >= 64 ? 128 : 64);
          tma_load_4d(dst, (op & 1) ? &tm_v : &tm_k, full + 8 * slot, 64 * half, in_page, at.head,
                      page >= 0 ? page : static_cast<int>(p.pages));
        }
        __syncwarp();
      } else {
        // a lane copies two rows of keys
        const int chunks = static_cast<int>(p.dim) / 8;
        int page[2], in_page[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int pos = pos0 + lane + 32 * i;
          page[i] = -1;
          in_page[i] = 0;
          if (pos < at.length) {
            const uint32_t n = static_cast<uint32_t>(pos);
            const uint32_t col = static_cast<uint32_t>(static_cast<uint64_t>(n) * by_page.mul >> by_page.shift);
            in_page[i] = static_cast<int>(n - col * static_cast<uint32_t>(p.block_size));
            page[i] = __ldg(p.table + at.r * p.table_stride + col);
            if (page[i] < 0 || page[i] >= p.pages) page[i] = -1;
          }
          bits[i] = __ballot_sync(0xffffffffu, page[i] >= 0);
        }
        mbar_wait(empty + 8 * slot, phase, abort_flag, status, SITE_ATTN_LOAD);
        __syncwarp();
        if (lane < 2) present[2 * slot + lane] = bits[lane];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const long long pg = max(page[i], 0);
          const T* k = static_cast<const T*>(p.k) + at.head * p.sk_h + pg * p.sk_p + in_page[i] * p.sk_t;
          const T* v = static_cast<const T*>(p.v) + at.head * p.sv_h + pg * p.sv_p + in_page[i] * p.sv_t;
          const uint32_t dst = ring + 2 * slot * S::TILE;
          for (int c = 0; c < chunks; ++c) {
            cp_async_16(dst + chunk_at<DP>(lane + 32 * i, c), k + 8 * c, page[i] >= 0);
            cp_async_16(dst + S::TILE + chunk_at<DP>(lane + 32 * i, c), v + 8 * c, page[i] >= 0);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(full + 8 * slot);  // for `present`; and each lane once its copies have landed
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full + 8 * slot) : "memory");
      }
      if (++slot == STAGES) {
        slot = 0;
        phase ^= 1;
      }
    }
    if (*abort_flag) {
      // a wait gave up: let the copies in flight land before the shared memory goes away
      for (int s = 0; s < STAGES && s < units; ++s)
        mbar_wait(full + 8 * s, ((units - 1 - s) / STAGES) & 1, nullptr, status, SITE_DRAIN, DRAIN_NS);
    }
    return;
  }

  // -------------------------------------------------------------- products
  if constexpr (S::LOADERS == 4) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
  // A wait that gives up records its status and the warps go on together (the
  // results are lost, the barriers between them are not).
  const int wr = warp / C, wc = warp % C;  // row group, key group
  const auto join = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * S::WARPS) : "memory"); };
  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];
  int stage = 0, phase = 0;
  bool fresh = true;
  while (at.left > 0) {
    const int tile_row = at.tile * M + wr * 16 + (lane >> 2);  // of this lane's first row, over nodes x group
    const int real = at.nodes * group;                         // rows of the item
    if (fresh) {
      fresh = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = tile_row + 8 * h;
        const T* q = static_cast<const T*>(p.q) + static_cast<long long>(at.row0 + row / group) * p.sq_t +
                     (static_cast<long long>(at.head) * group + row % group) * p.sq_h;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int e = 16 * k + 8 * x + 2 * (lane & 3);
            qf[k][h + 2 * x] = row < real && e < p.dim ? __ldg(reinterpret_cast<const uint32_t*>(q + e)) : 0u;
          }
        }
        m[h] = -INFINITY;
        l[h] = 0.0f;
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    }
    mbar_wait(full + 8 * stage, phase, abort_flag, status, SITE_ATTN_SOFTMAX);
    __syncwarp();
    const uint32_t k_tile = ring + stage * 2 * S::TILE, v_tile = k_tile + S::TILE;
    float s[KW / 8][4];
#pragma unroll
    for (int n = 0; n < KW / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
      for (int n = 0; n < KW / 16; ++n) {
        uint32_t b[4];
        ldmatrix_x4(b, k_tile + chunk_at<DP>(wc * KW + n * 16 + ((lane >> 4) << 3) + (lane & 7),
                                             2 * k + ((lane >> 3) & 1)));
        mma16816<T>(s[2 * n], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[0], b[1]);
        mma16816<T>(s[2 * n + 1], qf[k][0], qf[k][1], qf[k][2], qf[k][3], b[2], b[3]);
      }
    }
    // base-2 scores, -inf where a row sees nothing
    const int key0 = at.blk * KEYS + wc * KW;
    const int node_of[2] = {tile_row / group, (tile_row + 8) / group};
    const bool drafts = key0 + KW > at.context;  // some of these keys are nodes of the request
    const uint32_t mine = present[2 * stage + wc * KW / 32] >> (wc * KW % 32);  // this warp's keys, from bit 0
    if (!drafts && (KW == 32 ? mine == 0xffffffffu : (mine & 0xffffu) == 0xffffu)) {
#pragma unroll
      for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) s[n][x] *= p.scale_log2;
      }
    } else {
#pragma unroll
      for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int col = n * 8 + 2 * (lane & 3) + (x & 1);
          bool seen = (mine >> col) & 1u;
          const int j = key0 + col - at.context;
          if (j >= 0) {
            const int node = node_of[x >> 1];
            if (p.mask == nullptr) {
              seen = seen && j <= node;
            } else {
              seen = seen && node < at.nodes && (j >> 6) < p.mask_words &&
                     ((__ldg(p.mask + (at.row0 + node) * p.mask_words + (j >> 6)) >> (j & 63)) & 1ull);
            }
          }
          s[n][x] = seen ? s[n][x] * p.scale_log2 : -INFINITY;
        }
      }
      if (BULK && key0 + KW > at.length) {  // rows past the request's end hold anything
        const int from = max(at.length - key0, 0);
        for (int i = from * (DP / 8) + lane; i < KW * (DP / 8); i += 32)
          *reinterpret_cast<uint4*>(smem + (2 * stage + 1) * S::TILE + chunk_at<DP>(wc * KW + i / (DP / 8), i % (DP / 8))) =
              make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();  // before the next box lands here
        __syncwarp();
      }
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
#pragma unroll
    for (int k = 0; k < KW / 16; ++k) {
      const uint32_t a0 = pack_pair<T>(s[2 * k][0], s[2 * k][1]), a1 = pack_pair<T>(s[2 * k][2], s[2 * k][3]);
      const uint32_t a2 = pack_pair<T>(s[2 * k + 1][0], s[2 * k + 1][1]), a3 = pack_pair<T>(s[2 * k + 1][2], s[2 * k + 1][3]);
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, v_tile + chunk_at<DP>(wc * KW + k * 16 + (((lane >> 3) & 1) << 3) + (lane & 7),
                                                   2 * n + (lane >> 4)));
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

    if (at.left > 1 && at.blk + 1 < at.blocks) {
      advance(p, at, group, M);
      continue;
    }

    // The item's last block of this run: join the key groups' sums.
    fresh = true;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int row = wr * 16 + (lane >> 2) + 8 * h;
      if ((lane & 3) == 0) {
        part_m[row * C + wc] = m[h];
        part_l[row * C + wc] = l[h];
      }
    }
    join();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = wr * 16 + (lane >> 2) + 8 * h;
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < C; ++c) top = fmaxf(top, part_m[row * C + c]);
      const float fix = m[h] == -INFINITY ? 0.0f : ex2_ftz(m[h] - top);
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        o[n][2 * h] *= fix;
        o[n][2 * h + 1] *= fix;
      }
    }
#pragma unroll 1
    for (int c = 0; c < C; ++c) {
      if (c == wc) {
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float2* to = reinterpret_cast<float2*>(joined + (wr * 16 + (lane >> 2) + 8 * h) * S::PITCH + n * 8 + 2 * (lane & 3));
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
    const int rows_here = min(M, at.nodes * group - at.tile * M);
    const int item = units - at.left - at.blk;  // the item's first unit, counted from the run's
    const bool whole = item >= 0 && at.blk + 1 == at.blocks;
    float* slot = partials + (2ll * blockIdx.x + (item >= 0)) * S::PARTIAL;
    for (int row = warp; row < rows_here; row += S::WARPS) {
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int c = 0; c < C; ++c) top = fmaxf(top, part_m[row * C + c]);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float pm = part_m[row * C + c];
        sum += pm == -INFINITY ? 0.0f : part_l[row * C + c] * ex2_ftz(pm - top);
      }
      const float4 v = 4 * lane < DP ? *reinterpret_cast<const float4*>(joined + row * S::PITCH + 4 * lane)
                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (whole) {
        const int at_row = at.tile * M + row;
        store_row<T, DP>(p, at.row0 + at_row / group, at.head * group + at_row % group, lane, v, top, sum, vector_out);
      } else {
        if (4 * lane < DP) __stcg(reinterpret_cast<float4*>(slot + row * DP + 4 * lane), v);
        if (lane == 0) {
          __stcg(slot + M * DP + row, top);
          __stcg(slot + M * DP + M + row, sum);
        }
      }
    }
    if (!whole) {
      const int owner = static_cast<int>((first + item) / run.per);
      const int last = static_cast<int>((first + item + at.blocks - 1) / run.per);
      __threadfence();
      join();
      if (tid == 0) last_one = atomicAdd(counters + owner, 1) == last - owner;
      join();
      if (last_one) {
        __threadfence();
        for (int row = warp; row < rows_here; row += S::WARPS) {
          // CTA `owner` holds the item's first blocks in its second slot, the others in their first
          float top = -INFINITY;
          for (int b = owner + lane; b <= last; b += 32)
            top = fmaxf(top, __ldcg(partials + (2ll * b + (b == owner)) * S::PARTIAL + M * DP + row));
#pragma unroll
          for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          float sum = 0.0f;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
          for (int b = owner; b <= last; ++b) {
            const float* from = partials + (2ll * b + (b == owner)) * S::PARTIAL;
            const float pm = __ldcg(from + M * DP + row), pl = __ldcg(from + M * DP + M + row);
            const float4 w = 4 * lane < DP ? __ldcg(reinterpret_cast<const float4*>(from + row * DP + 4 * lane))
                                           : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float fix = pm == -INFINITY ? 0.0f : ex2_ftz(pm - top);
            sum = fmaf(pl, fix, sum);
            v.x = fmaf(w.x, fix, v.x);
            v.y = fmaf(w.y, fix, v.y);
            v.z = fmaf(w.z, fix, v.z);
            v.w = fmaf(w.w, fix, v.w);
          }
          const int at_row = at.tile * M + row;
          store_row<T, DP>(p, at.row0 + at_row / group, at.head * group + at_row % group, lane, v, top, sum, vector_out);
        }
        if (tid == 0) counters[owner] = 0;
      }
    }
    join();  // `joined` and the maxima may be written again
    advance(p, at, group, M);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(sym);
  });
  return fn;
}

// Pages [pages, kv_heads, block_size, dim] as boxes of `box_rows` slots x 64 (32)
// elements; what lies past the head or past the last page is filled with zeros.
bool encode_pages(CUtensorMap* map, const AttnArgs& a, const void* ptr, int64_t s_page, int64_t s_head, int64_t s_slot,
                  int box_rows, int width) {
  auto enc = encoder();
  if (enc == nullptr) return false;
  const auto bytes = [](int64_t s, int64_t n) { return static_cast<cuuint64_t>(n > 1 ? 2 * s : 16); };
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.dim), static_cast<cuuint64_t>(a.block_size),
                              static_cast<cuuint64_t>(a.kv_heads), static_cast<cuuint64_t>(a.pages)};
  const cuuint64_t strides[3] = {bytes(s_slot, a.block_size), bytes(s_head, a.kv_heads), bytes(s_page, a.pages)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(width), static_cast<cuuint32_t>(box_rows), 1, 1};
  const cuuint32_t unit[4] = {1, 1, 1, 1};
  return enc(map, a.dtype == KF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void*>(ptr), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
             width == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, typename S>
int launch_shape(const AttnArgs& a, const DeviceInfo& dev, int ctas, cudaStream_t stream) {
  static std::once_flag once;
  static cudaError_t attr = cudaSuccess;
  static bool registers_suffice = true;
  std::call_once(once, [] {
    attr = cudaFuncSetAttribute(tree_kernel<T, S, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (attr == cudaSuccess)
      attr = cudaFuncSetAttribute(tree_kernel<T, S, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    // the warpgroups' shares must not exceed what the block is launched with
    for (const bool bulk : {true, false}) {
      cudaFuncAttributes f{};
      if (attr == cudaSuccess)
        attr = bulk ? cudaFuncGetAttributes(&f, tree_kernel<T, S, true>) : cudaFuncGetAttributes(&f, tree_kernel<T, S, false>);
      if (S::LOADERS == 4 && attr == cudaSuccess && 3 * f.numRegs < 2 * 224 + 56) registers_suffice = false;
    }
  });
  if (attr != cudaSuccess) return cuda_error(attr, "tree attention attributes");
  if (!registers_suffice) return set_error(KF_ERR_UNSUPPORTED, "tree attention: built with too few registers to split");
  const uint64_t d = static_cast<uint64_t>(a.block_size);
  int s = 0;
  while ((1ull << s) < d) ++s;
  const Divisor by{static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), 31 + s};
  const int vector_out = reinterpret_cast<uintptr_t>(a.out) % 8 == 0 && a.so_t % 4 == 0 && a.so_h % 4 == 0;
  // Keys that lie in one page wherever a block starts; boxes of 8 or more keep
  // whole swizzle patterns. A cache that no tensor map describes (a stride of
  // zero or beyond its range) is copied row by row.
  CUtensorMap k{}, v{};
  const int box_rows = static_cast<int>(std::gcd(a.block_size, static_cast<int64_t>(KEYS)));
  const int width = S::DP < 64 ? 32 : 64;
  const bool bulk = box_rows >= 8 && encode_pages(&k, a, a.k, a.sk_p, a.sk_h, a.sk_t, box_rows, width) &&
                    encode_pages(&v, a, a.v, a.sv_p, a.sv_h, a.sv_t, box_rows, width);
  const auto kernel = bulk ? tree_kernel<T, S, true> : tree_kernel<T, S, false>;
  kernel<<<static_cast<unsigned>(ctas), S::THREADS, S::SMEM, stream>>>(k, v, a, by, box_rows, vector_out, dev.status);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(tree attention)");
}

// Rows of a tile by the query rows that a request has for a key head on
// average, and the CTAs that fit the GPU.
struct Plan {
  int m, ctas, dp;
};

Plan plan_for(const AttnArgs& a, int sm_count) {
  Plan plan;
  const int64_t each = ceil_div(a.rows, a.seqs > 0 ? a.seqs : 1) * (a.heads / a.kv_heads);
  plan.m = each <= 16 ? 16 : 64;
  plan.ctas = plan.m == 16 ? 2 * sm_count : sm_count;
  plan.dp = a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128;
  return plan;
}

template <typename T>
int launch_typed(const AttnArgs& a, const Plan& plan, const DeviceInfo& dev, cudaStream_t stream) {
  // no more CTAs than a table of full rows could give work
  const int64_t group = a.heads / a.kv_heads;
  const int64_t tiles = (a.rows * group / plan.m + a.seqs + 1) * a.kv_heads;
  const int64_t blocks = ceil_div(a.table_cols * a.block_size, KEYS) + 1;
  int ctas = plan.ctas;
  if (tiles < ctas && blocks < ctas && ceil_div(tiles * blocks, MIN_BLOCKS) < ctas)
    ctas = static_cast<int>(ceil_div(tiles * blocks, MIN_BLOCKS));
  const bool few = plan.m == 16;
  switch (plan.dp) {
    case 32:
      return few ? launch_shape<T, Shape<32, 1, 4, 8>>(a, dev, ctas, stream)
                 : launch_shape<T, Shape<32, 4, 2, 8>>(a, dev, ctas, stream);
    case 64:
      return few ? launch_shape<T, Shape<64, 1, 4, 6>>(a, dev, ctas, stream)
                 : launch_shape<T, Shape<64, 4, 2, 8>>(a, dev, ctas, stream);
    default:
      return few ? launch_shape<T, Shape<128, 1, 4, 3>>(a, dev, ctas, stream)
                 : launch_shape<T, Shape<128, 4, 2, 5>>(a, dev, ctas, stream);
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
         on_grid(a.q, 2, {a.sq_t, a.sq_h});
}

int64_t attention_tree_workspace_bytes(const AttnArgs& a, const DeviceInfo& dev) {
  const Plan plan = plan_for(a, dev.sm_count);
  return COUNTER_BYTES + 4ll * 2 * plan.ctas * plan.m * (plan.dp + 2);
}

int launch_attention_tree(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t need = attention_tree_workspace_bytes(a, dev);
  if (a.workspace == nullptr || a.workspace_bytes < need)
    return set_error(KF_ERR_WORKSPACE, "tree attention needs " + std::to_string(need) + " bytes of workspace; got " +
                                           std::to_string(a.workspace == nullptr ? 0 : a.workspace_bytes));
  const Plan plan = plan_for(a, dev.sm_count);
  if (plan.ctas > COUNTER_BYTES / 4) return set_error(KF_ERR_UNSUPPORTED, "tree attention: too many SMs");
  return a.dtype == KF_FP16 ? launch_typed<__half>(a, plan, dev, stream) : launch_typed<__nv_bfloat16>(a, plan, dev, stream);
}

}  // namespace kf
