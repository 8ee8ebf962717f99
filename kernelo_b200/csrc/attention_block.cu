// Attention on tiles of 16 or 64 rows in fp32 arithmetic: packed prompts and paged
// caches, every type, stride, head dimension up to 256 and mask. It takes what the
// tensor-core kernels do not: fp32 above all, whose products a 16-bit matrix
// instruction would round.
//
//   s = scale log2(e) q k^T,  m' = max(m, max s),  p = 2^(s - m'),
//   l = l 2^(m - m') + sum p,  O = O 2^(m - m') + p v
//
// The rows of a tile are (token, head) pairs of one request and one key head, so
// that all heads of a group read a key once. A CTA of 128 threads keeps the tile's
// queries and two blocks of 32 keys in shared memory as fp32, one of them on its
// way (cp.async; 16-bit elements are widened through registers) while the other is
// used; a thread computes the scores of an eighth of the rows x 2 keys and the sums
// of the same rows x DP / 16 columns, two values to an instruction (fma.rn.f32x2).
// The weights cross the threads of a warp through shared memory. Where tiles are
// few, up to 16 CTAs of a cluster share a tile's keys and add their sums in the
// order of the keys through distributed shared memory.
//
// A row that comes out non-finite where a key of its blocks that it does not see holds
// something not finite (0 x infinity) is computed again from the keys that it sees.
//
// The multiply-adds bound it. One fp32 prompt of 2047 tokens, 28 heads to 4, 80
// elements: 710 us, 26 TFLOP/s with the FMA pipe busy half of the time (two warps
// to a scheduler; a warp to a row and head, each reading its keys itself, took
// 11920). 4 caches of up to 16384 keys, 16 heads to 4, 80 elements, one token:
// 103 us, 104 MB at 1.0 TB/s (1050 by rows; 332 on tiles of 64 rows and 8 CTAs).
#include <cuda.h>

#include <mutex>

#include "attention.cuh"

namespace kf {
namespace {

constexpr int KEYS = 32;   // of a block
constexpr int THREADS = 128;
constexpr int GROUPS = THREADS / 16;    // of 16 threads: a group has rows g, g + GROUPS, ...
constexpr int TK = KEYS / 16;           // keys of a thread
constexpr int P_PITCH = KEYS + 4;       // floats: rows of weights start on different banks
constexpr int FEW = 16, MANY = 64;      // rows of a tile
constexpr int MAX_PARTS = 16;           // CTAs of a cluster: over 8 has to be allowed

template <int ROWS, int DP>
struct Shape {
  static constexpr int PITCH = DP + 4;  // floats: 16-byte reads of 8 consecutive rows meet all banks
  static constexpr int BLOCK = KEYS * (PITCH + DP);  // floats of K and V
  static constexpr int SMEM = 4 * (ROWS * PITCH + 2 * BLOCK + ROWS * P_PITCH);
};

struct Tile {
  int request, row0, nodes;  // the request's first row, and how many
  int first;                 // (token, head) pair that the tile begins with
  int count;                 // pairs of the tile; 0: no such tile
  int stop;                  // no row sees this key or a later one
  long long first_key;
};

// Tile `g`, counted through the requests, the last rows of a request (which see
// the most keys) first. Called by a whole warp.
template <int ROWS>
__device__ __forceinline__ void find_tile(const AttnArgs& p, long long g, int lane, Tile* out) {
  const int group = static_cast<int>(p.heads / p.kv_heads);
  for (int r0 = 0; r0 <= p.seqs; r0 += 32) {
    const int r = r0 + lane;
    int begin = 0, end = 0;
    if (r <= p.seqs) request_rows(p, r, &begin, &end);
    const long long pairs = static_cast<long long>(end - begin) * group;
    const long long tiles = (pairs + ROWS - 1) / ROWS;
    long long upto = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const long long total = __shfl_sync(0xffffffffu, upto, 31);
    if (g < total) {
      if (upto > g && upto - tiles <= g) {
        long long first, length;
        request_keys(p, r, end - begin, &first, &length);
        const long long from = (upto - 1 - g) * ROWS;
        out->request = r;
        out->row0 = begin;
        out->nodes = end - begin;
        out->first = static_cast<int>(from);
        out->count = static_cast<int>(min(static_cast<long long>(ROWS), pairs - from));
        out->first_key = first;
        const int last = (out->first + out->count - 1) / group;
        long long stop = length;
        if (!p.paged && p.causal) stop = min(length, max(0ll, last + 1 + length - out->nodes));
        if (p.paged && p.mask == nullptr && r < p.seqs) stop = min(length, max(__ldg(p.context + r), 0) + last + 1ll);
        out->stop = static_cast<int>(stop);
      }
      return;
    }
    g -= total;
  }
  if (lane == 0) out->count = 0;
}

__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, bool present) {
  // nothing is read where the element is absent: zeros
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(present ? 4 : 0) : "memory");
}

template <typename T, int NE>
__device__ __noinline__ void redo_row(const AttnArgs& p, int t, int head, int from, int to, int lane) {
  if (last_unseen_nonfinite<T, NE>(p, t, head, from, to, lane) < 0) return;
  float acc[NE], m, l;
  attend_row<T, NE>(p, t, head, lane, acc, &m, &l);
  write_row<T, NE>(p, t, head, lane, acc, m, l);
}

__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <typename T, int ROWS, int DP>
__global__ void __launch_bounds__(THREADS, DP <= 64 || ROWS == FEW && DP <= 128 ? 3 : DP <= 128 ? 2 : 1)
    attention_block_kernel(const __grid_constant__ AttnArgs p, int parts) {
  using S = Shape<ROWS, DP>;
  constexpr int TR = ROWS / GROUPS;  // rows of a thread
  constexpr int CP = DP / 32;  // column pairs of a thread
  extern __shared__ __align__(16) float smem[];
  float* const qs = smem;
  float* const ring = qs + ROWS * S::PITCH;  // two blocks of K and V
  float* const ps = ring + 2 * S::BLOCK;
  __shared__ Tile tile_word;
  __shared__ uint32_t seen[2][ROWS];  // of a block: by each row,
  __shared__ uint8_t __align__(4) present[2][THREADS / 32];  // and in any page
  __shared__ int prefix[ROWS];
  __shared__ float sum_m[ROWS], sum_l[ROWS];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, tx = tid & 15, ty = tid >> 4;
  const int rank = parts > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const long long unit = blockIdx.x / parts;
  const int kv_head = static_cast<int>(unit % p.kv_heads), group = static_cast<int>(p.heads / p.kv_heads);
  const int D = static_cast<int>(p.dim);
  if (warp == 0) find_tile<ROWS>(p, unit / p.kv_heads, lane, &tile_word);
  __syncthreads();
  const Tile tile = tile_word;
  if (tile.count == 0) return;  // every CTA of the cluster

  // queries times the scale, zeros past the head and the last row
  for (int row = warp; row < ROWS; row += THREADS / 32) {
    const int pair = tile.first + row, node = pair / group, head = kv_head * group + pair - node * group;
    const bool real = row < tile.count;
    const T* q = static_cast<const T*>(p.q) + (static_cast<long long>(tile.row0) + node) * p.sq_t + head * p.sq_h;
#pragma unroll
    for (int i = 0; i < CP; ++i) {
      const int e = lane + 32 * i;
      qs[row * S::PITCH + e] = real && e < D ? to_f32(q[e]) * p.scale_log2 : 0.0f;
    }
  }
  if (tid < ROWS) {  // the keys below `prefix` are all seen
    const int node = (tile.first + tid) / group;
    int n = 0;
    if (tid < tile.count) {
      if (p.paged) {
        n = tile.request < p.seqs ? max(__ldg(p.context + tile.request), 0) : 0;
        n = min(p.mask == nullptr ? (n > 0x7fffffff - node - 1 ? 0x7fffffff : n + node + 1) : n, tile.stop);
      } else {
        // `stop` is the last row's limit; this row ends as many keys earlier as it has tokens behind it
        n = p.causal ? max(0, tile.stop - ((tile.first + tile.count - 1) / group - node)) : tile.stop;
      }
    }
    prefix[tid] = n;
  }

  float m[TR], l[TR];
  uint64_t o[TR][CP];
#pragma unroll
  for (int i = 0; i < TR; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.0f;
#pragma unroll
    for (int c = 0; c < CP; ++c) o[i][c] = 0ull;
  }
  const int blocks = (tile.stop + KEYS - 1) / KEYS, share = (blocks + parts - 1) / parts;
  const T* const k = static_cast<const T*>(p.k) + kv_head * p.sk_h;
  const T* const v = static_cast<const T*>(p.v) + kv_head * p.sv_h;
  const int first = rank * share, end = min(blocks, first + share);
  // A warp brings a fourth of a block's keys, lane x < KW that of key x: its page, or
  // -1 where there is none (0 for packed keys), and its place there.
  constexpr int KW = KEYS / (THREADS / 32);
  int page = -1, place = 0;
  auto look_up = [&](int b) {
    const int pos = b * KEYS + warp * KW + lane;
    page = -1;
    if (lane >= KW || pos >= tile.stop || b >= end) return;
    place = pos;
    page = 0;
    if (p.paged) {
      const uint32_t col = static_cast<uint32_t>(pos) / static_cast<uint32_t>(p.block_size);
      place = pos - static_cast<int>(col * static_cast<uint32_t>(p.block_size));
      page = __ldg(p.table + tile.request * p.table_stride + col);
      if (page >= p.pages) page = -1;
    }
  };
  auto fill = [&](int b, int buf) {
    float* const ks = ring + buf * S::BLOCK + warp * KW * S::PITCH;
    float* const vs = ring + buf * S::BLOCK + KEYS * S::PITCH + warp * KW * DP;
    const uint32_t has = __ballot_sync(0xffffffffu, page >= 0);
    if (lane == 0) present[buf][warp] = static_cast<uint8_t>(has);
    const long long key = tile.first_key + place;  // first_key 0 in a cache, page 0 in packed keys
    const long long ko = page >= 0 ? page * p.sk_p + key * p.sk_t : 0, vo = page >= 0 ? page * p.sv_p + key * p.sv_t : 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int x = 0; x < KW; ++x) {
        const T* const kx = k + __shfl_sync(0xffffffffu, ko, x);
        const T* const vx = v + __shfl_sync(0xffffffffu, vo, x);
#pragma unroll
        for (int i = 0; i < CP; ++i) {
          const int e = lane + 32 * i;
          const bool real = ((has >> x) & 1u) && e < D;
          cp_async_4(smem_u32(ks + x * S::PITCH + e), real ? kx + e : p.q, real);
          cp_async_4(smem_u32(vs + x * DP + e), real ? vx + e : p.q, real);
        }
      }
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        T raw[KW][CP];
#pragma unroll
        for (int x = 0; x < KW; ++x) {
          const T* const at = half ? v + __shfl_sync(0xffffffffu, vo, x) : k + __shfl_sync(0xffffffffu, ko, x);
#pragma unroll
          for (int i = 0; i < CP; ++i) {
            const int e = lane + 32 * i;
            raw[x][i] = ((has >> x) & 1u) && e < D ? at[e] : from_f32<T>(0.0f);
          }
        }
#pragma unroll
        for (int x = 0; x < KW; ++x) {
#pragma unroll
          for (int i = 0; i < CP; ++i) (half ? vs + x * DP : ks + x * S::PITCH)[lane + 32 * i] = to_f32(raw[x][i]);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (tid >= ROWS) return;  // what each row sees of the block
    const int row = tid;
    const long long below = static_cast<long long>(prefix[row]) - b * KEYS;
    uint32_t bits = below >= KEYS ? 0xffffffffu : below > 0 ? (1u << below) - 1u : 0u;
    if (p.mask != nullptr && below < KEYS && row < tile.count) {
      const int node = (tile.first + row) / group;
      const unsigned long long* words = p.mask + (static_cast<long long>(tile.row0) + node) * p.mask_words;
      if (below <= 0) {  // the mask's bits from -below on
        const long long w = -below >> 6;
        const int sh = static_cast<int>(-below & 63);
        unsigned long long x = w < p.mask_words ? __ldg(words + w) >> sh : 0ull;
        if (sh > 32 && w + 1 < p.mask_words) x |= __ldg(words + w + 1) << (64 - sh);
        bits |= static_cast<uint32_t>(x);
      } else if (p.mask_words > 0) {
        bits |= static_cast<uint32_t>(__ldg(words) << below);
      }
    }
    seen[buf][row] = bits;
  };
  __syncthreads();  // prefix
  look_up(first);
  if (first < end) fill(first, 0);
  look_up(first + 1);
  for (int b = first; b < end; ++b) {
    const int buf = (b - first) & 1;
    if (b + 1 < end) {
      fill(b + 1, buf ^ 1);
      look_up(b + 2);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
    } else {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const float* const ks = ring + buf * S::BLOCK;
    const float* const vs = ks + KEYS * S::PITCH;

    uint64_t s[TR][TK];  // sums of even and of odd elements
#pragma unroll
    for (int i = 0; i < TR; ++i) {
#pragma unroll
      for (int j = 0; j < TK; ++j) s[i][j] = 0ull;
    }
#pragma unroll 2
    for (int e = 0; e < D; e += 4) {
      ulonglong2 kf[TK];
#pragma unroll
      for (int j = 0; j < TK; ++j) kf[j] = *reinterpret_cast<const ulonglong2*>(ks + (tx + 16 * j) * S::PITCH + e);
#pragma unroll
      for (int i = 0; i < TR; ++i) {
        const ulonglong2 qf = *reinterpret_cast<const ulonglong2*>(qs + (ty + GROUPS * i) * S::PITCH + e);
#pragma unroll
        for (int j = 0; j < TK; ++j) s[i][j] = f2_fma(qf.x, kf[j].x, s[i][j]);
#pragma unroll
        for (int j = 0; j < TK; ++j) s[i][j] = f2_fma(qf.y, kf[j].y, s[i][j]);
      }
    }
    const uint32_t here = *reinterpret_cast<const uint32_t*>(present[buf]);
#pragma unroll
    for (int i = 0; i < TR; ++i) {
      const int row = ty + GROUPS * i;
      const uint32_t bits = seen[buf][row] & here;
      float x[TK], top = m[i];
#pragma unroll
      for (int j = 0; j < TK; ++j) {
        const float2 two = f2_unpack(s[i][j]);
        x[j] = (bits >> (tx + 16 * j)) & 1u ? two.x + two.y : -INFINITY;
        top = fmaxf(top, x[j]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float base = top == -INFINITY ? 0.0f : top;
      const float fix = ex2_ftz(m[i] - base);
      m[i] = top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < TK; ++j) {
        x[j] = ex2_ftz(x[j] - base);
        ps[row * P_PITCH + tx + 16 * j] = x[j];
        sum += x[j];
      }
      l[i] = fmaf(l[i], fix, sum);  // of this thread's keys: joined at the end
      const uint64_t both = f2_splat(fix);
#pragma unroll
      for (int c = 0; c < CP; ++c) o[i][c] = f2_mul(o[i][c], both);
    }
    __syncwarp();
#pragma unroll 1
    for (int key = 0; key < KEYS; key += 4) {
      float4 w[TR];
#pragma unroll
      for (int i = 0; i < TR; ++i) w[i] = *reinterpret_cast<const float4*>(ps + (ty + GROUPS * i) * P_PITCH + key);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint64_t vf[CP];
#pragma unroll
        for (int c = 0; c < CP; ++c) vf[c] = *reinterpret_cast<const uint64_t*>(vs + (key + x) * DP + 2 * tx + 32 * c);
#pragma unroll
        for (int i = 0; i < TR; ++i) {
          const uint64_t both = f2_splat(x == 0 ? w[i].x : x == 1 ? w[i].y : x == 2 ? w[i].z : w[i].w);
#pragma unroll
          for (int c = 0; c < CP; ++c) o[i][c] = f2_fma(both, vf[c], o[i][c]);
        }
      }
    }
    __syncthreads();  // the block has been used
  }

  // sums to shared memory (in place of the queries), then a warp per row joins the parts
#pragma unroll
  for (int i = 0; i < TR; ++i) {
    const int row = ty + GROUPS * i;
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    if (tx == 0) {
      sum_m[row] = m[i];
      sum_l[row] = l[i];
    }
#pragma unroll
    for (int c = 0; c < CP; ++c) *reinterpret_cast<uint64_t*>(qs + row * S::PITCH + 2 * tx + 32 * c) = o[i][c];
  }
  if (parts > 1) cluster_sync_all(); else __syncthreads();
  const int step = THREADS / 32 * parts;
  for (int row = warp * parts + rank; row < tile.count; row += step) {
    float acc[CP], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < CP; ++i) acc[i] = 0.0f;
    for (int part = 0; part < parts; ++part) {
      const uint32_t at_m = parts > 1 ? mapa_shared(smem_u32(&sum_m[row]), part) : smem_u32(&sum_m[row]);
      const uint32_t at_l = parts > 1 ? mapa_shared(smem_u32(&sum_l[row]), part) : smem_u32(&sum_l[row]);
      const uint32_t at_o = (parts > 1 ? mapa_shared(smem_u32(qs), part) : smem_u32(qs)) + 4 * (row * S::PITCH + lane);
      const float pm = load_cluster(at_m), pl = load_cluster(at_l);
      const float higher = fmaxf(top, pm), base = higher == -INFINITY ? 0.0f : higher;
      const float fix = ex2_ftz(top - base), take = ex2_ftz(pm - base);
      sum = fmaf(sum, fix, pl * take);
#pragma unroll
      for (int i = 0; i < CP; ++i) acc[i] = fmaf(acc[i], fix, load_cluster(at_o + 128 * i) * take);
      top = higher;
    }
    bool fine = true;
#pragma unroll
    for (int i = 0; i < CP; ++i) fine = fine && fabsf(acc[i]) < INFINITY;
    const int pair = tile.first + row, node = pair / group, head = kv_head * group + pair - node * group;
    write_row<T, CP>(p, tile.row0 + node, head, lane, acc, top, sum);
    if (__any_sync(0xffffffffu, suspect(fine, sum)))
      redo_row<T, CP>(p, tile.row0 + node, head, prefix[row], tile.stop, lane);
  }
  __syncwarp();
  if (parts > 1) cluster_sync_all();  // the sums have been read
}

int64_t max_i64(int64_t a, int64_t b) { return a > b ? a : b; }

// Every request's last tile may be short, and so may that of the rows behind the last request.
int64_t tiles_at_most(const AttnArgs& a, int rows) { return a.rows * (a.heads / a.kv_heads) / rows + a.seqs + 1; }

template <typename T, int ROWS, int DP>
int launch_shape(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  using S = Shape<ROWS, DP>;
  static std::once_flag once;
  static cudaError_t attr = cudaSuccess;
  std::call_once(once, [] {
    const auto kernel = attention_block_kernel<T, ROWS, DP>;
    attr = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (attr == cudaSuccess) attr = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (attr != cudaSuccess) return cuda_error(attr, "attention block attributes");
  const int64_t pairs = a.rows * (a.heads / a.kv_heads);
  // tiles of requests of equal length, for the number of CTAs to a tile
  const int64_t usual = max_i64(a.seqs, 1) * ceil_div(ceil_div(pairs, max_i64(a.seqs, 1)), ROWS) * a.kv_heads;
  // 16 CTAs only where two fit on an SM: a cluster lies within the SMs of one processing cluster
  const int most = 2 * S::SMEM <= 220 * 1024 ? MAX_PARTS : MAX_PARTS / 2;
  // CTAs to a tile: up to two for every SM, or four where each has four blocks of keys or more.
  // One token each, fp32: a cache of 14618 keys, 32 heads to 8 of 112 elements, 146 us (683 with
  // two CTAs to a tile at most); four of up to 4000 keys, 32 heads of 64, 124 us (180 with two
  // CTAs for every SM). Five prompts of up to 169 tokens, 7 heads to 1 of 128 elements, 35 us
  // (42 with four for every SM, 54 with none of under four blocks).
  const int64_t room = a.paged ? a.table_cols * a.block_size : ceil_div(a.keys, max_i64(a.seqs, 1));
  int parts = 1;
  while (parts < most && usual * parts * 2 <= (parts * 2 * 4 * KEYS <= room ? 4 : 2) * dev.sm_count) parts *= 2;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(tiles_at_most(a, ROWS) * a.kv_heads * parts));
  config.blockDim = dim3(THREADS);
  config.dynamicSmemBytes = S::SMEM;
  config.stream = stream;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = static_cast<unsigned>(parts);
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = parts > 1 ? 1 : 0;
  const cudaError_t err = cudaLaunchKernelEx(&config, attention_block_kernel<T, ROWS, DP>, a, parts);
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(attention_block)");
}

template <typename T, int ROWS>
int launch_rows(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  if (a.dim <= 32) return launch_shape<T, ROWS, 32>(a, dev, stream);
  if (a.dim <= 64) return launch_shape<T, ROWS, 64>(a, dev, stream);
  if (a.dim <= 96) return launch_shape<T, ROWS, 96>(a, dev, stream);
  if (a.dim <= 128) return launch_shape<T, ROWS, 128>(a, dev, stream);
  return launch_shape<T, ROWS, 256>(a, dev, stream);
}

template <typename T>
int launch_typed(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  // Short tiles where a request has no more rows to a key head on average. 32 caches of up
  // to 1000 keys, 32 heads to 8 of 128 elements: one to five tokens each 143 us (183 on
  // tiles of 32 rows, 280 on 64), one token each 105 (142 with two CTAs for every SM, where
  // tiles of 32 rows took 179 and of 8 rows 133).
  if (a.rows * (a.heads / a.kv_heads) <= FEW * a.seqs) return launch_rows<T, FEW>(a, dev, stream);
  return launch_rows<T, MANY>(a, dev, stream);
}

}  // namespace

int launch_attention_block(const AttnArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  if (a.rows * (a.heads / a.kv_heads) > 0x7fffff00ll || tiles_at_most(a, FEW) * a.kv_heads > 0x7fffffffll / MAX_PARTS)
    return set_error(KF_ERR_UNSUPPORTED, "attention: rows x heads beyond the grid");
  switch (a.dtype) {
    case KF_FP16: return launch_typed<__half>(a, dev, stream);
    case KF_BF16: return launch_typed<__nv_bfloat16>(a, dev, stream);
    default: return launch_typed<float>(a, dev, stream);
  }
}

}  // namespace kf
