// Penalties for repeated tokens, biases and grammar masks on rows of logits:
//
//   x = logits[r][v], n = times that v stands in the answered part of r's history
//   v in the history at all:  x > 0 ? x / repetition : x * repetition
//   n > 0:                    x - (frequency * n + presence)
//   v in r's list of biases:  x + its value (of the last entry that names v)
//   v's bit in r's mask is 0: -infinity
//
// in fp32, rounded once. Bound by the bytes of the logits, read and written once.
// A block takes one chunk of one row: it starts its loads of the logits, counts
// the chunk's tokens in shared memory while they are on the way (each block reads
// the row's whole history, which is short beside its logits and comes from L2), and
// applies the counts as it writes. Counts are whole numbers and the last of several
// biases is found by its place, so no result depends on the order of the atomics.
// Rows start where they start: chunks and vectors lie on the 16-byte grid of
// memory, with single elements at a row's two ends.
#include <cuda.h>

#include <type_traits>

#include "kf_common.cuh"
#include "kf_internal.h"

namespace kf {
namespace {

constexpr int LOGITS_THREADS = 512;
constexpr uint32_t IN_PROMPT = 0x80000000u;  // beside the count of answered occurrences

template <typename T, int VE>
struct alignas(sizeof(T) * VE) Piece {
  T e[VE];
};

template <typename T, int VE, int EACH>
__global__ void __launch_bounds__(LOGITS_THREADS)
    logits_kernel(const __grid_constant__ kf_logits_args p, int chunks) {
  constexpr int CHUNK = LOGITS_THREADS * EACH * VE;
  extern __shared__ __align__(16) uint32_t shared[];
  const int tid = threadIdx.x;
  const long long row = blockIdx.x / chunks;
  const int vocab = static_cast<int>(p.vocab);
  const T* const in = static_cast<const T*>(p.logits) + row * p.s_row;
  T* const out = static_cast<T*>(p.out) + row * p.so_row;
  // Places count from the 16-byte boundary at or before the row: token v has place v + lead.
  const int lead = VE > 1 ? static_cast<int>(reinterpret_cast<uintptr_t>(in) / sizeof(T) % VE) : 0;
  const int first = static_cast<int>(blockIdx.x % chunks) * CHUNK;  // place
  const int span = min(CHUNK, vocab + lead - first);                // places of this chunk, up to the row's end
  if (span <= 0) return;

  Piece<T, VE> x[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int at = (j * LOGITS_THREADS + tid) * VE, v = first + at - lead;
    if (at >= span) continue;
    if (v >= 0 && v + VE <= vocab) {
      x[j] = *reinterpret_cast<const Piece<T, VE>*>(in + v);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (v + i >= 0 && v + i < vocab) x[j].e[i] = in[v + i];
    }
  }

  const bool counted = p.tokens != nullptr, biased = p.bias_tokens != nullptr;
  uint32_t* const counts = shared;
  uint32_t* const biases = shared + (counted ? CHUNK : 0);  // place in the list + 1, of a token's last entry
  if (counted || biased) {
    for (int i = tid * 4; i < span; i += LOGITS_THREADS * 4) {  // (a chunk is a multiple of four)
      if (counted) *reinterpret_cast<uint4*>(counts + i) = make_uint4(0, 0, 0, 0);
      if (biased) *reinterpret_cast<uint4*>(biases + i) = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    if (counted) {
      const int* const ids = p.tokens + row * p.st_row;
      const int most = static_cast<int>(p.token_cols);
      const int len = min(max(__ldg(p.token_lens + row), 0), most);
      const int prompt = p.prompt_lens != nullptr ? __ldg(p.prompt_lens + row) : 0;
#pragma unroll 4
      for (int i = tid; i < len; i += LOGITS_THREADS) {
        const int v = __ldg(ids + i);
        if (v < 0 || v >= vocab) continue;
        const int at = v + lead - first;
        if (at >= 0 && at < span) {
          if (i < prompt) atomicOr(counts + at, IN_PROMPT);
          else atomicAdd(counts + at, 1u);
        }
      }
    }
    if (biased) {
      const int* const ids = p.bias_tokens + row * p.sb_row;
      for (int i = tid; i < static_cast<int>(p.bias_cols); i += LOGITS_THREADS) {
        const int v = __ldg(ids + i);
        if (v < 0 || v >= vocab) continue;
        const int at = v + lead - first;
        if (at >= 0 && at < span) atomicMax(biases + at, static_cast<uint32_t>(i) + 1u);
      }
    }
    __syncthreads();
  }
  const float repetition = counted && p.repetition != nullptr ? __ldg(p.repetition + row) : 1.0f;
  const float frequency = counted && p.frequency != nullptr ? __ldg(p.frequency + row) : 0.0f;
  const float presence = counted && p.presence != nullptr ? __ldg(p.presence + row) : 0.0f;
  const float* const values = biased ? p.bias_values + row * p.sv_row : nullptr;
  const uint32_t* mask = nullptr;
  if (p.allowed != nullptr) {
    const long long which = p.allowed_rows != nullptr ? __ldg(p.allowed_rows + row) : row;
    if (which >= 0 && which < p.masks) mask = reinterpret_cast<const uint32_t*>(p.allowed) + which * p.sa_row;
  }

#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int at = (j * LOGITS_THREADS + tid) * VE, v = first + at - lead;
    if (at >= span) continue;
    uint32_t n[VE] = {}, b[VE] = {};
    if (counted) {
      if constexpr (VE % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VE; i += 4) *reinterpret_cast<uint4*>(n + i) = *reinterpret_cast<const uint4*>(counts + at + i);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) n[i] = counts[at + i];
      }
    }
    if (biased) {
      if constexpr (VE % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VE; i += 4) *reinterpret_cast<uint4*>(b + i) = *reinterpret_cast<const uint4*>(biases + at + i);
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) b[i] = biases[at + i];
      }
    }
    const bool whole = v >= 0 && v + VE <= vocab;
    uint32_t bits = 0xffffffffu;
    if (mask != nullptr) {
      // VE bits from bit v on: of one word, or of two
      const int from = max(v, 0), to = min(v + VE, vocab) - 1;
      const uint32_t low = __ldg(mask + (from >> 5)), high = (from >> 5) != (to >> 5) ? __ldg(mask + (to >> 5)) : 0u;
      bits = __funnelshift_r(low, high, from & 31) << (from - v);
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      if (!whole && (v + i < 0 || v + i >= vocab)) continue;
      if ((n[i] | b[i]) != 0) {
        float f = to_f32(x[j].e[i]);
        if (n[i] != 0) {
          f = f > 0.0f ? f / repetition : f * repetition;
          const uint32_t times = n[i] & ~IN_PROMPT;
          if (times != 0) f -= fmaf(frequency, static_cast<float>(times), presence);
        }
        if (b[i] != 0) f += __ldg(values + (b[i] - 1));
        x[j].e[i] = from_f32<T>(f);
      }
      if ((bits >> i & 1u) == 0) x[j].e[i] = from_f32<T>(__int_as_float(0xff800000));
      if (!whole) out[v + i] = x[j].e[i];
    }
    if (whole) *reinterpret_cast<Piece<T, VE>*>(out + v) = x[j];
  }
}

template <typename T, int VE, int EACH>
int launch_chunks(const kf_logits_args& a, cudaStream_t stream) {
  constexpr int CHUNK = LOGITS_THREADS * EACH * VE;
  const int64_t chunks = ceil_div(a.vocab + VE - 1, CHUNK), blocks = chunks * a.rows;
  if (blocks > 0x7fffffffll) return set_error(KF_ERR_UNSUPPORTED, "logits beyond the grid");
  const int smem = CHUNK * 4 * ((a.tokens != nullptr) + (a.bias_tokens != nullptr));
  const auto kernel = logits_kernel<T, VE, EACH>;
  if (smem > 48 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (err != cudaSuccess) return cuda_error(err, "attributes(logits)");
  }
  kernel<<<static_cast<unsigned>(blocks), LOGITS_THREADS, smem, stream>>>(a, static_cast<int>(chunks));
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(logits)");
}

template <typename T, int VE>
int launch_typed(const kf_logits_args& a, const DeviceInfo& dev, cudaStream_t stream) {
  // Chunks of 8192 tokens, or the smallest where those would leave SMs without a block.
  constexpr int EACH = 16 / VE;
  if (a.rows * ceil_div(a.vocab, 8192) >= dev.sm_count) return launch_chunks<T, VE, EACH>(a, stream);
  return launch_chunks<T, VE, VE == 1 ? 4 : 1>(a, stream);
}

template <typename T>
int pick(const kf_logits_args& a, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int VE = 16 / static_cast<int>(sizeof(T));
  const auto off = [](const void* x) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(x) / sizeof(T) % VE); };
  // Vectors where every row of the output lies as its logits do.
  const bool alike = off(a.logits) == off(a.out) && (a.rows <= 1 || (a.s_row - a.so_row) % VE == 0);
  return alike ? launch_typed<T, VE>(a, dev, stream) : launch_typed<T, 1>(a, dev, stream);
}

}  // namespace

int launch_logits(const kf_logits_args& a, const DeviceInfo& dev, cudaStream_t stream) {
  switch (a.dtype) {
    case KF_FP16: return pick<__half>(a, dev, stream);
    case KF_BF16: return pick<__nv_bfloat16>(a, dev, stream);
    default: return pick<float>(a, dev, stream);
  }
}

}  // namespace kf
