// Penalties for repeated tokens, biases and grammar masks on rows of logits:
//
//   x = logits[r][v], n = times that v stands in the answered part of r's history
//   v in the history at all:  x > 0 ? x / repetition : x * repetition
//   n > 0:                    x - (frequency * n + presence)
//   v in r's list of biases:  x + its value (of the last entry that names v)
//   v's bit in r's mask is 0: -infinity
//
// in fp32, rounded once. Bound by the bytes of the logits, read and written once.
// A block takes one chunk of one row: it starts its loads of the logits and of the
// history, counts the chunk's tokens in shared memory (each block reads the row's
// whole history, which is short beside its logits and comes from L2), and applies the
// counts as it writes. Biases are few: they are added behind the others, each by
// the thread that has its last entry. Counts are whole numbers and the last of several
// biases is found by its place: no result depends on the order of the atomics.
// Rows start where they start: chunks and vectors lie on the 16-byte grid of
// memory, with single elements at a row's two ends.
// 512 rows of 32000 in fp32: 18 us without anything to do, 19 with masks, 28 with histories of 1024 tokens, 25 with 32
// biases, 41 with all three and histories of up to 2048 (a copy's rate: 20); in bf16 9, 10, 21, 18 and 28. What counts and
// biases add is the instructions of the tokens that they touch and waits at the block's barriers.
#include <cuda.h>

#include "kf_common.cuh"
#include "kf_internal.h"
#include "packed.cuh"

namespace kf {
namespace {

constexpr int LOGITS_THREADS = 512;
// A token's word: its answered occurrences, whether the prompt has it, and whether a bias awaits it.
constexpr uint32_t IN_PROMPT = 0x80000000u, BIASED = 0x40000000u, TIMES = 0x3fffffffu;
constexpr int IDS_EACH = 4;  // tokens of the history that a thread holds at a time

// The vector with the elements whose bit of `off` is set at -infinity.
template <typename T, int VE>
__device__ __forceinline__ void mask_out(Vec<T, VE>& x, uint32_t off) {
#pragma unroll
  for (int i = 0; i < Vec<T, VE>::WORDS; ++i) {
    if constexpr (Vec<T, VE>::PAIRS) {
      constexpr uint32_t INF = DType<T>::code == KF_BF16 ? 0xff80ff80u : 0xfc00fc00u;
      const uint32_t gone = ((off >> 2 * i & 1u) != 0 ? 0xffffu : 0u) | ((off >> (2 * i + 1) & 1u) != 0 ? 0xffff0000u : 0u);
      x.w[i] = (x.w[i] & ~gone) | (INF & gone);
    } else {
      if ((off >> i & 1u) != 0) x.w[i] = from_f32<T>(__int_as_float(0xff800000));
    }
  }
}

// The elements of a vector that lie in a row of `vocab`, its first being element v.
template <typename T, int VE>
__device__ __forceinline__ void load_part(const T* row, int v, int vocab, Vec<T, VE>& x) {
  float f[VE];
#pragma unroll
  for (int i = 0; i < VE; ++i) f[i] = v + i >= 0 && v + i < vocab ? to_f32(row[v + i]) : 0.0f;
  narrow<T, VE>(f, x);
}
template <typename T, int VE>
__device__ __forceinline__ void store_part(T* row, int v, int vocab, const Vec<T, VE>& x) {
  float f[VE];
  widen<T, VE>(x, f);
#pragma unroll
  for (int i = 0; i < VE; ++i)
    if (v + i >= 0 && v + i < vocab) row[v + i] = from_f32<T>(f[i]);
}

struct Penalties {
  float repetition, inverse, frequency, presence;
  // x / repetition as a product: off by one more half unit of fp32, and a division is a dozen instructions
  __device__ __forceinline__ float apply(float x, uint32_t word) const {
    const uint32_t times = word & TIMES;
    const float less = times != 0 ? fmaf(frequency, static_cast<float>(times), presence) : 0.0f;
    return fmaf(x, x > 0.0f ? inverse : repetition, -less);
  }
};

template <typename T, int VE, int EACH>
__global__ void __launch_bounds__(LOGITS_THREADS, 3)
    logits_kernel(const __grid_constant__ kf_logits_args p, int chunks, int aligned) {
  constexpr int CHUNK = LOGITS_THREADS * EACH * VE;
  static_assert(CHUNK / 32 <= 2 * LOGITS_THREADS && 32 % VE == 0, "two mask words a thread at most, whole vectors in a word");
  extern __shared__ __align__(16) uint32_t words[];  // of the chunk's places, where there is a history or a list of biases
  __shared__ uint32_t allowed[CHUNK / 32];           // the mask's bits of the chunk's places
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

  // What the rest waits for, all at once.
  using V = Vec<T, VE>;
  V x[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int at = (j * LOGITS_THREADS + tid) * VE, v = first + at - lead;
    if (at >= span) continue;
    if (v >= 0 && v + VE <= vocab) x[j] = load_once<V>(in + v);
    else load_part<T, VE>(in, v, vocab, x[j]);
  }
  const uint32_t* mask = nullptr;
  if (p.allowed != nullptr) {
    const long long which = p.allowed_rows != nullptr ? __ldg(p.allowed_rows + row) : row;
    if (which >= 0 && which < p.masks) mask = reinterpret_cast<const uint32_t*>(p.allowed) + which * p.sa_row;
  }
  // Bit i of a word of places is bit `turn + i` of two words of tokens side by side (-1 and those past the last: none).
  const int turn = (first - lead) & 31, mask_words = (vocab + 31) >> 5;
  uint32_t bits[2] = {0, 0};
  if (mask != nullptr) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int word = tid + k * LOGITS_THREADS, of = ((first - lead) >> 5) + word;
      if (word * 32 >= span) continue;
      const uint32_t low = of >= 0 ? __ldg(mask + of) : 0u;
      bits[k] = turn == 0 ? low : __funnelshift_r(low, of + 1 < mask_words ? __ldg(mask + of + 1) : 0u, turn);
    }
  }
  const bool counted = p.tokens != nullptr, biased = p.bias_tokens != nullptr;
  const int* const ids = p.tokens + row * p.st_row;
  const int most = counted ? static_cast<int>(p.token_cols) : 0;
  int held[IDS_EACH];
  const auto place = [&](int from, int k) { return from + (aligned ? tid * IDS_EACH + k : k * LOGITS_THREADS + tid); };
  const auto load_ids = [&](int from, int end) {
    if (aligned) {
      int4 four = make_int4(-1, -1, -1, -1);
      if (place(from, 0) < end) four = __ldg(reinterpret_cast<const int4*>(ids + place(from, 0)));  // whole fours lie in a row
      held[0] = four.x, held[1] = four.y, held[2] = four.z, held[3] = four.w;
    } else {
#pragma unroll
      for (int k = 0; k < IDS_EACH; ++k) held[k] = place(from, k) < end ? __ldg(ids + place(from, k)) : -1;
    }
  };
  load_ids(0, most);
  const int len = counted ? min(max(__ldg(p.token_lens + row), 0), most) : 0;
  const int prompt = counted && p.prompt_lens != nullptr ? __ldg(p.prompt_lens + row) : 0;
  Penalties penalties;
  penalties.repetition = counted && p.repetition != nullptr ? __ldg(p.repetition + row) : 1.0f;
  penalties.inverse = 1.0f / penalties.repetition;
  penalties.frequency = counted && p.frequency != nullptr ? __ldg(p.frequency + row) : 0.0f;
  penalties.presence = counted && p.presence != nullptr ? __ldg(p.presence + row) : 0.0f;

  // A token's word in this chunk, or null.
  const auto word_of = [&](int v) -> uint32_t* {
    if (v < 0 || v >= vocab) return nullptr;
    const int at = v + lead - first;
    return at >= 0 && at < span ? words + at : nullptr;
  };
  const int* const bias_ids = p.bias_tokens + row * p.sb_row;
  const int n_biases = biased ? static_cast<int>(p.bias_cols) : 0;
  // Read anew in each pass, and found through the words: held in registers, or sought by a warp for short lists, they take
  // registers that the stream needs (42 of a thread; a few spilled, and 512 rows in fp32 stream in 21 us, not 18).
  const auto each_bias = [&](const auto& f) {
    for (int i = tid, k = 0; i < n_biases; i += LOGITS_THREADS, ++k) f(i, k, __ldg(bias_ids + i));
  };
  uint32_t last = 0;  // entries that count, of up to 32 of this thread's
  if (counted || biased) {
    for (int i = tid * 4; i < span; i += LOGITS_THREADS * 4)  // (a chunk is a multiple of four)
      *reinterpret_cast<uint4*>(words + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (biased) {
      each_bias([&](int i, int, int v) {
        if (uint32_t* const w = word_of(v)) atomicMax(w, static_cast<uint32_t>(i) + 1u);
      });
      __syncthreads();
      each_bias([&](int i, int k, int v) {
        if (uint32_t* const w = word_of(v)) last |= (*w == static_cast<uint32_t>(i) + 1u ? 1u : 0u) << k;
      });
      __syncthreads();
      each_bias([&](int, int k, int v) {
        if ((last >> k & 1u) != 0) *word_of(v) = BIASED;
      });
      __syncthreads();
    }
    constexpr int BATCH = IDS_EACH * LOGITS_THREADS;
    for (int from = 0; from < len; from += BATCH) {
      if (from > 0) load_ids(from, len);
#pragma unroll
      for (int k = 0; k < IDS_EACH; ++k) {
        uint32_t* const w = place(from, k) < len ? word_of(held[k]) : nullptr;
        if (w == nullptr) continue;
        if (place(from, k) < prompt) atomicOr(w, IN_PROMPT);
        else atomicAdd(w, 1u);
      }
    }
  }
  if (mask != nullptr) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (tid + k * LOGITS_THREADS < CHUNK / 32) allowed[tid + k * LOGITS_THREADS] = bits[k];
  }
  __syncthreads();

#pragma unroll
  for (int j = 0; j < EACH; ++j) {
    const int at = (j * LOGITS_THREADS + tid) * VE, v = first + at - lead;
    if (at >= span) continue;
    if (counted || biased) {
      uint32_t n[VE], any = 0;
      if constexpr (VE % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VE; i += 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(words + at + i);
          n[i] = w.x, n[i + 1] = w.y, n[i + 2] = w.z, n[i + 3] = w.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) n[i] = words[at + i];
      }
#pragma unroll
      for (int i = 0; i < VE; ++i) any |= n[i];
      if (any != 0) {
        float f[VE];
        widen<T, VE>(x[j], f);
#pragma unroll
        for (int i = 0; i < VE; ++i)  // a biased one stays as it is for the thread that has its bias
          if (n[i] != 0 && (n[i] & BIASED) == 0) f[i] = penalties.apply(f[i], n[i]);
        narrow<T, VE>(f, x[j]);
      }
    }
    if (mask != nullptr) mask_out<T, VE>(x[j], ~(allowed[at >> 5] >> (at & 31)));
    if (v >= 0 && v + VE <= vocab) *reinterpret_cast<V*>(out + v) = x[j];
    else store_part<T, VE>(out, v, vocab, x[j]);
  }
  if (!biased) return;
  __syncthreads();  // the block's stores, which the biased tokens passed through unchanged or masked
  each_bias([&](int i, int k, int v) {
    if ((last >> k & 1u) == 0) return;
    const int at = v + lead - first;
    if (mask != nullptr && (allowed[at >> 5] >> (at & 31) & 1u) == 0) return;
    const uint32_t n = words[at] & ~BIASED;
    const float f = to_f32(in[v]);
    out[v] = from_f32<T>((n != 0 ? penalties.apply(f, n) : f) + __ldg(p.bias_values + row * p.sv_row + i));
  });
}

template <typename T, int VE, int EACH>
int launch_chunks(const kf_logits_args& a, cudaStream_t stream) {
  constexpr int CHUNK = LOGITS_THREADS * EACH * VE;
  const int64_t chunks = ceil_div(a.vocab + VE - 1, CHUNK), blocks = chunks * a.rows;
  if (blocks > 0x7fffffffll) return set_error(KF_ERR_UNSUPPORTED, "logits beyond the grid");
  const int smem = a.tokens != nullptr || a.bias_tokens != nullptr ? CHUNK * 4 : 0;
  if constexpr (CHUNK * 4 > 48 * 1024) {
    const cudaError_t err =
        cudaFuncSetAttribute(logits_kernel<T, VE, EACH>, cudaFuncAttributeMaxDynamicSharedMemorySize, CHUNK * 4);
    if (err != cudaSuccess) return cuda_error(err, "attributes(logits)");
  }
  const int aligned = reinterpret_cast<uintptr_t>(a.tokens) % 16 == 0 && a.st_row % 4 == 0 && a.token_cols % 4 == 0;
  logits_kernel<T, VE, EACH><<<static_cast<unsigned>(blocks), LOGITS_THREADS, smem, stream>>>(a, static_cast<int>(chunks),
                                                                                           aligned);
  const cudaError_t err = cudaGetLastError();
  return err == cudaSuccess ? KF_OK : cuda_error(err, "launch(logits)");
}

template <typename T, int VE>
int launch_typed(const kf_logits_args& a, const DeviceInfo& dev, cudaStream_t stream) {
  // Four vectors a thread, or the smallest chunk where those would leave SMs without a block: 512 rows of 32000 with a
  // history of 1024 take 21.5 us in bf16 in chunks of 16384 (8192: 25.6) and 27.8 in fp32 in chunks of 8192 (16384: 28.9).
  constexpr int EACH = VE == 1 ? 16 : 4;
  if (a.rows * ceil_div(a.vocab, LOGITS_THREADS * EACH * VE) >= dev.sm_count) return launch_chunks<T, VE, EACH>(a, stream);
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
