// Logits of a batch before the softmax: penalties for tokens already seen, a sparse bias and a
// grammar mask, in one pass over [rows][vocab].
//
// Bound by HBM: the logits are read once and written once. A CTA owns a stretch of one row's
// vocabulary and counts, in shared memory, the occurrences of its tokens in the row's history (it
// reads the whole history, which the row's other CTAs read too, from L2; integer atomics, so the
// order does not matter). Counting per stretch needs no workspace and no second launch. Tokens are
// listed as they are first met. The pass over the stretch only copies and masks; the listed tokens
// are then computed again. (Looking the counters up in the pass itself sent nearly every warp through
// the penalties' divisions for a few of its 256 tokens: 67 us instead of HBM's 17 for 256 rows.)
//
// A row of odd length starts anywhere in a 16-byte granule. Stretches are therefore cut in the
// granules of the array, not of the row: position e of the stretch space of row r is token
// e - lead(r) with lead(r) = r * vocab mod (elements per granule), so that every whole granule is
// one 128-bit access; the granules that a row shares with its neighbours are handled by element.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "host_common.h"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

constexpr int kLogitsThreads = 256;

struct LogitsArgs {
  b200_logits_problem q;
  int stretch;   // positions per CTA, a multiple of kLogitsThreads
  int stretches; // CTAs per row
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

struct RowPenalties {
  float repetition, frequency, presence;
};

__device__ __forceinline__ float penalised(float x, uint32_t count, uint32_t seen_bit, const RowPenalties& p) {
  if (count == 0) return x;
  x = x > 0.f ? x / p.repetition : x * p.repetition;
  const uint32_t made = count & ~seen_bit;
  return made == 0 ? x : x - (p.frequency * static_cast<float>(made) + p.presence);
}

// Counters of a stretch: 32 bits per position, or 16 where the output is too short to overflow 15 (twice
// the stretch in the same shared memory, and half as many readings of the history).
template <bool kNarrow>
struct Counters {
  static constexpr uint32_t kSeen = kNarrow ? 1u << 15 : 1u << 31;   // in the prompt; the other bits count the output
  uint32_t* words;
  // Both say whether the token is met for the first time.
  __device__ __forceinline__ bool prompt(int at) const {
    if (kNarrow) return (atomicOr(words + (at >> 1), kSeen << (16 * (at & 1))) >> (16 * (at & 1)) & 0xffffu) == 0;
    return atomicOr(words + at, kSeen) == 0;
  }
  __device__ __forceinline__ bool output(int at) const {
    if (kNarrow) return (atomicAdd(words + (at >> 1), 1u << (16 * (at & 1))) >> (16 * (at & 1)) & 0xffffu) == 0;
    return atomicAdd(words + at, 1u) == 0;
  }
  __device__ __forceinline__ uint32_t operator[](int at) const {
    return kNarrow ? words[at >> 1] >> (16 * (at & 1)) & 0xffffu : words[at];
  }
};

// Minus infinity in the granule's elements whose bit is clear.
template <typename T>
__device__ __forceinline__ uint4 masked(uint4 v, uint32_t bits) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  if constexpr (sizeof(T) == 2) {
    constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // a bit moved to the top of a byte, whose sign fills half a word
      uint32_t keep;
      asm("prmt.b32 %0, %1, %2, 0xcc88;" : "=r"(keep) : "r"(bits << 7 >> 2 * i), "r"(bits << 6 >> 2 * i));
      w[i] = (w[i] & keep) | (kInf & ~keep);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((bits >> i & 1) == 0) w[i] = 0xff800000u;
  }
  return v;
}

// Counts the tokens of one history that fall into [first, first + positions).
template <bool kNarrow, bool kPrompt>
__device__ __forceinline__ void count_tokens(const int32_t* tokens, int64_t length, int64_t first, int positions, int64_t vocab,
                                             const Counters<kNarrow>& counts, uint16_t* list, int* listed) {
  // Tokens of the stretch that the vocabulary has, as an unsigned range.
  const int32_t low = static_cast<int32_t>(first > 0 ? first : 0);
  const uint32_t span = static_cast<uint32_t>((first + positions < vocab ? first + positions : vocab) - low);
  constexpr int kAhead = 8;
  for (int64_t i = threadIdx.x; i < length; i += kAhead * kLogitsThreads) {
    int32_t token[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) token[j] = i + j * kLogitsThreads < length ? __ldg(tokens + i + j * kLogitsThreads) : -1;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (token[j] >= 0 && static_cast<uint32_t>(token[j] - low) < span) {
        const int at = static_cast<int>(token[j] - first);
        if (kPrompt ? counts.prompt(at) : counts.output(at)) list[atomicAdd(listed, 1)] = static_cast<uint16_t>(at);
      }
    }
  }
}

template <typename T, bool kNarrow>
__global__ void __launch_bounds__(kLogitsThreads) logits_kernel(const LogitsArgs a) {
  extern __shared__ __align__(16) uint32_t words[];
  constexpr int kVec = 16 / sizeof(T);
  const b200_logits_problem& q = a.q;
  __shared__ int listed;
  const Counters<kNarrow> counts{words};
  uint16_t* list = reinterpret_cast<uint16_t*>(words + a.stretch / (kNarrow ? 2 : 1));
  constexpr uint32_t kSeen = Counters<kNarrow>::kSeen;
  grid_launch_dependents();
  if (threadIdx.x == 0) listed = 0;
  for (int i = threadIdx.x; i < a.stretch / (kNarrow ? 8 : 4); i += kLogitsThreads) reinterpret_cast<uint4*>(words)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  grid_dependency_wait();
  // The first stretches of all rows come first: frequent tokens have low numbers as a rule, and their
  // counting takes longest.
  const unsigned rows = static_cast<unsigned>(q.rows), stretch = blockIdx.x / rows;
  const int64_t row = blockIdx.x - stretch * rows;
  const int64_t lead = (row * q.vocab) % kVec;
  const int64_t first = static_cast<int64_t>(stretch) * a.stretch - lead;   // token of position 0; may be negative
  if (first >= q.vocab) return;
  RowPenalties p{1.f, 0.f, 0.f};
  if (q.repetition != nullptr) p.repetition = q.repetition[row];
  if (q.frequency != nullptr) p.frequency = q.frequency[row];
  if (q.presence != nullptr) p.presence = q.presence[row];
  // The thread's bias entry, on its way from the start: what it needs comes from far away, one after the other.
  __shared__ int bias_ids[kLogitsThreads];
  __shared__ float bias_values[kLogitsThreads];
  const T* x = static_cast<const T*>(q.logits) + row * q.vocab;
  int bias_id = -1;
  float bias_value = 0.f, bias_logit = 0.f;
  const auto fetch_bias = [&](int64_t from) {
    const int64_t i = from + threadIdx.x;
    bias_id = q.bias_ids != nullptr && i < q.bias_length ? __ldg(q.bias_ids + row * q.bias_length + i) : -1;
    if (bias_id < 0 || bias_id >= q.vocab) bias_id = -1;
    if (bias_id >= 0) bias_value = __ldg(q.bias_values + row * q.bias_length + i);
    if (bias_id >= first && bias_id >= 0 && bias_id < first + a.stretch) bias_logit = to_float(x[bias_id]);
  };
  fetch_bias(0);
  if (q.prompt_tokens != nullptr) count_tokens<kNarrow, true>(q.prompt_tokens + row * q.prompt_length, q.prompt_length, first, a.stretch, q.vocab, counts, list, &listed);
  if (q.output_tokens != nullptr) count_tokens<kNarrow, false>(q.output_tokens + row * q.output_length, q.output_length, first, a.stretch, q.vocab, counts, list, &listed);
  T* y = static_cast<T*>(q.out) + row * q.vocab;
  const uint32_t* allowed = q.allowed == nullptr ? nullptr : reinterpret_cast<const uint32_t*>(q.allowed) + row * q.allowed_stride;
  const auto finish = [&](int64_t token, float v) {
    const bool keep = allowed == nullptr || (__ldg(allowed + token / 32) >> (token % 32) & 1u) != 0;
    return from_float<T>(keep ? v : __int_as_float(0xff800000));
  };
  // Whole granules, four of them on their way per thread.
  constexpr int kAhead = 4;
  constexpr uint32_t kAll = (1u << kVec) - 1;
  for (int e0 = threadIdx.x * kVec; e0 < a.stretch; e0 += kAhead * kLogitsThreads * kVec) {
    uint4 v[kAhead];
    uint32_t bits[kAhead];
    bool whole[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int e = e0 + j * kLogitsThreads * kVec;
      const int64_t token = first + e;
      whole[j] = e < a.stretch && token >= 0 && token + kVec <= q.vocab;
      bits[j] = kAll;
      if (whole[j]) {
        v[j] = __ldcs(reinterpret_cast<const uint4*>(x + token));
        if (allowed != nullptr) {   // kVec bits from bit `token` on, out of one word or two
          const uint32_t at = static_cast<uint32_t>(token) / 32, shift = static_cast<uint32_t>(token) % 32;
          const uint32_t lo = __ldg(allowed + at), hi = shift + kVec > 32 ? __ldg(allowed + at + 1) : 0;
          bits[j] = __funnelshift_r(lo, hi, shift) & kAll;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int e = e0 + j * kLogitsThreads * kVec;
      const int64_t token = first + e;
      if (whole[j]) {
        __stcs(reinterpret_cast<uint4*>(y + token), bits[j] == kAll ? v[j] : masked<T>(v[j], bits[j]));
      } else if (e < a.stretch) {   // shared with the row before or behind
        for (int i = 0; i < kVec; ++i) {
          const int64_t t = token + i;
          if (t >= 0 && t < q.vocab) y[t] = finish(t, to_float(x[t]));
        }
      }
    }
  }
  __syncthreads();   // the counters are complete, and the stretch is stored
  for (int i = threadIdx.x; i < listed; i += kAhead * kLogitsThreads) {
    float value[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)   // all on their way before the first store
      if (i + j * kLogitsThreads < listed) value[j] = to_float(x[first + list[i + j * kLogitsThreads]]);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i + j * kLogitsThreads >= listed) break;
      const int at = list[i + j * kLogitsThreads];
      y[first + at] = finish(first + at, penalised(value[j], counts[at], kSeen, p));
    }
  }
  if (q.bias_ids == nullptr) return;
  // Biased tokens are computed once more from the start. The first entry of a token adds up the values
  // of all its entries, in their order. (More entries than threads: each pass looks at those before and
  // behind it in memory.)
  for (int64_t from = 0; from < q.bias_length; from += kLogitsThreads) {
    if (from > 0) fetch_bias(from);
    bias_ids[threadIdx.x] = bias_id, bias_values[threadIdx.x] = bias_value;
    __syncthreads();   // and the listed tokens are stored
    if (bias_id >= first && bias_id >= 0 && bias_id < first + a.stretch) {
      const int32_t* ids = q.bias_ids + row * q.bias_length;
      const float* values = q.bias_values + row * q.bias_length;
      const int here = static_cast<int>(q.bias_length - from < kLogitsThreads ? q.bias_length - from : kLogitsThreads);
      bool earlier = false;
      for (int64_t j = 0; j < from && !earlier; ++j) earlier = __ldg(ids + j) == bias_id;
      for (int j = 0; j < static_cast<int>(threadIdx.x); ++j) earlier |= bias_ids[j] == bias_id;
      if (!earlier) {
        float bias = 0.f;
        for (int j = threadIdx.x; j < here; ++j) bias += bias_ids[j] == bias_id ? bias_values[j] : 0.f;
        for (int64_t j = from + here; j < q.bias_length; ++j) bias += __ldg(ids + j) == bias_id ? __ldg(values + j) : 0.f;
        y[bias_id] = finish(bias_id, penalised(bias_logit, counts[static_cast<int>(bias_id - first)], kSeen, p) + bias);
      }
    }
    __syncthreads();
  }
}

template <typename T, bool kNarrow>
int launch_counted(const b200_logits_problem& q, cudaStream_t s) {
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  // 32 KiB of counters: seven CTAs per SM. A short stretch for few rows: at least two CTAs per SM where
  // the vocabulary allows it.
  LogitsArgs a{q, kNarrow ? 16384 : 8192, 0};
  const int64_t wanted = 2 * static_cast<int64_t>(sm_count());
  while (a.stretch > 1024 && q.rows * ((q.vocab + a.stretch - 1) / a.stretch) < wanted) a.stretch /= 2;
  a.stretches = static_cast<int>((q.vocab + kVec - 1 + a.stretch - 1) / a.stretch);
  const int64_t blocks = q.rows * a.stretches;
  if (blocks > 0x7fffffffLL) return B200_ERR_INVALID_PROBLEM;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kLogitsThreads);
  // Counters, and the list of the stretch's tokens that are in the history.
  const int64_t history = (q.prompt_tokens != nullptr ? q.prompt_length : 0) + (q.output_tokens != nullptr ? q.output_length : 0);
  cfg.dynamicSmemBytes = a.stretch * (kNarrow ? sizeof(uint16_t) : sizeof(uint32_t)) + sizeof(uint16_t) * (history < a.stretch ? history : a.stretch);
  cfg.stream = s;
  if (!ensure_dynamic_smem<logits_kernel<T, kNarrow>, 64 * 1024>()) return B200_ERR_LAUNCH_FAILED;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  if (cudaLaunchKernelEx(&cfg, logits_kernel<T, kNarrow>, a) != cudaSuccess) return launch_failed();
  return launch_status();
}

template <typename T>
int launch_logits(const b200_logits_problem& q, cudaStream_t s) {
  return q.output_length < (1 << 15) ? launch_counted<T, true>(q, s) : launch_counted<T, false>(q, s);
}

}  // namespace
}  // namespace b200

extern "C" int b200_process_logits(const b200_logits_problem* problem, b200_stream_t stream) {
  if (problem == nullptr) return B200_ERR_INVALID_ARGUMENT;
  const b200_logits_problem& q = *problem;
  if (q.rows < 0 || q.vocab < 0 || q.prompt_length < 0 || q.output_length < 0 || q.bias_length < 0) return B200_ERR_INVALID_ARGUMENT;
  if (q.vocab > (int64_t{1} << 30)) return B200_ERR_INVALID_PROBLEM;
  if ((q.bias_ids == nullptr) != (q.bias_values == nullptr)) return B200_ERR_INVALID_ARGUMENT;
  if (q.allowed != nullptr && q.allowed_stride != 0 && q.allowed_stride < (q.vocab + 31) / 32) return B200_ERR_INVALID_ARGUMENT;
  if (q.rows == 0 || q.vocab == 0) return B200_OK;
  if (q.logits == nullptr || q.out == nullptr) return B200_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(q.logits) % 16 != 0 || reinterpret_cast<uintptr_t>(q.out) % 16 != 0) return B200_ERR_MISALIGNED_OPERAND;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (q.dtype) {
    case B200_FP32: return b200::launch_logits<float>(q, s);
    case B200_FP16: return b200::launch_logits<__half>(q, s);
    case B200_BF16: return b200::launch_logits<__nv_bfloat16>(q, s);
    default: return B200_ERR_INVALID_ARGUMENT;
  }
}
