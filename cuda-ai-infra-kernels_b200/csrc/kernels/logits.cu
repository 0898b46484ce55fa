// Logits of a batch before the softmax: penalties for tokens already seen, a sparse bias and a
// grammar mask, in one pass over [rows][vocab].
//
// Bound by HBM: the logits are read once and written once. A CTA owns a stretch of one row's
// vocabulary and counts, in shared memory, the occurrences of its tokens in the row's history (it
// reads the whole history, which the row's other CTAs read too, from L2; integer atomics, so the
// order does not matter). Counting per stretch needs no workspace and no second launch.
//
// A row of odd length starts anywhere in a 16-byte granule. Stretches are therefore cut in the
// granules of the array, not of the row: position e of the stretch space of row r is token
// e - lead(r) with lead(r) = r * vocab mod (elements per granule), so that every whole granule is
// one 128-bit access; the granules that a row shares with its neighbours are handled by element.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_common.h"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

constexpr int kLogitsThreads = 256;
constexpr uint32_t kInPrompt = 1u << 31;   // the other bits count occurrences in the output

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

__device__ __forceinline__ float penalised(float x, uint32_t count, const RowPenalties& p) {
  if (count == 0) return x;
  x = x > 0.f ? x / p.repetition : x * p.repetition;
  const uint32_t made = count & ~kInPrompt;
  return made == 0 ? x : x - (p.frequency * static_cast<float>(made) + p.presence);
}

// Counts the tokens of one history that fall into [first, first + positions).
__device__ __forceinline__ void count_tokens(const int32_t* tokens, int64_t length, int64_t first, int positions, int64_t vocab,
                                             uint32_t* counts, bool prompt) {
  for (int64_t i = threadIdx.x; i < length; i += kLogitsThreads) {
    const int64_t token = __ldg(tokens + i);
    const int64_t at = token - first;
    if (token >= 0 && token < vocab && at >= 0 && at < positions) {
      if (prompt) atomicOr(counts + at, kInPrompt);
      else atomicAdd(counts + at, 1u);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kLogitsThreads) logits_kernel(const LogitsArgs a) {
  extern __shared__ __align__(16) uint32_t counts[];
  constexpr int kVec = 16 / sizeof(T);
  const b200_logits_problem& q = a.q;
  grid_launch_dependents();
  for (int i = threadIdx.x; i < a.stretch; i += kLogitsThreads) counts[i] = 0;
  __syncthreads();
  grid_dependency_wait();
  const int64_t row = blockIdx.x / a.stretches;
  const int64_t lead = (row * q.vocab) % kVec;
  const int64_t first = static_cast<int64_t>(blockIdx.x % a.stretches) * a.stretch - lead;   // token of position 0; may be negative
  RowPenalties p{1.f, 0.f, 0.f};
  if (q.repetition != nullptr) p.repetition = q.repetition[row];
  if (q.frequency != nullptr) p.frequency = q.frequency[row];
  if (q.presence != nullptr) p.presence = q.presence[row];
  if (q.prompt_tokens != nullptr) count_tokens(q.prompt_tokens + row * q.prompt_length, q.prompt_length, first, a.stretch, q.vocab, counts, true);
  if (q.output_tokens != nullptr) count_tokens(q.output_tokens + row * q.output_length, q.output_length, first, a.stretch, q.vocab, counts, false);
  __syncthreads();

  const T* x = static_cast<const T*>(q.logits) + row * q.vocab;
  T* y = static_cast<T*>(q.out) + row * q.vocab;
  const uint32_t* allowed = q.allowed == nullptr ? nullptr : reinterpret_cast<const uint32_t*>(q.allowed) + row * q.allowed_stride;
  const auto finish = [&](int64_t token, float v) {
    const bool keep = allowed == nullptr || (__ldg(allowed + token / 32) >> (token % 32) & 1u) != 0;
    return from_float<T>(keep ? v : __int_as_float(0xff800000));
  };
  for (int e = threadIdx.x * kVec; e < a.stretch; e += kLogitsThreads * kVec) {
    const int64_t token = first + e;
    if (token >= q.vocab) break;
    for (int i = 0; i < kVec; ++i) {
      const int64_t t = token + i;
      if (t >= 0 && t < q.vocab) y[t] = finish(t, penalised(to_float(x[t]), counts[e + i], p));
    }
  }
  if (q.bias_ids == nullptr) return;
  // Biased tokens are computed again from the start, after the pass above has stored them. The
  // first entry of a token adds up the values of all its entries, in their order.
  __syncthreads();
  const int32_t* ids = q.bias_ids + row * q.bias_length;
  const float* values = q.bias_values + row * q.bias_length;
  for (int64_t i = threadIdx.x; i < q.bias_length; i += kLogitsThreads) {
    const int64_t token = ids[i];
    const int64_t at = token - first;
    if (token < 0 || token >= q.vocab || at < 0 || at >= a.stretch) continue;
    bool earlier = false;
    for (int64_t j = 0; j < i; ++j) earlier |= ids[j] == token;
    if (earlier) continue;
    float bias = 0.f;
    for (int64_t j = i; j < q.bias_length; ++j) bias += ids[j] == token ? values[j] : 0.f;
    y[token] = finish(token, penalised(to_float(x[token]), counts[at], p) + bias);
  }
}

template <typename T>
int launch_logits(const b200_logits_problem& q, cudaStream_t s) {
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  LogitsArgs a{q, 8192, 0};
  // A short stretch for few rows: at least two CTAs per SM where the vocabulary allows it.
  const int64_t wanted = 2 * static_cast<int64_t>(sm_count());
  while (a.stretch > 1024 && q.rows * ((q.vocab + a.stretch - 1) / a.stretch) < wanted) a.stretch /= 2;
  a.stretches = static_cast<int>((q.vocab + kVec - 1 + a.stretch - 1) / a.stretch);
  const int64_t blocks = q.rows * a.stretches;
  if (blocks > 0x7fffffffLL) return B200_ERR_INVALID_PROBLEM;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kLogitsThreads);
  cfg.dynamicSmemBytes = a.stretch * sizeof(uint32_t);
  cfg.stream = s;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  if (cudaLaunchKernelEx(&cfg, logits_kernel<T>, a) != cudaSuccess) return launch_failed();
  return launch_status();
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
