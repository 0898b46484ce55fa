// Matrix-vector product with 4-bit weights and group scales, for 1 to 16 rows of x.
//
// Bound by HBM: every weight byte is read once, 2 * rows products per weight. The arithmetic must
// therefore cost a handful of instructions per eight weights, and goes through the warp-level matrix
// instruction m16n8k16 with the weights as its 16-row operand and the rows of x as its columns: the
// 5th-generation tensor cores would want 128 weight rows per tile in shared memory, a detour for
// bytes that are used once; here they go from global memory to registers to the multiply.
//
// A warp owns 16 or 32 rows of weights and a range of K. The sum over k does not care about its order, so
// each of the four threads that share a row takes its own run of consecutive weights (kBytes bytes
// per load) instead of the interleaved pairs that the instruction nominally wants, and loads the
// same run of x. Nibbles i and i + 4 of a 32-bit word become one pair of 16-bit values: the bits of
// a code c placed into the mantissa of 1024 (FP16) or 128 (BF16) give 1024 + c or 128 + c exactly, and
// subtracting 1024 + zero or 128 + zero leaves c - zero, exact. Each step of K lies inside one group:
// its FP32 product is multiplied by the group's scale when it is added to the running sum.
//
// What it measured: one BF16 row by 28672 x 8192 (117 MB of weights) 36.7 us, FP16 34.8, FP32 113, against
// 18.5 for the weights at the copy bandwidth: the integer pipe 67 % busy, issue slots 60 %; 16 BF16 rows 73,
// 8 FP32 rows 397. What brought it there
// from 44.7: a code's mask and its base in one instruction (38.5), and the divisions that place a warp in
// its row done by the host, the zero point of symmetric weights made once (36.8). What did not help, all
// timed side by side: 32 rows per warp (x shared, half the warps: 51.5 against 44.8); more warps by fewer
// registers (45.3 with five CTAs per SM instead of four); the warps side by side along K instead of in
// ranges (45.6 against 44.8); the next step's weights loaded a step ahead (39.3); x laid out as pairs in
// shared memory (37.3 against 38.5 here, but 21.0 against 18.3 for 11008 x 4096 in groups of 32 and 9.6
// against 8.7 for four rows by 4096 x 4096); and integer matrix instructions on the raw codes with x in
// signed 8-bit digits, a third of the instructions (62 against 44.8).
//
// FP32 x is written as the sum of three BF16 numbers (8 + 8 + 8 bits, by truncation: exact), which take
// three columns of the instruction and are added up at the end, so that products and sums are as
// accurate as FP32 arithmetic.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "host_common.h"
#include "ptx_sm100.cuh"

namespace b200 {
namespace {

constexpr int kMaxRows = 16;

struct W4Args {
  b200_matvec_w4_problem q;
  int groups, steps, group_steps;   // groups of a row, steps of a row and of a group
};

template <typename T> struct Pair;
template <> struct Pair<__half> {
  static constexpr uint32_t kBase = 0x64006400u;   // 1024, 1024
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Pair<__nv_bfloat16> {
  static constexpr uint32_t kBase = 0x43004300u;   // 128, 128
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Pair<float> : Pair<__nv_bfloat16> {};   // FP32 x travels as three BF16 columns

// The eight codes of a word, less their zero: pairs (0,4), (1,5), (2,6), (3,7). These are most of the
// kernel's instructions, so there are as few as the type allows:
// the ten mantissa bits of FP16 hold a code in bits 4..7 as well, sixteen times too large, which the
// subtraction's multiply-add takes back for nothing; the seven of BF16 do not.
struct ZeroPair {
  uint32_t low, high;   // what to subtract from a code in bits 0..3, and in bits 4..7
};
template <typename T>
__device__ __forceinline__ ZeroPair zero_pair(uint32_t z) {
  const uint32_t twice = z | z << 16;
  // 1024 + z as it is; a code in bits 4..7 reads 1024 + 16 c and is divided by 16, which leaves 64 + c.
  return {Pair<T>::kBase | twice, 0xd400d400u | twice << 4};   // FP16: -(64 + z)
}
// (v & kMask) | base in one instruction.
template <uint32_t kMask>
__device__ __forceinline__ uint32_t masked_onto(uint32_t base, uint32_t v) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "n"(kMask), "r"(base));
  return r;
}
template <typename T>
__device__ __forceinline__ void decode(uint32_t (&out)[4], uint32_t w, const ZeroPair& zero, uint32_t base) {
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t upper = w >> 8;
    const __half2 sixteenth = __half2half2(__ushort_as_half(0x2c00));
    const auto high = [&](uint32_t v) {
      const uint32_t c = masked_onto<0x00f000f0u>(base, v);
      const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&c), sixteenth, *reinterpret_cast<const __half2*>(&zero.high));
      return *reinterpret_cast<const uint32_t*>(&r);
    };
    out[0] = Pair<T>::sub(masked_onto<0x000f000fu>(base, w), zero.low), out[1] = high(w);
    out[2] = Pair<T>::sub(masked_onto<0x000f000fu>(base, upper), zero.low), out[3] = high(upper);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = Pair<T>::sub(masked_onto<0x000f000fu>(base, w >> (4 * j)), zero.low);
  }
}

template <int kBytes> struct Packed;
template <> struct Packed<16> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const uint8_t* p) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
};
template <> struct Packed<8> {
  uint32_t w[2];
  __device__ __forceinline__ void load(const uint8_t* p) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
  }
};
template <> struct Packed<4> {
  uint32_t w[1];
  __device__ __forceinline__ void load(const uint8_t* p) { w[0] = __ldg(reinterpret_cast<const uint32_t*>(p)); }
};

// Eight consecutive x of one column as four pairs (x0,x4), (x1,x5), (x2,x6), (x3,x7).
template <typename T>
__device__ __forceinline__ void load_pairs(uint32_t (&out)[4], const T* p, int) {
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));   // (x0,x1) (x2,x3) (x4,x5) (x6,x7)
  out[0] = __byte_perm(v.x, v.z, 0x5410), out[1] = __byte_perm(v.x, v.z, 0x7632);
  out[2] = __byte_perm(v.y, v.w, 0x5410), out[3] = __byte_perm(v.y, v.w, 0x7632);
}
// Term `part` of an FP32 number as a sum of three BF16 ones, in the upper half of the result.
__device__ __forceinline__ uint32_t bf16_term(float x, int part) {
  const uint32_t hi = __float_as_uint(x) & 0xffff0000u;
  if (part == 0) return hi;
  // What an infinity leaves is nothing: the first term carries it alone. What a NaN leaves is one, so that
  // it stays one even where its first term reads as an infinity (a payload in the lower half only).
  const float r1 = fabsf(x) == __uint_as_float(0x7f800000u) ? 0.f : x - __uint_as_float(hi);
  const uint32_t mid = __float_as_uint(r1) & 0xffff0000u;
  if (part == 1) return mid;
  return __float_as_uint(r1 - __uint_as_float(mid));
}
template <>
__device__ __forceinline__ void load_pairs<float>(uint32_t (&out)[4], const float* p, int part) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  out[0] = __byte_perm(bf16_term(a.x, part), bf16_term(b.x, part), 0x7632);
  out[1] = __byte_perm(bf16_term(a.y, part), bf16_term(b.y, part), 0x7632);
  out[2] = __byte_perm(bf16_term(a.z, part), bf16_term(b.z, part), 0x7632);
  out[3] = __byte_perm(bf16_term(a.w, part), bf16_term(b.w, part), 0x7632);
}

__device__ __forceinline__ float scale_at(const void* scales, int dtype, int64_t at) {
  if (dtype == B200_FP32) return __ldg(static_cast<const float*>(scales) + at);
  if (dtype == B200_FP16) return __half2float(__ldg(static_cast<const __half*>(scales) + at));
  return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(scales) + at));
}
__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// kTiles groups of eight columns; kHeight times 16 rows of weights per warp; kBytes weight bytes per thread, row and step (a step is 8 * kBytes
// values of K: it has to lie inside a group).
template <typename T, int kTiles, int kBytes, int kHeight, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) matvec_w4_kernel(const W4Args a) {
  constexpr int kParts = sizeof(T) == 4 ? 3 : 1;   // columns per row of x
  constexpr int kStep = 8 * kBytes;
  __shared__ float sums[kWarps][16 * kHeight][8 * kTiles + 1];
  constexpr int kRows = 2 * kHeight;   // weight rows per thread, eight apart
  const b200_matvec_w4_problem& q = a.q;
  grid_launch_dependents();
  grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int quad = lane >> 2, t = lane & 3;
  const int row0 = blockIdx.x * 16 * kHeight;
  const int groups = a.groups, group_steps = a.group_steps, steps = a.steps;
  const int begin = static_cast<int>(static_cast<int64_t>(steps) * warp / kWarps), end = static_cast<int>(static_cast<int64_t>(steps) * (warp + 1) / kWarps);
  // This thread's weight rows. Rows behind the last are read as the last one and not stored.
  const uint8_t* w[kRows];
  int64_t at[kRows];   // of the group's scale and zero
  const int group = group_steps == 1 ? begin : begin / group_steps;
  int left = (group + 1) * group_steps - begin;   // steps left in the group
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t r = min(row0 + 8 * i + quad, q.n - 1);
    w[i] = q.qweight + r * (q.k / 2) + t * kBytes + static_cast<int64_t>(begin) * (kStep / 2);
    at[i] = r * groups + group;
  }

  float total[kHeight][kTiles][4] = {};
  float scale[kRows];
  ZeroPair zero[kRows];
  uint32_t base;   // a register that the compiler takes for no constant, which would cost an instruction per use
  asm volatile("mov.b32 %0, %1;" : "=r"(base) : "n"(Pair<T>::kBase));
#pragma unroll
  for (int i = 0; i < kRows; ++i) zero[i] = zero_pair<T>(8);
  bool fresh = true;
#pragma unroll(kHeight == 1 ? 2 : 1)
  for (int s = begin; s < end; ++s) {
    Packed<kBytes> p[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) p[i].load(w[i]), w[i] += kStep / 2;
    if (fresh) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        scale[i] = scale_at(q.scales, q.scale_dtype, at[i]);
        if (q.zeros != nullptr) zero[i] = zero_pair<T>(__ldg(q.zeros + at[i]) & 15u);
        ++at[i];
      }
    }
    fresh = --left == 0;
    if (fresh) left = group_steps;
    float acc[kHeight][kTiles][4] = {};
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) {
      uint32_t m[kRows][4];
#pragma unroll
      for (int r = 0; r < kRows; ++r) decode<T>(m[r], p[r].w[i], zero[r], base);
      const int64_t k = static_cast<int64_t>(s) * kStep + t * 2 * kBytes + i * 8;
#pragma unroll
      for (int c = 0; c < kTiles; ++c) {
        const int column = c * 8 + quad;
        uint32_t x[4] = {0, 0, 0, 0};
        if (column < q.rows * kParts) load_pairs<T>(x, static_cast<const T*>(q.x) + static_cast<int64_t>(column / kParts) * q.k + k, column % kParts);
#pragma unroll
        for (int h = 0; h < kHeight; ++h) {
          const uint32_t(&upper)[4] = m[2 * h], (&lower)[4] = m[2 * h + 1];
          const uint32_t first[4] = {upper[0], lower[0], upper[1], lower[1]}, second[4] = {upper[2], lower[2], upper[3], lower[3]};
          Pair<T>::mma(acc[h][c], first, x[0], x[1]);
          Pair<T>::mma(acc[h][c], second, x[2], x[3]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < kHeight; ++h)
#pragma unroll
      for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) total[h][c][e] += scale[2 * h + e / 2] * acc[h][c][e];
  }
#pragma unroll
  for (int h = 0; h < kHeight; ++h)
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) sums[warp][16 * h + 8 * (e / 2) + quad][c * 8 + 2 * t + e % 2] = total[h][c][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * kHeight * q.rows; i += kWarps * 32) {
    const int n = i % (16 * kHeight), m = i / (16 * kHeight);
    if (row0 + n >= q.n) continue;
    float sum = 0.f;
    for (int v = 0; v < kWarps; ++v)
#pragma unroll
      for (int part = 0; part < kParts; ++part) sum += sums[v][n][m * kParts + part];
    store_out(static_cast<T*>(q.y) + static_cast<int64_t>(m) * q.n + row0 + n, sum);
  }
}

template <typename T, int kTiles, int kBytes, int kHeight, int kWarps>
int launch_shape(const b200_matvec_w4_problem& q, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(q.n) + 16 * kHeight - 1) / (16 * kHeight)));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = s;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  if (cudaLaunchKernelEx(&cfg, matvec_w4_kernel<T, kTiles, kBytes, kHeight, kWarps>, W4Args{q, q.k / q.group, q.k / (8 * kBytes), q.group / (8 * kBytes)}) != cudaSuccess) return launch_failed();
  return launch_status();
}

// Warps of 32 rows of weights read x half as often, but there are half as many of them. That pays when x
// is what a CTA mostly reads, from L2: with six columns or more, and two CTAs left for every
// multiprocessor. BF16 by 28672 x 8192, 32 against 16 rows: 47 and 58 us of 8 rows, 72 and 93 of 16, but
// 43 and 39 of 4; 8 rows by 4096 x 4096 13.3 and 10.8. Short runs of codes (groups of 64) lose with
// 16-bit x (19.9 and 18.0 of 8 rows by 14336 x 4096); FP32 x, three times as much work, gains (69 and 122).
template <typename T, int kTiles, int kBytes>
int launch(const b200_matvec_w4_problem& q, cudaStream_t s) {
  constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
  if constexpr (kTiles <= 3 && kBytes >= (kParts == 3 ? 8 : 16)) {
    if (q.rows * kParts >= 6 && q.n >= 2 * 32 * sm_count()) return launch_shape<T, kTiles, kBytes, 2, 8>(q, s);
  }
  // Few CTAs: as many warps in each as leave all CTAs room at once, one or two per multiprocessor. 16
  // against 8 warps, BF16: one row by 4096 x 4096 5.7 and 8.3 us, by 4096 x 14336 12.1 and 22.6, 16 rows
  // by 2048 x 8192 9.0 and 18.7. Two CTAs of 16 warps have 64 registers per thread, which only 16-bit x of
  // up to eight rows does with; else 12 warps (16 rows by 4096 x 14336 23.3, 8 warps 34.1, 16 24.5).
  // More CTAs than that lose by it (16 rows by 5120 x 5120 13.5 with 8 warps, 18.9 with 12).
  if constexpr (kTiles <= 3) {
    constexpr bool kSmall = kTiles == 1 && kParts == 1;
    const int round = 16 * sm_count();   // rows of one CTA per multiprocessor
    if (q.n <= (kSmall ? 2 * round : round)) return launch_shape<T, kTiles, kBytes, 1, 16>(q, s);
    if constexpr (!kSmall) {
      if (q.n <= 2 * round) return launch_shape<T, kTiles, kBytes, 1, 12>(q, s);
    }
  }
  return launch_shape<T, kTiles, kBytes, 1, 8>(q, s);
}

template <typename T, int kTiles>
int launch_bytes(const b200_matvec_w4_problem& q, cudaStream_t s) {
  if (q.group % 128 == 0) return launch<T, kTiles, 16>(q, s);
  if (q.group % 64 == 0) return launch<T, kTiles, 8>(q, s);
  return launch<T, kTiles, 4>(q, s);
}

template <typename T>
int launch_tiles(const b200_matvec_w4_problem& q, cudaStream_t s) {
  const int columns = q.rows * (sizeof(T) == 4 ? 3 : 1);
  if (columns <= 8) return launch_bytes<T, 1>(q, s);
  if (columns <= 16) return launch_bytes<T, 2>(q, s);
  if constexpr (sizeof(T) == 4) return columns <= 24 ? launch_bytes<T, 3>(q, s) : launch_bytes<T, 6>(q, s);
  return B200_ERR_INTERNAL;
}

}  // namespace
}  // namespace b200

extern "C" int b200_matvec_w4(const b200_matvec_w4_problem* problem, b200_stream_t stream) {
  if (problem == nullptr) return B200_ERR_INVALID_ARGUMENT;
  const b200_matvec_w4_problem& q = *problem;
  if (q.dtype < B200_FP32 || q.dtype > B200_BF16 || (q.scale_dtype != q.dtype && q.scale_dtype != B200_FP32)) return B200_ERR_INVALID_ARGUMENT;
  if (q.rows < 0 || q.n < 0 || q.k <= 0 || q.group <= 0) return B200_ERR_INVALID_ARGUMENT;
  if (q.rows > b200::kMaxRows) return B200_ERR_NOT_SUPPORTED;
  if (q.group % 32 != 0 || q.k % q.group != 0) return B200_ERR_INVALID_PROBLEM;
  if (q.rows == 0 || q.n == 0) return B200_OK;
  if (q.x == nullptr || q.qweight == nullptr || q.scales == nullptr || q.y == nullptr) return B200_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(q.x) % 16 != 0 || reinterpret_cast<uintptr_t>(q.qweight) % 16 != 0) return B200_ERR_MISALIGNED_OPERAND;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (q.dtype) {
    case B200_FP32: return b200::launch_tiles<float>(q, s);
    case B200_FP16: return b200::launch_tiles<__half>(q, s);
    default: return b200::launch_tiles<__nv_bfloat16>(q, s);
  }
}
