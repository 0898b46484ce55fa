// Attention for FP32 operands, on the FMA pipe.
//
// One pass over the keys with a running maximum and sum: for a tile of rows (i, g) and a block of 64
// keys, S = Q K^T, m' = max(m, rowmax S), P = 2^(S - m'), l = l 2^(m - m') + rowsum P,
// O = O 2^(m - m') + P V; the rows are divided by l at the end. Q is scaled by scale * log2(e) when it
// is staged. A thread holds a 4 x 4 patch of S and four rows of O; 16 threads share a row, whose
// maximum and sum they exchange by shuffles.
#include "attention.cuh"

namespace b200 {
namespace {

constexpr int kKeys = kSimtKeyBlock;
constexpr float kMinusInf = -__builtin_huge_valf();

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }

__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rows of `count` floats [rows][dim] -> shared [rows][pitch]; rows from `live` on become zeros, so that
// nothing outside the sequence enters a product.
template <int kThreads>
__device__ __forceinline__ void stage_rows(float* dst, const float* src, int64_t stride, int rows, int live, int dim, int pitch) {
  const int quads = dim / 4;
  for (int i = threadIdx.x; i < rows * quads; i += kThreads) {
    const int r = i / quads, c = (i - r * quads) * 4;
    store4(dst + r * pitch + c, r < live ? load4(src + r * stride + c) : make_float4(0.f, 0.f, 0.f, 0.f));
  }
}

template <int kRows>
__global__ void __launch_bounds__(kRows * 4) attention_simt_kernel(const AttentionArgs a) {
  constexpr int kThreads = kRows * 4;
  extern __shared__ __align__(16) float smem[];
  __shared__ WorkScratch scratch;
  const int pitch = a.dim + 4;
  float* qs = smem;
  float* ks = qs + kRows * pitch;
  float* vs = ks + kKeys * pitch;
  float* ps = vs + kKeys * pitch;   // [kRows][kKeys + 4]
  constexpr int kPitchP = kKeys + 4;
  grid_launch_dependents();
  grid_dependency_wait();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  SegmentWalk<kKeys> walk(a, find_range<kKeys, kThreads>(a, &scratch));
  Segment g;
  if (threadIdx.x == 0) start_records(a);
  while (walk.next(&g)) {
    if (threadIdx.x == 0) record(a, g);
    int pitch_rows;
    const int64_t slot = slot_of(a, g, &pitch_rows);
    const int row0 = g.unit * a.unit_rows;
    const int rows = min(a.unit_rows, g.seq.n * a.group - row0);
    __syncthreads();   // the last segment's readers are done
    for (int i = threadIdx.x; i < kRows * (a.dim / 4); i += kThreads) {
      const int r = i / (a.dim / 4), c = (i - r * (a.dim / 4)) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows) {
        const int token = (row0 + r) / a.group, head = g.head * a.group + (row0 + r - token * a.group);
        v = load4(static_cast<const float*>(a.q) + static_cast<int64_t>(g.seq.q_row + token) * a.q_row + head * a.q_head + c);
      }
      store4(qs + r * pitch + c, make_float4(v.x * a.scale_log2, v.y * a.scale_log2, v.z * a.scale_log2, v.w * a.scale_log2));
    }
    int seen[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) seen[i] = visible_keys(a, g.seq, (row0 + ty * 4 + i) / a.group);
    float m[4], l[4];
    float4 o[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = kMinusInf, l[i] = 0.f, o[i][0] = o[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int s = g.seq.source;
    const float* k = static_cast<const float*>(a.k[s]) + (s == 1 ? g.seq.batch * a.k_batch : 0) + g.seq.k_row * a.k_row[s] + g.head * a.k_head[s];
    const float* v = static_cast<const float*>(a.v[s]) + (s == 1 ? g.seq.batch * a.v_batch : 0) + g.seq.k_row * a.v_row[s] + g.head * a.v_head[s];
    for (int b = g.block_begin; b < g.block_end; ++b) {
      const int64_t key0 = static_cast<int64_t>(b) * kKeys;
      const int live = min(kKeys, static_cast<int>(g.seq.m - key0));
      __syncthreads();
      stage_rows<kThreads>(ks, k + key0 * a.k_row[s], a.k_row[s], kKeys, live, a.dim, pitch);
      stage_rows<kThreads>(vs, v + key0 * a.v_row[s], a.v_row[s], kKeys, live, a.dim, pitch);
      __syncthreads();
      float x[4][4] = {};
      for (int d = 0; d < a.dim; d += 4) {
        float4 qv[4], kv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(qs + (ty * 4 + i) * pitch + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(ks + (tx + 16 * j) * pitch + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            x[i][j] += qv[i].x * kv[j].x + qv[i].y * kv[j].y + qv[i].z * kv[j].z + qv[i].w * kv[j].w;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float top = kMinusInf;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (key0 + tx + 16 * j >= seen[i]) x[i][j] = kMinusInf;   // chosen, not added: the product may be NaN
          top = fmaxf(top, x[i][j]);
        }
        const float next = fmaxf(m[i], half_warp_max(top));
        const float base = next == kMinusInf ? 0.f : next;   // nothing seen yet: all terms are 2^(-inf)
        const float keep = exp2f(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2f(x[i][j] - base);
          ps[(ty * 4 + i) * kPitchP + tx + 16 * j] = p;
          sum += p;
        }
        l[i] = l[i] * keep + half_warp_sum(sum);
        m[i] = next;
#pragma unroll
        for (int c = 0; c < 2; ++c) o[i][c].x *= keep, o[i][c].y *= keep, o[i][c].z *= keep, o[i][c].w *= keep;
      }
      __syncwarp();   // a row's probabilities are written and read by the same half warp
      for (int key = 0; key < kKeys; key += 4) {
        float4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(ps + (ty * 4 + i) * kPitchP + key);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int d = tx * 4 + 64 * c;
          if (d < a.dim) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 w = *reinterpret_cast<const float4*>(vs + (key + e) * pitch + d);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float pe = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
                o[i][c].x += pe * w.x, o[i][c].y += pe * w.y, o[i][c].z += pe * w.z, o[i][c].w += pe * w.w;
              }
            }
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = ty * 4 + i;
      if (r >= rows) continue;
      if (is_partial(a, g)) {
        if (tx == 0) a.partial_ml[slot + r] = make_float2(m[i], l[i]);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (tx * 4 + 64 * c < a.dim) store4(a.partial_o + slot * a.dim + (static_cast<int64_t>(tx + 16 * c) * pitch_rows + r) * 4, o[i][c]);
      } else {
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        float* y = static_cast<float*>(a.out) + output_row(a, g.seq.q_row, g.head, row0 + r) * a.dim;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (tx * 4 + 64 * c < a.dim)
            store4(y + tx * 4 + 64 * c, make_float4(o[i][c].x * inv, o[i][c].y * inv, o[i][c].z * inv, o[i][c].w * inv));
      }
    }
  }
}

constexpr size_t simt_smem_bytes(int rows, int dim) {
  return sizeof(float) * ((rows + 2 * static_cast<size_t>(kKeys)) * (dim + 4) + static_cast<size_t>(rows) * (kKeys + 4));
}

template <int kRows>
int launch(const AttentionArgs& a, cudaStream_t s) {
  if (!ensure_dynamic_smem<attention_simt_kernel<kRows>, simt_smem_bytes(kRows, 128)>()) return B200_ERR_LAUNCH_FAILED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.ctas));
  cfg.blockDim = dim3(kRows * 4);
  cfg.dynamicSmemBytes = simt_smem_bytes(kRows, a.dim);
  cfg.stream = s;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  if (cudaLaunchKernelEx(&cfg, attention_simt_kernel<kRows>, a) != cudaSuccess) return launch_failed();
  return launch_status();
}

}  // namespace

void plan_attention_simt(AttentionArgs* a, int sms) {
  // Tiles of 16 rows where the rows of a sequence would leave most of a 64-row tile empty; whole tokens
  // where the group allows it.
  const int64_t rows_per_sequence = a->kind == kShared ? a->group : static_cast<int64_t>(a->q_rows) * a->group / (a->sequences > 0 ? a->sequences : 1);
  const int tile = rows_per_sequence <= 16 ? 16 : 64;
  a->tokens = tile / a->group;
  a->unit_rows = a->tokens > 0 ? a->tokens * a->group : tile;
  a->unit_cost = 1, a->pair_cost = 1;
  a->ctas = sms * (tile == 16 ? 3 : 2);
}

int launch_attention_simt(const AttentionArgs& a, cudaStream_t s) {
  return a.unit_rows > 16 ? launch<64>(a, s) : launch<16>(a, s);
}

}  // namespace b200
