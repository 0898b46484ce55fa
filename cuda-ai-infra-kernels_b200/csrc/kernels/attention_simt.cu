// Attention for FP32 operands, on the FMA pipe.
//
// One pass over the keys with a running maximum and sum: for a tile of rows (i, g) and a block of 64
// keys, S = Q K^T, m' = max(m, rowmax S), P = 2^(S - m'), l = l 2^(m - m') + rowsum P,
// O = O 2^(m - m') + P V; the rows are divided by l at the end. Q is scaled by scale * log2(e) when it
// is staged. 16 threads share a row, whose maximum and sum they exchange by shuffles; a thread holds
// four columns of S and a sixteenth of O for 8, 4 or 2 rows. Bound by the FMA pipe, beside which the
// shared-memory pipe has to keep up: with 8 rows a thread loads 12 granules per 128 multiply-adds.
// Both products run on packed pairs (two multiply-adds per instruction): S over even and odd d apart.
//
// 2048 and 1000 causal tokens, 16 heads of 64: 354 us, 29 TFLOP/s of the 70 that the pipe reaches on
// multiply-adds alone (64-row tiles, two CTAs per SM: 453; one buffer filled between barriers: 466).
//
// Keys and values have one buffer each. The next keys are copied (cp.async) while the exponentials and
// the second product run, the next values while the first product does.
#include "attention.cuh"

namespace b200 {

cudaError_t attention_simt_status_read_clear(uint32_t* word) { return status_word_read_clear(word); }

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

__device__ __forceinline__ void copy_async(void* dst, const void* src, uint32_t bytes) {   // 16 bytes, zeros behind `bytes`
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory");
}

// kKeys rows of keys or values; rows from `live` on become zeros, so that nothing outside the sequence
// enters a product.
template <int kThreads>
__device__ __forceinline__ void copy_rows(float* dst, const float* src, int64_t stride, int live, int dim, int pitch) {
  const int quads = dim / 4;
  for (int i = threadIdx.x; i < kKeys * quads; i += kThreads) {
    const int r = i / quads, c = (i - r * quads) * 4;
    copy_async(dst + r * pitch + c, src + (r < live ? r : 0) * stride + c, r < live ? 16 : 0);
  }
}

// Four consecutive floats as two pairs.
__device__ __forceinline__ ulonglong2 pairs_at(const float* p) { return *reinterpret_cast<const ulonglong2*>(p); }

template <int kRows, int kThreads, int kColumns, typename Line>
__global__ void __launch_bounds__(kThreads, kRows == 16 ? 4 : kRows == 64 ? 2 : 1) attention_simt_kernel(const __grid_constant__ AttentionArgs a) {
  constexpr int kPer = kRows / (kThreads / 16);   // rows of a thread
  constexpr int kQuads = kColumns / 64;           // groups of four of its columns of O
  constexpr int kPitchP = kKeys + 4;
  extern __shared__ __align__(16) float smem[];
  __shared__ WorkScratch<Line> scratch;
  const int pitch = a.dim + 4;
  float* qs = smem;
  float* ks = qs + kRows * pitch;
  float* vs = ks + kKeys * pitch;
  float* ps = vs + kKeys * pitch;   // [kRows][kPitchP]
  grid_launch_dependents();
  grid_dependency_wait();
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const WorkStart<Line> start = find_range<kKeys, kThreads, Line>(a, &scratch);
  clear_unowned_rows(a, start.sequence == kRefused, threadIdx.x, kThreads);
  SegmentWalk<kKeys, Line> walk(a, start);
  Segment g;
  if (threadIdx.x == 0) start_records(a);
  while (walk.next(&g)) {
    if (threadIdx.x == 0) record(a, g);
    int slot_rows;
    const int64_t slot = slot_of(a, g, &slot_rows);
    const int row0 = g.unit * a.unit_rows;
    const int rows = min(a.unit_rows, g.seq.n * a.group - row0);
    const int s = g.seq.source;
    const float* k = static_cast<const float*>(a.k[s]) + (s == 1 ? g.seq.batch * a.k_batch : 0) + g.seq.k_row * a.k_row[s] + g.head * a.k_head[s];
    const float* v = static_cast<const float*>(a.v[s]) + (s == 1 ? g.seq.batch * a.v_batch : 0) + g.seq.k_row * a.v_row[s] + g.head * a.v_head[s];
    const auto copy_block = [&](float* dst, const float* src, int64_t stride, int b) {
      const int64_t key0 = static_cast<int64_t>(b) * kKeys;
      if (b < g.block_end) copy_rows<kThreads>(dst, src + key0 * stride, stride, min(kKeys, static_cast<int>(g.seq.m - key0)), a.dim, pitch);
      copy_commit();
    };
    __syncthreads();   // the last segment's readers are done
    copy_block(ks, k, a.k_row[s], g.block_begin);
    copy_block(vs, v, a.v_row[s], g.block_begin);
    for (int i = threadIdx.x; i < kRows * (a.dim / 4); i += kThreads) {
      const int r = i / (a.dim / 4), c = (i - r * (a.dim / 4)) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows) {
        const int token = (row0 + r) / a.group, head = g.head * a.group + (row0 + r - token * a.group);
        x = load4(static_cast<const float*>(a.q) + static_cast<int64_t>(g.seq.q_row + token) * a.q_row + head * a.q_head + c);
      }
      store4(qs + r * pitch + c, make_float4(x.x * a.scale_log2, x.y * a.scale_log2, x.z * a.scale_log2, x.w * a.scale_log2));
    }
    float m[kPer], l[kPer];
    uint64_t o[kPer][2 * kQuads];
    int seen[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      m[i] = kMinusInf, l[i] = 0.f, seen[i] = visible_keys(a, g.seq, (row0 + ty * kPer + i) / a.group);
#pragma unroll
      for (int c = 0; c < 2 * kQuads; ++c) o[i][c] = 0;
    }
    for (int b = g.block_begin; b < g.block_end; ++b) {
      const int key0 = b * kKeys;
      copy_wait<1>();    // the keys
      __syncthreads();
      uint64_t x2[kPer][4] = {};   // sums over even and odd d
#pragma unroll 4
      for (int d = 0; d < a.dim; d += 4) {
        ulonglong2 qv[kPer], kv[4];
#pragma unroll
        for (int i = 0; i < kPer; ++i) qv[i] = pairs_at(qs + (ty * kPer + i) * pitch + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) kv[j] = pairs_at(ks + (tx + 16 * j) * pitch + d);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) x2[i][j] = fma_f32x2(qv[i].y, kv[j].y, fma_f32x2(qv[i].x, kv[j].x, x2[i][j]));
      }
      __syncthreads();   // the keys have been read
      copy_block(ks, k, a.k_row[s], b + 1);
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float x[4], top = kMinusInf;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 pair = unpack_f32x2(x2[i][j]);
          x[j] = key0 + tx + 16 * j < seen[i] ? pair.x + pair.y : kMinusInf;   // chosen, not added: the product may be NaN
          top = fmaxf(top, x[j]);
        }
        const float next = fmaxf(m[i], half_warp_max(top));
        const float base = next == kMinusInf ? 0.f : next;   // nothing seen yet: all terms are 2^(-inf)
        const float keep = exp2f(m[i] - base);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = exp2f(x[j] - base);
          ps[(ty * kPer + i) * kPitchP + tx + 16 * j] = p;
          sum += p;
        }
        l[i] = l[i] * keep + half_warp_sum(sum);
        m[i] = next;
        const uint64_t keep2 = pack_f32x2(keep, keep);
#pragma unroll
        for (int c = 0; c < 2 * kQuads; ++c) o[i][c] = fma_f32x2(o[i][c], keep2, 0);
      }
      copy_wait<1>();    // the values
      __syncthreads();
#pragma unroll 4
      for (int key = 0; key < kKeys; key += 4) {
        float4 p[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) p[i] = *reinterpret_cast<const float4*>(ps + (ty * kPer + i) * kPitchP + key);
#pragma unroll
        for (int c = 0; c < kQuads; ++c) {
          const int d = tx * 4 + 64 * c;
          if (d < a.dim) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const ulonglong2 w = pairs_at(vs + (key + e) * pitch + d);
#pragma unroll
              for (int i = 0; i < kPer; ++i) {
                const float pe = e == 0 ? p[i].x : e == 1 ? p[i].y : e == 2 ? p[i].z : p[i].w;
                const uint64_t pe2 = pack_f32x2(pe, pe);
                o[i][2 * c] = fma_f32x2(pe2, w.x, o[i][2 * c]), o[i][2 * c + 1] = fma_f32x2(pe2, w.y, o[i][2 * c + 1]);
              }
            }
          }
        }
      }
      __syncthreads();   // the values have been read
      copy_block(vs, v, a.v_row[s], b + 1);
    }
    copy_wait<0>();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = ty * kPer + i;
      if (r >= rows) continue;
      const bool partial = is_partial(a, g);
      if (partial && tx == 0) a.partial_ml[slot + r] = make_float2(m[i], l[i]);
      const float inv = partial ? 1.f : l[i] == 0.f ? 0.f : 1.f / l[i];
      float* y = partial ? a.partial_o + slot * a.dim + r * 4 : static_cast<float*>(a.out) + output_row(a, g.seq.q_row, g.head, row0 + r) * a.dim;
#pragma unroll
      for (int c = 0; c < kQuads; ++c) {
        const int quad = tx + 16 * c;
        if (quad * 4 >= a.dim) continue;
        const float2 lo = unpack_f32x2(o[i][2 * c]), hi = unpack_f32x2(o[i][2 * c + 1]);
        store4(y + (partial ? static_cast<int64_t>(quad) * slot_rows : quad) * 4, make_float4(lo.x * inv, lo.y * inv, hi.x * inv, hi.y * inv));
      }
    }
  }
}

constexpr size_t simt_smem_bytes(int rows, int dim) {
  return sizeof(float) * ((rows + 2 * static_cast<size_t>(kKeys)) * (dim + 4) + static_cast<size_t>(rows) * (kKeys + 4));
}

template <int kRows, int kThreads, int kColumns, typename Line>
int launch_line(const AttentionArgs& a, cudaStream_t s) {
  if (!ensure_dynamic_smem<attention_simt_kernel<kRows, kThreads, kColumns, Line>, simt_smem_bytes(kRows, kColumns)>()) return B200_ERR_LAUNCH_FAILED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = simt_smem_bytes(kRows, a.dim);
  cfg.stream = s;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  if (cudaLaunchKernelEx(&cfg, attention_simt_kernel<kRows, kThreads, kColumns, Line>, a) != cudaSuccess) return launch_failed();
  return launch_status();
}

template <int kRows, int kThreads, int kColumns>
int launch_columns(const AttentionArgs& a, cudaStream_t s) {
  return wide_line(a) ? launch_line<kRows, kThreads, kColumns, int64_t>(a, s) : launch_line<kRows, kThreads, kColumns, int>(a, s);
}

template <int kRows, int kThreads>
int launch(const AttentionArgs& a, cudaStream_t s) {
  return a.dim <= 64 ? launch_columns<kRows, kThreads, 64>(a, s) : launch_columns<kRows, kThreads, 128>(a, s);
}

// The smallest tile that holds the rows that a sequence has on average, and a whole token.
int tile_of(const AttentionArgs& a) {
  const int64_t rows = a.kind == kShared ? a.group : static_cast<int64_t>(a.q_rows) * a.group / (a.sequences > 0 ? a.sequences : 1);
  const int64_t needed = rows > a.group ? rows : a.group;
  return needed <= 16 ? 16 : needed <= 64 ? 64 : 128;
}

}  // namespace

void plan_attention_simt(AttentionArgs* a, int sms) {
  const int tile = tile_of(*a);
  a->tokens = tile / a->group;
  a->unit_rows = a->tokens * a->group;
  a->unit_cost = 1, a->pair_shift = 0;
  // As many CTAs as an SM's shared memory holds, up to what its registers do.
  const int fit = static_cast<int>((227 * 1024) / (simt_smem_bytes(tile, a->dim) + 2048));
  const int most = tile == 16 ? 4 : tile == 64 ? 2 : 1;
  a->ctas = sms * (fit < 1 ? 1 : fit < most ? fit : most);
}

int launch_attention_simt(const AttentionArgs& a, cudaStream_t s) {
  const int tile = tile_of(a);
  return tile == 16 ? launch<16, 128>(a, s) : tile == 64 ? launch<64, 256>(a, s) : launch<128, 256>(a, s);
}

}  // namespace b200
