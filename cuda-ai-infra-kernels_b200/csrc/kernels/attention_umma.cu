// Attention for 16-bit operands on the 5th-generation tensor cores.
//
// For a tile of 128 rows and a block of 128 keys: S = Q K^T into tensor memory (tcgen05.mma, both
// operands in shared memory), the row maxima and P = 2^(scale S - m) in registers, one thread per
// row, P back into tensor memory as a 16-bit operand in the columns that held S, and O += P V with P
// read from there. O stays in tensor memory for the whole unit. P is rounded to the operand type
// (relative 2^-9 or 2^-12 per probability, of the size of the output's own rounding); the denominator
// adds up the unrounded FP32 values.
//
// The products of one block take about as long as its exponentials, and each waits for the other.
// Two streams therefore alternate, each with its own S and O: the tensor pipe works for one while
// the warps work for the other. The streams are the two row tiles of a unit of 256 rows, over the
// same blocks of keys; or, where a unit has at most one tile of rows (a decoding request, a short
// prompt), the even and the odd blocks for the same tile, joined at the end: thread r of both groups
// of warps owns row r and may read both accumulators.
//
// The maximum is followed lazily: O and the denominator are rescaled only when a row's maximum has
// grown by more than 2^8 since the last time, which the first block or two settle. Until then
// P <= 256 and nothing overflows; the quotient is the same.
//
// Warps 0-3 and 4-7: streams 0 and 1, warp w owning TMEM lanes 32 (w mod 4) ... Warp 8: copies (TMA).
// Warp 9: issues the MMAs, and clears the value rows behind the last key of a sequence, which hold
// foreign data that 0 * NaN would let in.
#include "attention.cuh"

namespace b200 {

cudaError_t attention_status_read_clear(uint32_t* word) { return status_word_read_clear(word); }

namespace {

constexpr int kThreads = 320;
constexpr int kTile = 128;          // rows of a tile, keys of a block
constexpr float kMinusInf = -__builtin_huge_valf();
constexpr float kLazy = 8.f;        // growth of a maximum, in powers of two, that forces a rescale
constexpr uint32_t kColS = 0, kColO = 256, kColStream = 128;   // TMEM columns

struct UmmaAttentionArgs {
  CUtensorMap q, k[2], v[2];
  AttentionArgs a;
};

template <int kDim>
struct Smem {
  static constexpr int kHalves = kDim / 64;                 // 128-byte spans per row
  static constexpr int kHalfBytes = kTile * 128;
  static constexpr int kTileBytes = kHalves * kHalfBytes;   // a tile of Q, a block of K or of V
  static constexpr int kSlots = kDim == 128 ? 5 : 10;
  static constexpr size_t kTiles = (2 + kSlots) * static_cast<size_t>(kTileBytes);
};

struct Shared {   // behind the tiles
  uint64_t full[10], empty[10];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_ready[2];
  uint64_t o_full, o_empty;
  uint32_t tmem;
  float2 exchange[2][kTile];   // maximum and denominator of both streams
  WorkScratch scratch;
};

// After tcgen05.wait::ld: keeps uses of loaded registers behind the wait.
template <int kN>
__device__ __forceinline__ void loaded(float (&v)[kN]) {
#pragma unroll
  for (int i = 0; i < kN; ++i) asm volatile("" : "+f"(v[i]));
}

// Thread t of a warp: 32 columns of lane (base lane + t).
__device__ __forceinline__ void load_columns(uint32_t at, float (&v)[32]) {
  tmem_ld_32x32(at, *reinterpret_cast<uint32_t(*)[32]>(&v));
  tmem_ld_wait();
  loaded(v);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if constexpr (kBf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// How the two streams share a segment.
struct Shape {
  int blocks;
  bool pair;   // two row tiles over all blocks; else one tile, even and odd blocks
  __device__ __forceinline__ int items() const { return pair ? 2 * blocks : blocks; }
  __device__ __forceinline__ int of_stream(int s) const { return pair ? blocks : (blocks + 1 - s) / 2; }
};
__device__ __forceinline__ Shape shape_of(const AttentionArgs& a, const Segment& g) {
  const int64_t rows = static_cast<int64_t>(g.seq.n) * a.group - static_cast<int64_t>(g.unit) * a.unit_rows;
  return Shape{g.block_end - g.block_begin, rows > a.unit_rows / 2};
}

// ------------------------------------------------------------------------------------- copies

template <int kDim>
__device__ __forceinline__ void copy_role(const UmmaAttentionArgs& p, const WorkStart& start, uint8_t* smem, Shared* b) {
  using S = Smem<kDim>;
  const AttentionArgs& a = p.a;
  const int tokens = a.unit_rows / 2 / a.group;   // of a tile
  SegmentWalk<kUmmaKeyBlock> walk(a, start);
  Segment g;
  bool ok = true;
  uint32_t load = 0, segment = 0;
  while (walk.next(&g)) {
    const Shape shape = shape_of(a, g);
    if (shape.blocks == 0) continue;
    ok = ok && mbar_wait(&b->q_empty, (segment & 1) ^ 1, kSiteAttention);
    ++segment;
    if (!ok) return;
    const int tiles = shape.pair ? 2 : 1;
    mbar_expect_tx(&b->q_full, tiles * S::kHalves * tokens * a.group * 128);
    for (int t = 0; t < tiles; ++t)
      for (int h = 0; h < S::kHalves; ++h)
        tma_load_3d(smem + t * S::kTileBytes + h * S::kHalfBytes, &p.q, &b->q_full, h * 64, g.head * a.group,
                    g.seq.q_row + (2 * g.unit + t) * tokens);
    const auto block = [&](const CUtensorMap* map, int i) {
      const uint32_t slot = load % S::kSlots, round = load / S::kSlots;
      ++load;
      ok = ok && mbar_wait(&b->empty[slot], (round & 1) ^ 1, kSiteAttention);
      if (!ok) return;
      mbar_expect_tx(&b->full[slot], S::kTileBytes);
      for (int h = 0; h < S::kHalves; ++h)
        tma_load_4d(smem + (2 + slot) * S::kTileBytes + h * S::kHalfBytes, map, &b->full[slot], h * 64, g.head,
                    g.seq.k_row + (g.block_begin + i) * kTile, g.seq.batch);
    };
    // In the order in which the MMAs will want them.
    const CUtensorMap *k = &p.k[g.seq.source], *v = &p.v[g.seq.source];
    const int ahead = shape.pair ? 1 : 2;
    for (int i = 0; i < ahead && i < shape.blocks; ++i) block(k, i);
    for (int i = 0; i < shape.blocks; ++i) {
      block(v, i);
      if (i + ahead < shape.blocks) block(k, i + ahead);
    }
  }
}

// --------------------------------------------------------------------------------------- MMAs

template <int kDim, bool kBf16>
__device__ __forceinline__ void mma_role(const UmmaAttentionArgs& p, const WorkStart& start, uint8_t* smem, Shared* b, uint32_t tmem) {
  using S = Smem<kDim>;
  const AttentionArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  const uint32_t idesc_s = umma_idesc_f16(kTile, kTile, kBf16, false, false);
  const uint32_t idesc_o = umma_idesc_f16(kTile, (a.dim + 15) / 16 * 16, kBf16, false, true);
  const int steps = (a.dim + 15) / 16;   // of 16 along the head dimension; what lies behind it reads as zero
  SegmentWalk<kUmmaKeyBlock> walk(a, start);
  Segment g;
  bool ok = true;
  uint32_t load = 0, segment = 0, item[2] = {0, 0};
  while (walk.next(&g)) {
    const Shape shape = shape_of(a, g);
    if (shape.blocks == 0) continue;
    ok = ok && mbar_wait(&b->q_full, segment & 1, kSiteAttention);
    uint32_t k_slot = 0, v_slot = 0;
    const auto arrived = [&]() {   // the next block of the ring
      const uint32_t slot = load % S::kSlots, round = load / S::kSlots;
      ++load;
      ok = ok && mbar_wait(&b->full[slot], round & 1, kSiteAttention);
      return slot;
    };
    const int items = shape.items();
    const auto block_of = [&](int j) { return shape.pair ? j / 2 : j; };
    const auto first_use = [&](int j) { return !shape.pair || j % 2 == 0; };
    const auto last_use = [&](int j) { return !shape.pair || j % 2 == 1; };
    const auto scores = [&](int j) {
      if (first_use(j)) k_slot = arrived();
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      if (lane == 0) {
        tcgen05_fence_after_sync();
        const uint32_t q_at = smem_u32(smem) + (shape.pair ? (j & 1) * S::kTileBytes : 0);
        const uint32_t k_at = smem_u32(smem) + (2 + k_slot) * S::kTileBytes;
        const uint64_t qd = umma_smem_desc(q_at, 16, 1024, kUmmaSwizzle128B), kd = umma_smem_desc(k_at, 16, 1024, kUmmaSwizzle128B);
        for (int step = 0; step < steps; ++step) {
          const uint32_t at = (step >> 2) * S::kHalfBytes + (step & 3) * 32;
          umma_f16(tmem + kColS + (j & 1) * kColStream, umma_desc_advance(qd, at), umma_desc_advance(kd, at), idesc_s, step > 0);
        }
        if (last_use(j)) umma_commit(&b->empty[k_slot]);
        if (j + 1 == items) umma_commit(&b->q_empty);
        umma_commit(&b->s_full[j & 1]);
      }
      __syncwarp();
    };
    for (int j = 0; j < 2 && j < items; ++j) scores(j);
    for (int j = 0; j < items; ++j) {
      const int s = j & 1;
      if (first_use(j)) {
        v_slot = arrived();
        const int live = g.seq.m - (g.block_begin + block_of(j)) * kTile;
        if (ok && live < kTile) {   // rows of other owners: zero, whatever they are
          uint8_t* v = smem + (2 + v_slot) * S::kTileBytes;
          for (int i = live * 8 + lane; i < kTile * 8; i += 32)
            for (int h = 0; h < S::kHalves; ++h)
              *reinterpret_cast<uint4*>(v + h * S::kHalfBytes + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
      }
      if (j == 0) ok = ok && mbar_wait(&b->o_empty, (segment & 1) ^ 1, kSiteAttention);
      ok = ok && mbar_wait(&b->p_ready[s], item[s] & 1, kSiteAttention);
      ++item[s];
      ok = __all_sync(0xffffffffu, ok);
      if (ok && lane == 0) {
        tcgen05_fence_after_sync();
        const uint64_t vd = umma_smem_desc(smem_u32(smem) + (2 + v_slot) * S::kTileBytes, S::kHalfBytes, 1024, kUmmaSwizzle128B);
        for (int step = 0; step < kTile / 16; ++step)
          umma_f16_tmem_a(tmem + kColO + s * kColStream, tmem + kColS + s * kColStream + step * 8, umma_desc_advance(vd, step * 2048), idesc_o,
                          j >= 2 || step > 0);
        if (last_use(j)) umma_commit(&b->empty[v_slot]);
        if (j + 1 == items) umma_commit(&b->o_full);
      }
      __syncwarp();
      if (j + 2 < items) scores(j + 2);
    }
    ++segment;
  }
}

// ------------------------------------------------------------------------------------ softmax

// The thread's row of a stream.
struct RowState {
  float m, l;   // base of the exponentials (scaled, base 2) and denominator
};

template <bool kBf16, bool kMasked>
__device__ __forceinline__ void softmax_block(uint32_t s_at, uint32_t o_at, int chunks, int seen, float scale, bool first, RowState* row) {
  float x[kTile];
#pragma unroll
  for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_at + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&x[32 * c]));
  tmem_ld_wait();
  loaded(x);
  float top[4] = {kMinusInf, kMinusInf, kMinusInf, kMinusInf};
#pragma unroll
  for (int i = 0; i < kTile; ++i) {
    if (kMasked && i >= seen) x[i] = kMinusInf;   // chosen, not added: the product may be NaN
    top[i & 3] = fmaxf(top[i & 3], x[i]);
  }
  const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
  if (first) {
    row->m = m;
  } else {
    const bool grown = m > row->m + kLazy;
    if (__any_sync(0xffffffffu, grown)) {
      const float next = grown ? m : row->m;
      const float keep = grown ? exp2_fast(row->m - next) : 1.f;
      row->l *= keep;
      row->m = next;
      for (int c = 0; c < chunks; ++c) {
        float o[32];
        load_columns(o_at + 32 * c, o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] *= keep;
        tmem_st_32x32(o_at + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&o));
      }
    }
  }
  const float base = row->m == kMinusInf ? 0.f : row->m;   // nothing seen yet: all terms are 2^(-inf)
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint32_t packed[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float lo = exp2_fast(fmaf(x[64 * half + 2 * i], scale, -base)), hi = exp2_fast(fmaf(x[64 * half + 2 * i + 1], scale, -base));
      sum[(2 * i) & 3] += lo, sum[(2 * i + 1) & 3] += hi;
      packed[i] = pack<kBf16>(lo, hi);
    }
    tmem_st_32x32(s_at + 32 * half, packed);
  }
  row->l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  tmem_st_wait();
}

// 32 finished columns of a row.
template <bool kBf16>
__device__ __forceinline__ void store_columns(const AttentionArgs& a, int64_t row, int column, const float (&y)[32]) {
  if (a.split != 0) {
    float* out = a.partial_o + row * a.dim + column;
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      if (column + i < a.dim) *reinterpret_cast<float4*>(out + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
  } else {
    uint16_t* out = static_cast<uint16_t*>(a.out) + row * a.dim + column;
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      if (column + i < a.dim)
        *reinterpret_cast<uint4*>(out + i) = make_uint4(pack<kBf16>(y[i], y[i + 1]), pack<kBf16>(y[i + 2], y[i + 3]),
                                                        pack<kBf16>(y[i + 4], y[i + 5]), pack<kBf16>(y[i + 6], y[i + 7]));
  }
}

template <bool kBf16>
__device__ __forceinline__ void softmax_role(const UmmaAttentionArgs& p, const WorkStart& start, Shared* b, uint32_t tmem) {
  const AttentionArgs& a = p.a;
  const int s = threadIdx.x >> 7;                    // stream
  const int r = threadIdx.x & 127;                   // row of the tile, TMEM lane
  const int warp_row = r & ~31, lane = r & 31;
  const uint32_t lanes = static_cast<uint32_t>(warp_row) << 16;
  const uint32_t s_at = tmem + lanes + kColS + s * kColStream, o_at = tmem + lanes + kColO + s * kColStream;
  const int tile_rows = a.unit_rows / 2;
  const int chunks = (a.dim + 31) / 32;
  SegmentWalk<kUmmaKeyBlock> walk(a, start);
  Segment g;
  bool ok = true;
  uint32_t segment = 0, item = 0;
  while (walk.next(&g)) {
    const Shape shape = shape_of(a, g);
    const int64_t rows = static_cast<int64_t>(g.seq.n) * a.group;
    const int64_t tile0 = static_cast<int64_t>(g.unit) * a.unit_rows + (shape.pair && s == 1 ? tile_rows : 0);
    const int64_t flat = tile0 + r;
    const bool live = r < tile_rows && flat < rows;
    const bool warp_live = warp_row < tile_rows && tile0 + warp_row < rows;   // some row of the warp is there
    RowState row{kMinusInf, 0.f};
    if (shape.blocks > 0) {
      const int seen = live ? visible_keys(a, g.seq, static_cast<int>(flat / a.group)) : 0;
      // All rows of the warp that are there see at least what its first row sees.
      const int seen_by_all = warp_live ? visible_keys(a, g.seq, static_cast<int>((tile0 + warp_row) / a.group)) : 0;
      const int items = shape.of_stream(s);
      for (int i = 0; i < items; ++i) {
        const int key0 = (g.block_begin + (shape.pair ? i : 2 * i + s)) * kTile;
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&b->s_full[s], item & 1, kSiteAttention));
        ++item;
        if (ok && warp_live) {
          tcgen05_fence_after_sync();
          if (key0 + kTile <= seen_by_all) softmax_block<kBf16, false>(s_at, o_at, chunks, 0, a.scale_log2, i == 0, &row);
          else softmax_block<kBf16, true>(s_at, o_at, chunks, seen - key0, a.scale_log2, i == 0, &row);
          tcgen05_fence_before_sync();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->p_ready[s]);
      }
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&b->o_full, segment & 1, kSiteAttention));
      ++segment;
      tcgen05_fence_after_sync();
    }
    // Rows of one tile that two streams worked on: the same thread of both warp groups owns them, and
    // each finishes every other 32 columns.
    float mine = 1.f, other = 0.f, total = row.l, base = row.m;
    const bool joined = !shape.pair && shape.blocks > 1;
    if (joined) {
      b->exchange[s][r] = make_float2(row.m, row.l);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const float2 peer = b->exchange[s ^ 1][r];
      base = fmaxf(row.m, peer.x);
      const float zero = base == kMinusInf ? 0.f : base;
      mine = exp2_fast(row.m - zero), other = exp2_fast(peer.x - zero);
      total = row.l * mine + peer.y * other;
      asm volatile("bar.sync 1, 256;" ::: "memory");   // read by all before the next segment writes
    }
    if (ok && warp_live && (shape.pair || s == 0 || joined)) {
      const int64_t at = live ? (a.split != 0 ? partial_row(a, g, flat) : output_row(a, g, flat)) : 0;
      if (a.split != 0 && live && (shape.pair || s == 0)) a.partial_ml[at] = make_float2(base, total);
      const float inv = a.split != 0 ? 1.f : (total == 0.f ? 0.f : 1.f / total);
      const float f0 = mine * inv, f1 = other * inv;
      for (int c = joined ? s : 0; c < chunks; c += joined ? 2 : 1) {
        float y[32];
        if (shape.blocks > 0) {
          load_columns(o_at + 32 * c, y);
          // A row that saw nothing keeps its zeros whatever its accumulator holds.
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = total == 0.f ? 0.f : y[i] * f0;
          if (joined) {
            float z[32];
            load_columns(tmem + lanes + kColO + (s ^ 1) * kColStream + 32 * c, z);
#pragma unroll
            for (int i = 0; i < 32; ++i) y[i] = total == 0.f ? 0.f : y[i] + z[i] * f1;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = 0.f;
        }
        if (live) store_columns<kBf16>(a, at, 32 * c, y);
      }
    }
    if (shape.blocks > 0) {
      tcgen05_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b->o_empty);
    }
  }
}

template <int kDim, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1) attention_umma_kernel(const __grid_constant__ UmmaAttentionArgs p) {
  using S = Smem<kDim>;
  extern __shared__ __align__(1024) uint8_t smem[];   // the swizzle's period
  Shared& bars = *reinterpret_cast<Shared*>(smem + S::kTiles);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&p.q);
    for (int s = 0; s < S::kSlots; ++s) mbar_init(&bars.full[s], 1), mbar_init(&bars.empty[s], 1);
    mbar_init(&bars.q_full, 1), mbar_init(&bars.q_empty, 1);
    for (int s = 0; s < 2; ++s) mbar_init(&bars.s_full[s], 1), mbar_init(&bars.p_ready[s], 4);
    mbar_init(&bars.o_full, 1), mbar_init(&bars.o_empty, 8);
    mbar_init_fence();
  }
  if (warp == 9) {
    tmem_alloc<512>(&bars.tmem);
    tmem_relinquish();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = bars.tmem;
  grid_launch_dependents();   // after the allocation: a following kernel may want tensor memory too
  grid_dependency_wait();
  const WorkStart start = find_attention_work<kUmmaKeyBlock, kThreads>(p.a, &bars.scratch);
  if (warp < 8) {
    softmax_role<kBf16>(p, start, &bars, tmem);
  } else if (warp == 8) {
    if (lane == 0) copy_role<kDim>(p, start, smem, &bars);
  } else {
    mma_role<kDim, kBf16>(p, start, smem, &bars, tmem);
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  if (warp == 9) tmem_dealloc<512>(tmem);
}

template <int kDim, bool kBf16>
int launch(const UmmaAttentionArgs& p, int64_t blocks, cudaStream_t s) {
  constexpr size_t kBytes = Smem<kDim>::kTiles + sizeof(Shared);
  static_assert(kBytes <= 227 * 1024, "shared memory of one CTA");
  if (!ensure_dynamic_smem<attention_umma_kernel<kDim, kBf16>, kBytes>()) return B200_ERR_LAUNCH_FAILED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = s;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  if (cudaLaunchKernelEx(&cfg, attention_umma_kernel<kDim, kBf16>, p) != cudaSuccess) return launch_failed();
  return launch_status();
}

// [rows][heads][dim] as (dim, heads, rows, batch); a box is one head's 128 rows, 64 columns.
bool make_key_map(CUtensorMap* out, const void* base, const AttentionArgs& a, int64_t rows, int64_t row_stride, int64_t head_stride,
                  int64_t batch, int64_t batch_stride) {
  const uint64_t dims[4] = {static_cast<uint64_t>(a.dim), static_cast<uint64_t>(a.kv_heads), static_cast<uint64_t>(rows),
                            static_cast<uint64_t>(batch)};
  // The stride of a dimension with one entry is never used, but has to be a valid one.
  const auto stride = [&](int64_t elements, uint64_t entries) { return static_cast<uint64_t>(entries > 1 ? elements : a.dim) * 2; };
  const uint64_t strides[3] = {stride(head_stride, dims[1]), stride(row_stride, dims[2]), stride(batch_stride, dims[3])};
  const uint32_t box[4] = {64, 1, kTile, 1};
  return make_tensor_map_16bit(out, base, 4, dims, strides, box, a.dtype == B200_BF16);
}

}  // namespace

void plan_attention_umma(AttentionArgs* a, int sms) {
  // Tiles hold whole tokens: a copy brings (dim, group, tokens) boxes.
  a->unit_rows = 2 * (kTile / a->group) * a->group;
  a->ctas = sms;
}

int launch_attention_umma(const AttentionArgs& a, cudaStream_t s, int64_t units) {
  const int64_t blocks = a.split != 0 ? a.ctas : units * a.kv_heads;
  if (blocks > 0x7fffffffLL) return B200_ERR_INVALID_PROBLEM;
  UmmaAttentionArgs p;
  p.a = a;
  const bool bf16 = a.dtype == B200_BF16;
  const auto entries = [](int64_t n) { return static_cast<uint64_t>(n > 1 ? n : 1); };
  const uint64_t dims[3] = {static_cast<uint64_t>(a.dim), static_cast<uint64_t>(a.heads), entries(a.q_rows)};
  const uint64_t strides[2] = {static_cast<uint64_t>(a.heads > 1 ? a.q_head : a.dim) * 2, static_cast<uint64_t>(a.q_rows > 1 ? a.q_row : a.dim) * 2};
  const uint32_t box[3] = {64, static_cast<uint32_t>(a.group), static_cast<uint32_t>(kTile / a.group)};
  bool ok = make_tensor_map_16bit(&p.q, a.q, 3, dims, strides, box, bf16);
  // An array without rows is never copied from; its map describes some other memory.
  for (int i = 0; i < 2; ++i) {
    const int64_t rows = i == 0 ? a.k_rows : a.room, batch = i == 0 ? 1 : a.q_rows;
    const bool there = i == 0 ? rows > 0 : a.kind == kShared && rows > 0;
    if (there) {
      ok = ok && make_key_map(&p.k[i], a.k[i], a, rows, a.k_row[i], a.k_head[i], batch, a.k_batch) &&
           make_key_map(&p.v[i], a.v[i], a, rows, a.v_row[i], a.v_head[i], batch, a.v_batch);
    } else {
      p.k[i] = p.v[i] = p.q;
    }
  }
  if (!ok) return B200_ERR_INVALID_PROBLEM;
  if (a.dim <= 64) return bf16 ? launch<64, true>(p, blocks, s) : launch<64, false>(p, blocks, s);
  return bf16 ? launch<128, true>(p, blocks, s) : launch<128, false>(p, blocks, s);
}

}  // namespace b200
