// Attention for 16-bit operands on the 5th-generation tensor cores.
//
// For a tile of 128 rows and 64 keys: S = Q K^T into tensor memory (tcgen05.mma, both operands in
// shared memory), the row maxima and P = 2^(scale S - m) in registers, one thread per row, P back into
// tensor memory as a 16-bit operand in columns that held S, and O += P V with P read from there. O
// stays in tensor memory for the whole unit. P is rounded to the operand type (at most 2^-8 or 2^-11
// of a probability, as the output's own rounding); the denominator adds up the unrounded
// FP32 values. FP16 holds P times 2^7, which it has the room for: unscaled, a probability below 2^-14 of
// the largest would be subnormal and one below 2^-25 nothing, and 100000 such keys are 0.003 of the row.
// So the limits are 2^-21 and 2^-32, and what is lost below them is at most 2^-32 per key.
//
// Two streams, each with its own group of four warps, O and S: the two row tiles of a unit of 256
// rows, over the same blocks of 128 keys; or, where a unit has at most one tile of rows (a decoding
// request, a short prompt), the first and the second 64 keys of each block for the same tile, joined
// at the end: thread r of both groups of warps owns row r and may read both accumulators. (Even and odd
// blocks instead kept two blocks at a time in the ring, whose next copies then came too late: a block
// took as long as one of two tiles.) Each stream has two S: while the
// warps work on one half block of 64 keys, the tensor pipe multiplies the P of the half before and
// fills its place with the scores of the half after, so that neither waits for the other. (One S of
// 128 keys per stream left the warps idle during the products: 4400 cycles per block of both streams
// against the pipe's 2048.)
//
// The maximum is followed lazily: O and the denominator are rescaled only when a row's maximum has
// grown by more than 2^8 since the last time, which the first block or two settle. Until then
// P <= 2^8 (FP16: 2^15) and nothing overflows; the quotient is the same.
//
// Warps 0-3 and 4-7: streams 0 and 1, warp w owning TMEM lanes 32 (w mod 4) ... Warp 8: copies (TMA).
// Warps 9 and 10: one MMA-issuing thread per stream (a lone thread spends as long on barriers and
// commits as the tensor pipe on its products, and held the pipe at half its rate; with two, one
// waits while the other issues). Warp 11 walks the CTA's segments and hands them out through a small
// ring, so that nobody else carries the walk's state or waits for its arithmetic; and it clears
// the value rows behind the last key of a sequence, which hold foreign data that 0 * NaN would let in.
#include "attention.cuh"

namespace b200 {

cudaError_t attention_status_read_clear(uint32_t* word) { return status_word_read_clear(word); }

namespace {

constexpr int kThreads = 384;
// Registers: 168 per thread at launch; a softmax thread holds 64 scores, or 32 columns of both accumulators.
constexpr int kSoftmaxRegisters = 216, kOtherRegisters = 72;
static_assert(256 * kSoftmaxRegisters + 128 * kOtherRegisters <= kThreads * 168, "registers of the CTA");
constexpr int kTile = 128;          // rows of a tile, keys of a block
constexpr float kMinusInf = -__builtin_huge_valf();
constexpr float kLazy = 8.f;        // growth of a maximum, in powers of two, that forces a rescale
constexpr float kRaiseFp16 = 7.f;   // FP16 holds P times 2^7
constexpr int kHalf = 64;           // keys of one S
constexpr uint32_t kColS = 0, kColO = 256, kColStream = 128, kColHalf = 64;   // TMEM columns

struct UmmaAttentionArgs {
  CUtensorMap q, k[2], v[2], out;
  int boxed;   // a warp's 32 rows of the output are a box of `out`
  AttentionArgs a;
};

template <int kDim>
struct Smem {
  static constexpr int kHalves = kDim / 64;                 // 128-byte spans per row
  static constexpr int kHalfBytes = kTile * 128;
  static constexpr int kTileBytes = kHalves * kHalfBytes;   // a tile of Q, a block of K or of V
  static constexpr int kSlots = kDim == 128 ? 4 : 8;
  static constexpr size_t kStaging = (2 + kSlots) * static_cast<size_t>(kTileBytes);   // 4 KiB per softmax warp
  static constexpr size_t kTiles = kStaging + 8 * 4096;
};

// What the roles need of a segment (attention.cuh), for a unit of whole tokens.
struct SegmentEntry {
  int blocks;              // of keys; -1: no more segments
  int pair;                // two row tiles over all keys; else one tile, its keys shared by the streams
  int q_row, tokens;       // the unit's first query row, and tokens from there to the sequence's end
  int k_row, batch, source, head;   // k_row: of the first block
  int keys, ahead;         // from the first block on: keys of the sequence; keys that token t of the unit sees
                           // are ahead + t, cut to 0 .. keys
  int halves;              // half blocks that some row sees: 2 * blocks, or one less
  int live_keys;           // of the last block
  int partial, pitch;
  int64_t slot;            // of the partial result
};
constexpr int kEntries = 4;

struct Shared {   // behind the tiles
  uint64_t full[8], empty[8], raw[8];
  uint64_t entry_full[kEntries], entry_empty[kEntries];
  uint64_t q_full, q_empty;
  uint64_t s_full[2][2], p_ready[2][2];   // [stream][half]
  uint64_t drained[2];         // all products but the last half's are in the accumulator
  uint64_t o_full[2], o_empty[2];
  uint64_t exchanged;          // eight warps have written, then eight have read
  uint32_t tmem;
  SegmentEntry entries[kEntries];
  float2 exchange[2][kTile];   // maximum and denominator of both streams
  WorkScratch<int64_t> scratch;
};
constexpr int kEntryReaders = 1 + 2 + 8;

// Half blocks of a stream: all of the segment's, or every other one.
__device__ __forceinline__ int items_of(const SegmentEntry& e, int s) { return e.pair != 0 ? e.halves : (e.halves + 1 - s) / 2; }

// A role's place in the ring of segments. Called by whole warps or by single threads.
struct EntryReader {
  Shared* b;
  uint32_t count = 0;
  bool ok = true;
  __device__ __forceinline__ const SegmentEntry* wait() {
    ok = ok && mbar_wait(&b->entry_full[count % kEntries], count / kEntries & 1, kSiteAttention);
    return &b->entries[count % kEntries];
  }
  __device__ __forceinline__ void release() { mbar_arrive(&b->entry_empty[count++ % kEntries]); }
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

// ------------------------------------------------------------------------ segments, value rows

template <int kDim, typename Line>
__device__ __forceinline__ void segment_role(const UmmaAttentionArgs& p, const WorkStart<Line>& start, uint8_t* smem, Shared* b) {
  using S = Smem<kDim>;
  const AttentionArgs& a = p.a;
  const int lane = threadIdx.x & 31;
  SegmentWalk<kUmmaKeyBlock, Line> walk(a, start);
  Segment g;
  bool ok = true;
  if (lane == 0) start_records(a);
  // Blocks whose last rows have to be cleared, at most kDelay segments behind the newest: the slot of
  // the ring and the live rows.
  constexpr uint32_t kDelay = 2;
  int dirty[kDelay] = {-1, -1}, live_of[kDelay] = {0, 0};
  uint32_t loads = 0, raw_phase = 0;
  const auto clear = [&](int i) {
    const int slot = dirty[i];
    if (slot < 0) return;
    dirty[i] = -1;
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&b->raw[slot], raw_phase >> slot & 1, kSiteAttention));
    raw_phase ^= 1u << slot;
    if (!ok) return;
    uint8_t* v = smem + (2 + slot) * S::kTileBytes;
    for (int j = live_of[i] * 8 + lane; j < kTile * 8; j += 32)
#pragma unroll
      for (int h = 0; h < S::kHalves; ++h) *reinterpret_cast<uint4*>(v + h * S::kHalfBytes + j * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&b->full[slot]);
  };
  for (uint32_t count = 0;; ++count) {
    const bool more = walk.next(&g);
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&b->entry_empty[count % kEntries], (count / kEntries & 1) ^ 1, kSiteAttention));
    SegmentEntry e{};
    if (more) {
      const int first = g.block_begin * kTile, token0 = g.unit * a.tokens;
      e.blocks = g.block_end - g.block_begin;
      e.tokens = g.seq.n - token0;
      e.pair = e.tokens > a.tokens / 2;
      e.q_row = g.seq.q_row + token0, e.k_row = g.seq.k_row + first;
      e.batch = g.seq.batch, e.source = g.seq.source, e.head = g.head;
      e.keys = g.seq.m - first;
      e.ahead = a.kind == kShared || a.causal == 0 ? e.keys : g.seq.m - g.seq.n + token0 + 1 - first;
      e.halves = 2 * e.blocks;
      if (e.blocks > 0) {   // the unit's last row sees most
        const int seen = clamp_int(e.ahead + min(a.tokens, e.tokens) - 1, 0, e.keys);
        if (seen <= e.blocks * kTile - kHalf) --e.halves;
      }
      e.live_keys = min(kTile, g.seq.m - (g.block_end - 1) * kTile);
      e.partial = is_partial(a, g);
      e.slot = slot_of(a, g, &e.pitch);
      if (lane == 0) record(a, g);
    } else {
      e.blocks = -1;
    }
    if (lane == 0) {
      b->entries[count % kEntries] = e;
      mbar_arrive(&b->entry_full[count % kEntries]);
    }
    clear(count % kDelay);   // the segment before the last one
    if (!more) {
      clear((count + 1) % kDelay);
      clear_unowned_rows(a, start.sequence == kRefused, lane, 32);   // last: nobody waits for it
      return;
    }
    if (e.blocks > 0) {
      loads += 2 * e.blocks;
      if (e.live_keys < kTile) dirty[count % kDelay] = (loads - 1) % S::kSlots, live_of[count % kDelay] = e.live_keys;
    }
  }
}

// ------------------------------------------------------------------------------------- copies

template <int kDim>
__device__ __forceinline__ void copy_role(const UmmaAttentionArgs& p, uint8_t* smem, Shared* b) {
  using S = Smem<kDim>;
  const AttentionArgs& a = p.a;
  const int tokens = a.tokens / 2;   // of a tile
  EntryReader reader{b};
  uint32_t load = 0, segment = 0;
  while (true) {
    const SegmentEntry e = *reader.wait();
    reader.release();
    if (!reader.ok || e.blocks < 0) return;
    if (e.blocks == 0) continue;
    bool ok = mbar_wait(&b->q_empty, (segment & 1) ^ 1, kSiteAttention);
    ++segment;
    if (!ok) return;
    const int tiles = e.pair != 0 ? 2 : 1;
    mbar_expect_tx(&b->q_full, tiles * S::kHalves * tokens * a.group * 128);
    for (int t = 0; t < tiles; ++t)
      for (int h = 0; h < S::kHalves; ++h)
        tma_load_3d(smem + t * S::kTileBytes + h * S::kHalfBytes, &p.q, &b->q_full, h * 64, e.head * a.group, e.q_row + t * tokens);
    const CUtensorMap *k = &p.k[e.source], *v = &p.v[e.source];
    for (int i = 0; i < 2 * e.blocks; ++i) {   // K and V of each block in turn
      const uint32_t slot = load % S::kSlots, round = load / S::kSlots;
      ++load;
      if (!mbar_wait(&b->empty[slot], (round & 1) ^ 1, kSiteAttention)) return;
      // Values with rows to be cleared arrive elsewhere first; who clears them signals `full`.
      uint64_t* arrival = i + 1 == 2 * e.blocks && e.live_keys < kTile ? &b->raw[slot] : &b->full[slot];
      mbar_expect_tx(arrival, S::kTileBytes);
      for (int h = 0; h < S::kHalves; ++h)
        tma_load_4d(smem + (2 + slot) * S::kTileBytes + h * S::kHalfBytes, (i & 1) != 0 ? v : k, arrival, h * 64, e.head, e.k_row + (i >> 1) * kTile,
                    e.batch);
    }
  }
}

// --------------------------------------------------------------------------------------- MMAs

// One thread per stream.
template <int kDim, bool kBf16>
struct MmaIssuer {
  using S = Smem<kDim>;
  static constexpr uint32_t kIdescS = umma_idesc_f16(kTile, kHalf, kBf16, false, false);
  Shared* b;
  int s, steps;   // stream; steps of 16 along the head dimension: what lies behind it reads as zero
  uint32_t idesc_o, s_at, o_at;
  uint64_t q_desc, k_desc, v_desc;
  uint32_t load = 0, own_segment = 0, p_phase = 0;   // p_phase: a bit per S

  __device__ __forceinline__ MmaIssuer(const AttentionArgs& a, uint8_t* smem, Shared* shared, uint32_t tmem, int stream) : b(shared), s(stream) {
    steps = (a.dim + 15) / 16;
    idesc_o = umma_idesc_f16(kTile, (a.dim + 15) / 16 * 16, kBf16, false, true);
    s_at = tmem + kColS + s * kColStream, o_at = tmem + kColO + s * kColStream;
    q_desc = umma_smem_desc(smem_u32(smem), 16, 1024, kUmmaSwizzle128B);
    k_desc = umma_smem_desc(smem_u32(smem) + 2 * S::kTileBytes, 16, 1024, kUmmaSwizzle128B);
    v_desc = umma_smem_desc(smem_u32(smem) + 2 * S::kTileBytes, S::kHalfBytes, 1024, kUmmaSwizzle128B);
  }
  __device__ __forceinline__ bool arrived(uint32_t at) const { return mbar_wait(&b->full[at % S::kSlots], at / S::kSlots & 1, kSiteAttention); }

  // Hands a block of the ring back when the products so far are done. Of a single tile only; see softmax_role.
  __device__ __forceinline__ void release(uint32_t at) const { umma_commit(&b->empty[at % S::kSlots]); }

  // Item j is S buffer j & 1, over 64 keys of a block: both halves of it in turn, or (one tile) the
  // stream's own.
  template <bool kPair>
  __device__ __forceinline__ uint32_t load_of(int j) const { return load + 2 * (kPair ? j >> 1 : j); }
  template <bool kPair>
  __device__ __forceinline__ uint32_t offset_of(uint32_t at, int j) const {   // of the item's keys or values in the ring
    return at % S::kSlots * S::kTileBytes + (kPair ? j & 1 : s) * (kHalf * 128);
  }
  template <bool kPair>
  __device__ __forceinline__ void scores(int j, int items) const {   // K is there
    const uint64_t qd = kPair ? umma_desc_advance(q_desc, s * S::kTileBytes) : q_desc;
    const uint64_t kd = umma_desc_advance(k_desc, offset_of<kPair>(load_of<kPair>(j), j));
    const uint32_t at = s_at + (j & 1) * kColHalf;
#pragma unroll
    for (int step = 0; step < kDim / 16; ++step) {
      if (step >= steps) break;
      const uint32_t offset = (step >> 2) * S::kHalfBytes + (step & 3) * 32;
      umma_f16(at, umma_desc_advance(qd, offset), umma_desc_advance(kd, offset), kIdescS, step > 0);
    }
    umma_commit(&b->s_full[s][j & 1]);
    if (!kPair) release(load_of<kPair>(j));
    if (j + 1 == items) umma_commit(&b->q_empty);
  }
  template <bool kPair>
  __device__ __forceinline__ bool segment(int items) {
    if (!arrived(load)) return false;
    tcgen05_fence_after_sync();
    scores<kPair>(0, items);
    if (items > 1) {
      if (!kPair && !arrived(load_of<kPair>(1))) return false;
      scores<kPair>(1, items);
    }
    for (int j = 0; j < items; ++j) {
      const uint32_t buffer = j & 1, at = load_of<kPair>(j);
      const bool opens = !kPair || (j & 1) == 0, more = j + 2 < items;
      // A wait costs a few hundred cycles even when it is over already: what is due by now is waited for
      // before P. (Not so the keys after next of a single tile: they are loaded only once the products
      // before have freed a place in the ring.)
      if (opens && !arrived(at + 1)) return false;
      if (kPair && opens && more && !arrived(at + 2)) return false;
      if (j == 0 && !mbar_wait(&b->o_empty[s], (own_segment & 1) ^ 1, kSiteAttention)) return false;
      if (!mbar_wait(&b->p_ready[s][buffer], p_phase >> buffer & 1, kSiteAttention)) return false;
      p_phase ^= 1u << buffer;
      tcgen05_fence_after_sync();
      const uint64_t vd = umma_desc_advance(v_desc, offset_of<kPair>(at + 1, j));
#pragma unroll
      for (int step = 0; step < kHalf / 16; ++step)
        umma_f16_tmem_a(o_at, s_at + buffer * kColHalf + step * 8, umma_desc_advance(vd, step * 2048), idesc_o, j > 0 || step > 0);
      if (!kPair) release(at + 1);
      if (more) {
        if (!kPair && !arrived(load_of<kPair>(j + 2))) return false;
        scores<kPair>(j + 2, items);
      }
      if (j + 2 == items) umma_commit(&b->drained[s]);
      if (j + 1 == items) umma_commit(&b->o_full[s]);
    }
    ++own_segment;
    return true;
  }

  __device__ __forceinline__ void run() {
    EntryReader reader{b};
    uint32_t segments = 0;
    while (true) {
      const SegmentEntry* entry = reader.wait();
      const int blocks = entry->blocks, items = items_of(*entry, s);
      const bool pair = entry->pair != 0;
      reader.release();
      if (!reader.ok || blocks < 0) return;
      if (blocks == 0) continue;
      if (!mbar_wait(&b->q_full, segments++ & 1, kSiteAttention)) return;
      if (items == 0) mbar_arrive(&b->q_empty);
      else if (!(pair ? segment<true>(items) : segment<false>(items))) return;
      if (!pair && items < blocks) {   // the last block has no keys for this stream
        for (uint32_t at = load + 2 * blocks - 2; at != load + 2 * blocks; ++at) {
          if (!arrived(at)) return;
          mbar_arrive(&b->empty[at % S::kSlots]);
        }
      }
      load += 2 * blocks;
    }
  }
};

// ------------------------------------------------------------------------------------ softmax

// The thread's row of a stream.
struct RowState {
  float m, l;   // base of the exponentials (scaled, base 2) and denominator
};

// One half block. `settled` waits until the products of the half before are in O.
// A NaN among the scores that a row sees, or +infinity, whose difference from itself is one, makes its
// maximum NaN and with it everything that follows.
template <bool kBf16, bool kMasked, class Settled>
__device__ __forceinline__ void softmax_half(uint32_t s_at, uint32_t o_at, int chunks, bool live, int seen, float scale, bool first, RowState* row,
                                             const Settled& settled) {
  float x[kHalf];
  tmem_ld_32x32(s_at, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
  tmem_ld_32x32(s_at + 32, *reinterpret_cast<uint32_t(*)[32]>(&x[32]));
  tmem_ld_wait();
  loaded(x);
  float top[4] = {kMinusInf, kMinusInf, kMinusInf, kMinusInf};
  if (kMasked) {
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
      if (i >= seen) x[i] = kMinusInf;   // chosen, not added: the product may be NaN
  }
#pragma unroll
  for (int i = 0; i < kHalf; i += 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) top[j] = max3_nan(top[j], x[i + j], x[i + 4 + j]);
  }
  float m = max3_nan(max3_nan(top[0], top[1], top[2]), top[3], top[3]) * scale;
  if (m == -kMinusInf) m = __int_as_float(0x7fffffff);
  if (!live) m = 0.f;   // lanes without a row hold anything; they must not ask for rescaling
  if (!kBf16) m -= kRaiseFp16;
  if (first) {
    row->m = m;
  } else {
    const bool grown = !(m <= row->m + kLazy);   // or NaN
    if (__any_sync(0xffffffffu, grown)) {
      const float next = grown ? m : row->m;
      const float keep = grown ? exp2_fast(row->m - next) : 1.f;
      row->l *= keep;
      row->m = next;
      settled();
      for (int c = 0; c < 2 * chunks; ++c) {
        float o[16];
        tmem_ld_32x16(o_at + 16 * c, *reinterpret_cast<uint32_t(*)[16]>(&o));
        tmem_ld_wait();
        loaded(o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] *= keep;
        tmem_st_32x16(o_at + 16 * c, *reinterpret_cast<uint32_t(*)[16]>(&o));
      }
    }
  }
  const float base = row->m == kMinusInf ? 0.f : row->m;   // nothing seen yet: all terms are 2^(-inf)
  const uint64_t scale2 = pack_f32x2(scale, scale), base2 = pack_f32x2(-base, -base);
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    uint32_t packed[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 y = unpack_f32x2(fma_f32x2(pack_f32x2(x[32 * part + 2 * i], x[32 * part + 2 * i + 1]), scale2, base2));
      const float lo = exp2_fast(y.x), hi = exp2_fast(y.y);
      sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(lo, hi));
      packed[i] = pack<kBf16>(lo, hi);
    }
    tmem_st_32x16(s_at + 16 * part, packed);
  }
  const float2 total = unpack_f32x2(add_f32x2(sum[0], sum[1]));
  row->l += total.x + total.y;
  tmem_st_wait();
}

// A warp's 32 finished rows, 64 columns at a time. Each thread holds its own row, and rows lie far apart:
// stored from the registers, every instruction would touch 32 lines of memory, which the load/store
// unit takes one per cycle. Where the 32 rows are all there they are laid out in the warp's 4 KiB of
// shared memory, in the 128-byte swizzle, and leave as one box.
template <bool kBf16>
__device__ __forceinline__ void stage_columns(uint8_t* stage, int lane, int half, const float (&y)[32]) {
  uint4* row = reinterpret_cast<uint4*>(stage + lane * 128);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    row[(half * 4 + i) ^ (lane & 7)] = make_uint4(pack<kBf16>(y[8 * i], y[8 * i + 1]), pack<kBf16>(y[8 * i + 2], y[8 * i + 3]),
                                                  pack<kBf16>(y[8 * i + 4], y[8 * i + 5]), pack<kBf16>(y[8 * i + 6], y[8 * i + 7]));
}

template <bool kBf16, uint32_t kSlots>
__device__ __forceinline__ void softmax_role(const UmmaAttentionArgs& p, Shared* b, uint8_t* staging, uint32_t tmem) {
  const AttentionArgs& a = p.a;
  const int s = threadIdx.x >> 7;                    // stream
  const int r = threadIdx.x & 127;                   // row of the tile, TMEM lane
  const int warp_row = r & ~31, lane = r & 31;
  const uint32_t lanes = static_cast<uint32_t>(warp_row) << 16;
  const uint32_t s_at = tmem + lanes + kColS + s * kColStream, o_at = tmem + lanes + kColO + s * kColStream;
  const uint32_t other_o_at = tmem + lanes + kColO + (s ^ 1) * kColStream;
  uint8_t* stage = staging + (threadIdx.x >> 5) * 4096;
  const int tile_rows = a.unit_rows / 2, tile_tokens = a.tokens / 2;
  const int token_r = r / a.group, head_r = r - token_r * a.group, token_warp = warp_row / a.group;   // within the tile
  const int chunks = (a.dim + 31) / 32;
  EntryReader reader{b};
  bool ok = true;
  uint32_t load = 0, s_phase = 0, drain_phase = 0, o_count[2] = {0, 0}, met = 0;
  // All eight warps; a bounded wait, which a plain barrier has not.
  const auto meet = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&b->exchanged);
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&b->exchanged, met & 1, kSiteAttention));
    ++met;
  };
  while (true) {
    const SegmentEntry* entry = reader.wait();
    ok = __all_sync(0xffffffffu, ok && reader.ok);
    const int blocks = ok ? entry->blocks : -1;
    const bool pair = entry->pair != 0, partial = entry->partial != 0;
    const int keys = entry->keys, ahead = entry->ahead, tokens = entry->tokens;
    const int token0 = pair && s == 1 ? tile_tokens : 0;   // of the tile within the unit
    const int q_row = entry->q_row + token0, head = entry->head * a.group;
    const int64_t slot = entry->slot;
    const int items = ok ? items_of(*entry, s) : 0, halves = entry->halves;
    const int pitch = entry->pitch, slot_row = (pair && s == 1 ? tile_rows : 0) + r;
    __syncwarp();
    if (lane == 0) reader.release();
    else ++reader.count;
    if (blocks < 0) {
      if (lane == 0) tma_store_wait_read<0>();   // shared memory must outlive the copies' reads
      return;
    }
    const bool live = r < tile_rows && token0 + token_r < tokens;
    const bool warp_live = warp_row < tile_rows && token0 + token_warp < tokens;   // some row of the warp is there
    RowState row{kMinusInf, 0.f};
    const int seen = live ? clamp_int(ahead + token0 + token_r, 0, keys) : 0;
    // All rows of the warp that are there see at least what its first row sees.
    const int seen_by_all = clamp_int(ahead + token0 + token_warp, 0, keys);
    // Two tiles hand blocks of the ring back here, one arrival per stream: scores that have arrived tell
    // that their keys have been read, and the values of the half before the last one too. Commits by the
    // MMA threads would say so earlier, but cost those threads, which everybody waits for, 130 cycles
    // each (16384 tokens 1073 -> 996 us). A single tile passes through the ring twice as fast, and needs
    // the places back at once (64 requests 142 us this way, 120 by commits).
    const auto hand_back = [&](int j, int values) {   // keys or values of item j, if it is its block's last
      if (pair && r == 0 && j >= 0 && ((j & 1) == 1 || j + 1 == items)) mbar_arrive(&b->empty[(load + 2 * (j >> 1) + values) % kSlots]);
    };
    for (int j = 0; j < items; ++j) {
      const uint32_t half = j & 1;
      const int key0 = (pair ? j : 2 * j + s) * kHalf;
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&b->s_full[s][half], s_phase >> half & 1, kSiteAttention));
      s_phase ^= 1u << half;
      hand_back(j, 0), hand_back(j - 2, 1);
      if (ok && warp_live) {
        tcgen05_fence_after_sync();
        // Scores of the half after are issued behind the products of the half before; the last half
        // has a signal of its own.
        const auto settled = [&]() {
          const bool more = j + 1 < items;
          ok = __all_sync(0xffffffffu, ok && mbar_wait(more ? &b->s_full[s][half ^ 1] : &b->drained[s],
                                                       more ? s_phase >> (half ^ 1) & 1 : drain_phase, kSiteAttention));
          tcgen05_fence_after_sync();
        };
        const uint32_t at = s_at + half * kColHalf;
        if (key0 + kHalf <= seen_by_all) softmax_half<kBf16, false>(at, o_at, chunks, live, 0, a.scale_log2, j == 0, &row, settled);
        else softmax_half<kBf16, true>(at, o_at, chunks, live, seen - key0, a.scale_log2, j == 0, &row, settled);
        tcgen05_fence_before_sync();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&b->p_ready[s][half]);
    }
    if (items > 1) drain_phase ^= 1;
    if (items > 0) {
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&b->o_full[s], o_count[s] & 1, kSiteAttention));
      ++o_count[s];
      hand_back(items - 2, 1), hand_back(items - 1, 1);
    }
    load += 2 * blocks;
    // Rows of one tile that two streams worked on: the same thread of both warp groups owns them, and
    // each finishes 64 of their columns.
    const bool joined = !pair && halves > 1;
    float mine = 1.f, other = 0.f, total = row.l, base = row.m;
    if (joined) {
      b->exchange[s][r] = make_float2(row.m, row.l);
      meet();
      const float2 peer = b->exchange[s ^ 1][r];
      base = fmaxf(row.m, peer.x);
      const float zero = base == kMinusInf ? 0.f : base;
      mine = exp2_fast(row.m - zero), other = exp2_fast(peer.x - zero);
      total = row.l * mine + peer.y * other;
      meet();   // read by all before the next segment writes
    }
    if (pair || joined) {   // the other stream has an accumulator too
      if (joined) ok = __all_sync(0xffffffffu, ok && mbar_wait(&b->o_full[s ^ 1], o_count[s ^ 1] & 1, kSiteAttention));
      if (blocks > 0) ++o_count[s ^ 1];
    } else if (s == 1 && blocks > 0) {
      ++o_count[0];
    }
    tcgen05_fence_after_sync();
    if (ok && warp_live && (pair || s == 0 || joined)) {
      if (partial && live && (pair || s == 0)) a.partial_ml[slot + slot_row] = make_float2(base, total);
      const float inv = partial ? 1.f : (total == 0.f ? 0.f : 1.f / total);
      const uint64_t f0 = pack_f32x2(mine * inv, mine * inv), f1 = pack_f32x2(other * inv, other * inv);
      const bool boxed = !partial && p.boxed != 0 && warp_row + 32 <= tile_rows && token0 + (warp_row + 31) / a.group < tokens;
      float* o_slot = a.partial_o + slot * a.dim + slot_row * 4;
      uint16_t* o_row = static_cast<uint16_t*>(a.out) + (static_cast<int64_t>(q_row + token_r) * a.heads + head + head_r) * a.dim;
      // Two warps that own the same rows take 64 columns each.
      for (int c = joined ? 2 * s : 0; c < (joined ? min(chunks, 2 * s + 2) : chunks); ++c) {
        float y[32];
        if (blocks > 0) {
          load_columns(o_at + 32 * c, y);
          if (joined) {
            float z[32];
            load_columns(other_o_at + 32 * c, z);
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t v = fma_f32x2(pack_f32x2(z[i], z[i + 1]), f1, 0);
              const float2 w = unpack_f32x2(fma_f32x2(pack_f32x2(y[i], y[i + 1]), f0, v));
              y[i] = w.x, y[i + 1] = w.y;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float2 w = unpack_f32x2(fma_f32x2(pack_f32x2(y[i], y[i + 1]), f0, 0));
              y[i] = w.x, y[i + 1] = w.y;
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) y[i] = 0.f;
        }
        if (boxed) {
          if ((c & 1) == 0) {   // the box's last copy has been read
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
          }
          stage_columns<kBf16>(stage, lane, c & 1, y);
          if ((c & 1) == 1 || c + 1 == chunks) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              const int token = warp_row / a.group;
              tma_store_3d(&p.out, stage, (c & ~1) * 32, head + warp_row - token * a.group, q_row + token);
              tma_store_commit();
            }
          }
        } else if (live && partial) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (32 * c + 4 * i < a.dim)
              *reinterpret_cast<float4*>(o_slot + static_cast<int64_t>(8 * c + i) * pitch * 4) = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
        } else if (live) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (32 * c + 8 * i < a.dim)
              *reinterpret_cast<uint4*>(o_row + 32 * c + 8 * i) = make_uint4(pack<kBf16>(y[8 * i], y[8 * i + 1]), pack<kBf16>(y[8 * i + 2], y[8 * i + 3]),
                                                                             pack<kBf16>(y[8 * i + 4], y[8 * i + 5]), pack<kBf16>(y[8 * i + 6], y[8 * i + 7]));
        }
      }
    }
    tcgen05_fence_before_sync();
    __syncwarp();
    if (lane == 0) {   // eight arrivals free an accumulator
      if (joined) mbar_arrive(&b->o_empty[0]), mbar_arrive(&b->o_empty[1]);
      else if (items > 0) mbar_arrive(&b->o_empty[s]), mbar_arrive(&b->o_empty[s]);
    }
  }
}

template <int kDim, bool kBf16, typename Line>
__global__ void __launch_bounds__(kThreads, 1) attention_umma_kernel(const __grid_constant__ UmmaAttentionArgs p) {
  using S = Smem<kDim>;
  extern __shared__ __align__(1024) uint8_t smem[];   // the swizzle's period
  Shared& b = *reinterpret_cast<Shared*>(smem + S::kTiles);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kSlots; ++i) mbar_init(&b.full[i], 1), mbar_init(&b.empty[i], 2), mbar_init(&b.raw[i], 1);
    for (int i = 0; i < kEntries; ++i) mbar_init(&b.entry_full[i], 1), mbar_init(&b.entry_empty[i], kEntryReaders);
    mbar_init(&b.q_full, 1), mbar_init(&b.q_empty, 2), mbar_init(&b.exchanged, 8);
    for (int s = 0; s < 2; ++s) {
      for (int h = 0; h < 2; ++h) mbar_init(&b.s_full[s][h], 1), mbar_init(&b.p_ready[s][h], 4);
      mbar_init(&b.drained[s], 1);
      mbar_init(&b.o_full[s], 1), mbar_init(&b.o_empty[s], 8);
    }
    mbar_init_fence();
  }
  if (threadIdx.x == 256) {
    prefetch_tensormap(&p.q), prefetch_tensormap(&p.out);
    for (int i = 0; i < (p.a.kind == kShared ? 2 : 1); ++i) prefetch_tensormap(&p.k[i]), prefetch_tensormap(&p.v[i]);
  }
  if (warp == 9) {
    tmem_alloc<512>(&b.tmem);
    tmem_relinquish();
  }
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  const uint32_t tmem = b.tmem;
  grid_launch_dependents();   // after the allocation: a following kernel may want tensor memory too
  grid_dependency_wait();
  const WorkStart<Line> start = find_range<kUmmaKeyBlock, kThreads, Line>(p.a, reinterpret_cast<WorkScratch<Line>*>(&b.scratch));
  if (warp < 8) {
    registers_raise<kSoftmaxRegisters>();
    softmax_role<kBf16, S::kSlots>(p, &b, smem + S::kStaging, tmem);
  } else {
    registers_lower<kOtherRegisters>();
    if (warp == 8 && lane == 0) copy_role<kDim>(p, smem, &b);
    if ((warp == 9 || warp == 10) && lane == 0) MmaIssuer<kDim, kBf16>(p.a, smem, &b, tmem, warp - 9).run();
    if (warp == 11) segment_role<kDim, Line>(p, start, smem, &b);
  }
  __syncwarp();
  tcgen05_fence_before_sync();
  __syncthreads();
  tcgen05_fence_after_sync();
  if (warp == 9) tmem_dealloc<512>(tmem);
}

template <int kDim, bool kBf16, typename Line>
int launch_line(const UmmaAttentionArgs& p, cudaStream_t s) {
  constexpr size_t kBytes = Smem<kDim>::kTiles + sizeof(Shared);
  static_assert(kBytes <= 227 * 1024, "shared memory of one CTA");
  if (!ensure_dynamic_smem<attention_umma_kernel<kDim, kBf16, Line>, kBytes>()) return B200_ERR_LAUNCH_FAILED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.a.ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kBytes;
  cfg.stream = s;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  if (cudaLaunchKernelEx(&cfg, attention_umma_kernel<kDim, kBf16, Line>, p) != cudaSuccess) return launch_failed();
  return launch_status();
}

template <int kDim, bool kBf16>
int launch(const UmmaAttentionArgs& p, cudaStream_t s) {
  return wide_line(p.a) ? launch_line<kDim, kBf16, int64_t>(p, s) : launch_line<kDim, kBf16, int>(p, s);
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
  a->tokens = 2 * (kTile / a->group);
  a->unit_rows = a->tokens * a->group;
  a->unit_cost = 3, a->pair_shift = 1;   // a block of one tile takes about 1.2 us, a unit beside its blocks 2 to 3
  a->ctas = sms;
}

int launch_attention_umma(const AttentionArgs& a, cudaStream_t s) {
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
  // A warp's rows are a box where they are whole tokens or lie within one.
  p.boxed = (a.group <= 32 ? 32 % a.group : a.group % 32) == 0;
  const uint64_t out_strides[2] = {static_cast<uint64_t>(a.dim) * 2, static_cast<uint64_t>(a.heads) * a.dim * 2};
  const uint32_t out_box[3] = {64, static_cast<uint32_t>(a.group < 32 ? a.group : 32), static_cast<uint32_t>(a.group < 32 ? 32 / a.group : 1)};
  if (p.boxed != 0) ok = ok && make_tensor_map_16bit(&p.out, a.out, 3, dims, out_strides, out_box, bf16);
  else p.out = p.q;
  if (!ok) return B200_ERR_INVALID_PROBLEM;
  if (a.dim <= 64) return bf16 ? launch<64, true>(p, s) : launch<64, false>(p, s);
  return bf16 ? launch<128, true>(p, s) : launch<128, false>(p, s);
}

}  // namespace b200
