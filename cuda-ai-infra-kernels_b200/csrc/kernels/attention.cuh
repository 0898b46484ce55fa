// Work decomposition shared by the attention kernels (attention_simt.cu) and the pass that joins
// partial results (attention.cu).
//
// Both operators are lists of sequences: n query tokens that see m keys. A prompt call has one per
// packed sequence (and a last one for the rows behind them, which sees nothing); a shared-prefix
// call has the whole batch over the prefix first and then every request over its own part of the
// cache. The rows of a key head are (token, query head of its group) pairs in that order, row
// i * group + g, so that all rows that read the same keys sit side by side whatever the head layout
// is: a decoding batch fills a tile with requests and heads as a prompt fills it with tokens.
//
// A unit is `unit_rows` such rows of one key head; its keys are cut in blocks, 128 or 64 keys each. All
// blocks of all units, in the order sequence, head, unit, block, are dealt out in equal contiguous
// ranges, one per CTA, whatever the lengths are. (One CTA per unit, longest first, left the tensor
// pipe idle at the start and end of every unit and the machine uneven at the end of a call.) A unit
// that lies inside one range is finished by its CTA. One that is cut by a range boundary leaves one
// partial result (sum, maximum, denominator) per CTA that worked on it, and a second launch joins
// them in CTA order: at most one unit per boundary, so the traffic does not grow with the call. In a
// shared-prefix call every row has two units, one per part of its keys, and all results are partial.
// In a prompt call a unit that sees no key counts as one block, so that somebody writes its zeros.
// Lengths are read on the device only. Offsets and lengths are clamped to the arrays here.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_common.h"
#include "ptx_sm100.cuh"

namespace b200 {

enum AttentionKind : int { kPrompt = 0, kShared = 1 };

struct AttentionArgs {
  const void* q;
  int64_t q_row, q_head;             // strides, in elements
  const void *k[2], *v[2];           // [1]: the cache of a shared-prefix call
  int64_t k_row[2], k_head[2], v_row[2], v_head[2];
  int64_t k_batch, v_batch;          // of the cache
  void* out;
  const int32_t *cu_q, *cu_k, *lengths;
  int kind, dtype;
  int sequences;                     // prompt: without the rows behind the last one; shared: 1 + batch
  int q_rows, k_rows, room;          // k_rows: keys of the packed array, or of the prefix
  int heads, kv_heads, group, dim;
  float scale_log2;                  // scale * log2(e): exponentials are powers of two
  int causal;
  int unit_rows;
  int tokens;                        // of a unit; 0 where a group is larger than a unit, and units cut tokens
  int token_shift;                   // its logarithm where it is a power of two, else -1
  int ctas;                          // ranges
  // Partial results: [row][dim], not divided by the denominator. First come the rows of units that
  // are continued from the CTA before (unit_rows for each CTA), then those of units that are opened:
  // unit_rows for each CTA in a prompt call, (part, output row) in a shared-prefix call.
  float* partial_o;
  float2* partial_ml;                // maximum (scaled, base 2), denominator
};

struct Sequence {
  int q_row, n;        // first query row, queries
  int k_row, m;        // first key row, keys
  int source, batch;   // which pair of key and value arrays
};

inline int log2_or_minus_one(int v) {
  if (v <= 0 || (v & (v - 1)) != 0) return -1;
  int shift = 0;
  while (1 << shift < v) ++shift;
  return shift;
}

__host__ __device__ inline int clamp_int(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

__device__ __forceinline__ int sequence_count(const AttentionArgs& a) { return a.sequences + (a.kind == kPrompt ? 1 : 0); }

__device__ __forceinline__ Sequence sequence_of(const AttentionArgs& a, int s) {
  Sequence r{};
  if (a.kind == kShared) {
    if (s == 0) {
      r.n = a.q_rows, r.m = a.k_rows;
    } else {
      r.q_row = r.batch = s - 1, r.n = 1, r.source = 1;
      r.m = clamp_int(__ldg(a.lengths + s - 1), 0, a.room);
    }
    return r;
  }
  r.q_row = clamp_int(__ldg(a.cu_q + s), 0, a.q_rows);
  if (s == a.sequences) {
    r.n = a.q_rows - r.q_row;
    return r;
  }
  r.n = clamp_int(__ldg(a.cu_q + s + 1), r.q_row, a.q_rows) - r.q_row;
  r.k_row = clamp_int(__ldg(a.cu_k + s), 0, a.k_rows);
  r.m = clamp_int(__ldg(a.cu_k + s + 1), r.k_row, a.k_rows) - r.k_row;
  return r;
}

// Keys that query i of the sequence sees: a prefix of its keys, aligned so that the last query sees all.
__device__ __forceinline__ int visible_keys(const AttentionArgs& a, const Sequence& s, int i) {
  if (a.kind == kShared || a.causal == 0) return s.m;
  return clamp_int(s.m - s.n + i + 1, 0, s.m);
}

__device__ __forceinline__ int unit_count(const AttentionArgs& a, const Sequence& s) {
  return a.tokens > 0 ? (s.n + a.tokens - 1) / a.tokens : (s.n * a.group + a.unit_rows - 1) / a.unit_rows;
}

template <int kKeys>
__device__ __forceinline__ int unit_blocks(const AttentionArgs& a, const Sequence& s, int unit) {
  const int last = a.tokens > 0 ? (unit + 1) * a.tokens - 1 : ((unit + 1) * a.unit_rows - 1) / a.group;
  return (visible_keys(a, s, min(last, s.n - 1)) + kKeys - 1) / kKeys;
}

// What a unit counts in the ranges.
template <int kKeys>
__device__ __forceinline__ int unit_weight(const AttentionArgs& a, const Sequence& s, int unit) {
  const int blocks = unit_blocks<kKeys>(a, s, unit);
  return blocks == 0 && a.kind == kPrompt ? 1 : blocks;
}

// Quotient of numbers that are small as a rule: a 64-bit division costs a hundred instructions.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  if (((x | y) >> 32) == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(y);
  return x / y;
}

// sum over i = 0 .. n - 1 of floor((a i + b) / m), for a, b >= 0: the whole multiples of m in a and b
// come out as closed sums; what is left counts lattice points under a line, and counting them by
// the other coordinate is the same sum with a and m exchanged, as in Euclid's algorithm.
__device__ __forceinline__ int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
  int64_t sum = 0;
  while (n > 0) {
    const int64_t whole_a = quotient(a, m), whole_b = quotient(b, m);
    sum += n * (n - 1) / 2 * whole_a + n * whole_b;
    a -= whole_a * m, b -= whole_b * m;
    const int64_t top = a * n + b;
    if (top < m) break;
    n = quotient(top, m), b = top - n * m;
    const int64_t t = m;
    m = a, a = t;
  }
  return sum;
}

// Weight of the first `units` units of one key head of the sequence.
template <int kKeys>
__device__ __noinline__ int64_t weight_before(const AttentionArgs& a, const Sequence& s, int units) {
  if (units == 0) return 0;
  if (a.kind == kShared || a.causal == 0) return static_cast<int64_t>(units) * unit_weight<kKeys>(a, s, 0);
  if (a.tokens == 0) {
    int64_t sum = 0;
    for (int t = 0; t < units; ++t) sum += unit_weight<kKeys>(a, s, t);
    return sum;
  }
  // Unit t holds whole tokens; but for the last of all, its last token sees c + tokens * (t + 1) keys.
  // Where tokens is a power of two that divides the block, t advances the quotient by one every
  // 2^shift units, and where it is a multiple of the block by a constant: no division.
  const int tokens = a.tokens, all = unit_count(a, s);
  const int64_t c = static_cast<int64_t>(s.m) - s.n;
  const int64_t regular = units < all ? units : all - 1;
  const int64_t blind = c >= 0 ? 0 : min(quotient(-c, tokens), regular);   // units that see nothing, one each
  const int64_t n = regular - blind, b = c + tokens * (blind + 1) + kKeys - 1;
  int64_t sum = blind;
  if (a.token_shift < 0) {
    sum += floor_sum(n, kKeys, tokens, b);
  } else if (tokens >= kKeys) {
    sum += n * (n - 1) / 2 * (tokens / kKeys) + n * (b / kKeys);
  } else {
    // floor((tokens i + b) / kKeys) = floor((i + first) / r) with r = kKeys / tokens, first = floor(b / tokens);
    // below x the quotients y / r add up to r q (q - 1) / 2 + q (x mod r), q = x / r.
    constexpr int kLog = kKeys == 128 ? 7 : 6;
    static_assert(1 << kLog == kKeys, "key blocks of 64 or 128");
    const int64_t r = kKeys >> a.token_shift, first = b >> a.token_shift;
    const auto below = [&](int64_t x) {
      const int64_t q = x >> (kLog - a.token_shift);
      return r * (q * (q - 1) / 2) + q * (x - q * r);
    };
    sum += below(first + n) - below(first);
  }
  if (units == all) sum += unit_weight<kKeys>(a, s, all - 1);
  return sum;
}

template <int kKeys>
__device__ __forceinline__ int64_t head_weight(const AttentionArgs& a, const Sequence& s) {
  return weight_before<kKeys>(a, s, unit_count(a, s));
}

// ------------------------------------------------------------------------- finding a CTA's work

struct WorkStart {
  int sequence;               // -1: nothing to do
  int head, unit, block;
  int64_t per, length;        // blocks per range, and of this one
  int64_t position, before;   // of the range; of the first block of `unit`
};

struct WorkScratch {
  int64_t sums[32];
  WorkStart start;
};

// Where range `range` starts: prefix sums over the sequences by all kThreads threads of the CTA.
template <int kKeys, int kThreads>
__device__ __forceinline__ WorkStart find_range(const AttentionArgs& a, WorkScratch* scratch, int range) {
  const int count = sequence_count(a);
  const int chunk = (count + kThreads - 1) / kThreads;
  const int lo = min(static_cast<int>(threadIdx.x) * chunk, count), hi = min(lo + chunk, count);
  const auto weight = [&](int s) { return a.kv_heads * head_weight<kKeys>(a, sequence_of(a, s)); };
  int64_t mine = 0;
  for (int s = lo; s < hi; ++s) mine += weight(s);
  int64_t upto = mine;   // inclusive over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
    if ((threadIdx.x & 31) >= o) upto += other;
  }
  if ((threadIdx.x & 31) == 31) scratch->sums[threadIdx.x >> 5] = upto;
  __syncthreads();
  int64_t before = upto - mine, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 5)) before += scratch->sums[w];
    total += scratch->sums[w];
  }
  const int64_t per = quotient(total + a.ctas - 1, a.ctas);
  const int64_t position = range * per;
  WorkStart& start = scratch->start;
  if (threadIdx.x == 0) start = WorkStart{-1, 0, 0, 0, per, 0, position, 0};
  __syncthreads();
  if (position >= before && position < before + mine) {
    int s = lo;
    int64_t size = mine;
    for (; s < hi; ++s) {
      size = hi - lo == 1 ? mine : weight(s);
      if (position < before + size) break;
      before += size;
    }
    const int64_t per_head = quotient(size, a.kv_heads);
    start.sequence = s;
    start.head = static_cast<int>(quotient(position - before, per_head));
    start.length = min(per, total - position);
    start.before = before + start.head * per_head;   // of the head, until the unit is known
  }
  __syncthreads();
  const WorkStart found = start;
  if (found.sequence < 0) return found;
  // The last unit that does not start behind the position, by all threads at once.
  const Sequence seq = sequence_of(a, found.sequence);
  const int64_t rest = position - found.before;
  int low = 0, high = unit_count(a, seq);
  while (true) {
    const int step = (high - low + kThreads - 1) / kThreads;
    const int mid = low + step * static_cast<int>(threadIdx.x), end = min(mid + step, high);
    __syncthreads();
    if (mid < high) {
      const int64_t first = weight_before<kKeys>(a, seq, mid);
      if (first <= rest && (end == high || rest < weight_before<kKeys>(a, seq, end)))
        start.unit = mid, start.block = static_cast<int>(rest - first), start.before = found.before + first;
    }
    __syncthreads();
    low = start.unit, high = min(low + step, high);
    if (step <= 1) return start;
  }
}

// A contiguous run of key blocks of one unit.
struct Segment {
  Sequence seq;
  int head, unit;
  int block_begin, block_end;   // of the unit's blocks; none for rows that see no key
  bool opens, whole;            // starts at the unit's first block; is all of it
};

// Walks the segments of a CTA's range. Every role of a CTA walks for itself and sees the same ones.
template <int kKeys>
struct SegmentWalk {
  const AttentionArgs& a;
  int64_t left;      // blocks still to be handed out
  int sequence, units;
  Sequence seq;
  int head, unit, block;

  __device__ __forceinline__ SegmentWalk(const AttentionArgs& args, const WorkStart& start) : a(args), left(0), sequence(start.sequence) {
    if (sequence < 0) return;
    seq = sequence_of(a, sequence);
    units = unit_count(a, seq);
    left = start.length, head = start.head, unit = start.unit, block = start.block;
  }

  __device__ __forceinline__ bool next(Segment* out) {
    if (left <= 0) return false;
    int blocks = unit_blocks<kKeys>(a, seq, unit), weight = a.kind == kPrompt ? max(blocks, 1) : blocks;
    while (block >= weight) {   // on to the next unit that counts; there is one while `left` > 0
      block = 0;
      if (++unit >= units) {
        unit = 0;
        if (++head >= a.kv_heads) {
          head = 0;
          do {
            seq = sequence_of(a, ++sequence);
            units = unit_count(a, seq);
          } while (units == 0);
        }
      }
      blocks = unit_blocks<kKeys>(a, seq, unit), weight = a.kind == kPrompt ? max(blocks, 1) : blocks;
    }
    const int take = static_cast<int>(min(static_cast<int64_t>(weight - block), left));
    *out = Segment{seq, head, unit, block, min(block + take, blocks), block == 0, take == weight};
    block += take;
    left -= take;
    return true;
  }
};

// Where rows go: row `row` of a unit is the output row `out` (token * heads + head).
__device__ __forceinline__ int64_t continued_row(const AttentionArgs& a, int cta, int row) {
  return static_cast<int64_t>(cta) * a.unit_rows + row;
}
__device__ __forceinline__ int64_t opened_row(const AttentionArgs& a, const Sequence& s, int64_t out, int cta, int row) {
  const int64_t first = static_cast<int64_t>(a.ctas) * a.unit_rows;
  return first + (a.kind == kPrompt ? continued_row(a, cta, row) : s.source * static_cast<int64_t>(a.q_rows) * a.heads + out);
}
__device__ __forceinline__ bool is_partial(const AttentionArgs& a, const Segment& g) { return a.kind == kShared || !g.whole; }
__device__ __forceinline__ int64_t partial_row(const AttentionArgs& a, const Segment& g, int64_t out, int row) {
  return g.opens ? opened_row(a, g.seq, out, blockIdx.x, row) : continued_row(a, blockIdx.x, row);
}
// Output row of row `flat` of a sequence's rows of a key head.
__device__ __forceinline__ int64_t output_row(const AttentionArgs& a, const Sequence& s, int head, int flat) {
  const int token = flat / a.group;
  return static_cast<int64_t>(s.q_row + token) * a.heads + head * a.group + (flat - token * a.group);
}

// The kernels: rows of a unit and CTAs that the machine holds at once, and launch. The key block of
// each is needed by the join.
constexpr int kSimtKeyBlock = 64;
constexpr int kUmmaKeyBlock = 128;
void plan_attention_umma(AttentionArgs* a, int sms);
void plan_attention_simt(AttentionArgs* a, int sms);
int launch_attention_umma(const AttentionArgs& a, cudaStream_t s);
int launch_attention_simt(const AttentionArgs& a, cudaStream_t s);

}  // namespace b200
