// Work decomposition shared by the attention kernels (attention_simt.cu) and the pass that joins
// partial results (attention.cu).
//
// Both operators are lists of sequences: n query tokens that see m keys. A prompt call has one per
// packed sequence (and a last one for the rows behind them, which sees nothing; the rows in front of
// them are cleared apart from all that); a shared-prefix call has the whole batch over the prefix
// first and then every request over its own part of the cache. The rows of a key head are (token, query
// head of its group) pairs in that order, row i * group + g, so that all rows that read the same keys
// sit side by side whatever the head layout is: a decoding batch fills a tile with requests and heads
// as a prompt fills it with tokens.
//
// A unit is `unit_rows` such rows of one key head; its keys are cut in blocks, 128 or 64 keys each. All
// units, in the order sequence, head, unit, are laid end to end, each as long as its blocks (twice,
// where the kernel works on two tiles of rows) plus `unit_cost` for what a unit costs beside them, and
// the line is dealt out in equal contiguous ranges, one per CTA, whatever the lengths are. (One CTA per unit, longest first, left the tensor
// pipe idle at the start and end of every unit and the machine uneven at the end of a call.) A unit
// that lies inside one range is finished by its CTA. One that is cut by a range boundary leaves one
// partial result (sum, maximum, denominator) per CTA that worked on it, and a second launch joins
// them in CTA order: at most one unit per boundary, so the traffic does not grow with the call. In a
// shared-prefix call every row has two units, one per part of its keys, and all results are partial.
// Positions on the line are of type Line: 32 bits, or 64 where the arrays are large enough for a line that
// passes them (a million causal tokens of 64 heads). With 64 throughout, the segment walk's registers
// and divisions cost 64 requests behind a prefix 10 of 112 us and ragged prompts 6 of 119.
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
  int tokens;                        // of a unit: it holds whole ones
  int token_shift;                   // its logarithm where it is a power of two, else -1
  int unit_cost, pair_shift;         // on the line: of a unit; logarithm of a block's for a unit of more than half the rows
  int ctas;                          // ranges
  int64_t longest_line;              // the longest that sequences which do not overlap can make
  // Partial results, in slots of some rows: maximum (scaled, base 2) and denominator [row], and the sum,
  // not divided by it, as [dim / 4][row][4], so that the threads of a warp, which own one row
  // each, write and read whole lines. First the slots of units continued from the CTA before,
  // one of unit_rows rows per CTA, then those of units that a CTA opens: one per CTA in a prompt call;
  // in a shared-prefix call one per prefix unit and head, and then `group` rows per request and head.
  float* partial_o;
  float2* partial_ml;
  struct CutRecord* cuts;            // of each CTA in a prompt call, of each unit in a shared-prefix call
};

// What the join has to know about an opened unit; written by the CTA that opens it.
struct CutRecord {
  int first, last;         // CTAs that worked on it
  int rows;                // prompt: 0 where the CTA left no unit open
  int q_row, head, row0;   // prompt: the sequence's first query row, the key head, the unit's first row
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
  const int next = min(s + 1, a.sequences);   // all four on their way at once
  const int q0 = __ldg(a.cu_q + s), q1 = __ldg(a.cu_q + next), k0 = __ldg(a.cu_k + s), k1 = __ldg(a.cu_k + next);
  r.q_row = clamp_int(q0, 0, a.q_rows);
  r.k_row = clamp_int(k0, 0, a.k_rows);
  if (s == a.sequences) {
    r.n = a.q_rows - r.q_row;
  } else {
    r.n = clamp_int(q1, r.q_row, a.q_rows) - r.q_row;
    r.m = clamp_int(k1, r.k_row, a.k_rows) - r.k_row;
  }
  return r;
}

// Keys that query i of the sequence sees: a prefix of its keys, aligned so that the last query sees all.
__device__ __forceinline__ int visible_keys(const AttentionArgs& a, const Sequence& s, int i) {
  if (a.kind == kShared || a.causal == 0) return s.m;
  return clamp_int(s.m - s.n + i + 1, 0, s.m);
}

__device__ __forceinline__ int unit_count(const AttentionArgs& a, const Sequence& s) {
  return (s.n + a.tokens - 1) / a.tokens;
}

template <int kKeys>
__device__ __forceinline__ int unit_blocks(const AttentionArgs& a, const Sequence& s, int unit) {
  return (visible_keys(a, s, min((unit + 1) * a.tokens, s.n) - 1) + kKeys - 1) / kKeys;
}

__device__ __forceinline__ int block_shift(const AttentionArgs& a, const Sequence& s, int unit) {   // logarithm of its length
  return s.n - unit * a.tokens > a.tokens / 2 ? a.pair_shift : 0;
}

// Length of a unit on the line. A prompt's unit that sees no key is there all the same: somebody has
// to write its zeros.
template <int kKeys>
__device__ __forceinline__ int unit_length(const AttentionArgs& a, const Sequence& s, int unit) {
  const int blocks = unit_blocks<kKeys>(a, s, unit);
  return blocks > 0 || a.kind == kPrompt ? (blocks << block_shift(a, s, unit)) + a.unit_cost : 0;
}

// sum over i = 0 .. n - 1 of floor((a i + b) / m), for a, b >= 0: the whole multiples of m in a and b
// come out as closed sums; what is left counts lattice points under a line, and counting them by
// the other coordinate is the same sum with a and m exchanged, as in Euclid's algorithm.
static __device__ __noinline__ int64_t floor_sum(int n, int m, int a, int b) {
  int64_t sum = 0;
  while (n > 0) {
    const int whole_a = a / m, whole_b = b / m;
    sum += static_cast<int64_t>(n) * (n - 1) / 2 * whole_a + static_cast<int64_t>(n) * whole_b;
    a -= whole_a * m, b -= whole_b * m;
    const int64_t top = static_cast<int64_t>(a) * n + b;
    if (top < m) break;
    n = static_cast<int>(top / m), b = static_cast<int>(top - static_cast<int64_t>(n) * m);
    const int t = m;
    m = a, a = t;
  }
  return sum;
}

// Length of the first `units` of the `all` units of one key head of the sequence. Not inlined: a CTA
// calls it three or four times as it starts, when every instruction has to be fetched before it runs.
template <int kKeys, typename Line>
__device__ __noinline__ Line length_before(const AttentionArgs& a, const Sequence& s, int units, int all) {
  if (units == 0) return 0;
  const int regular = units < all ? units : all - 1;   // all but the last have all their rows
  const int rest = units == all ? unit_length<kKeys>(a, s, all - 1) : 0;
  if (a.kind == kShared || a.causal == 0) return (regular > 0 ? static_cast<Line>(regular) * unit_length<kKeys>(a, s, 0) : 0) + rest;
  // Unit t holds whole tokens; but for the last of all, its last token sees c + tokens * (t + 1) keys.
  const int tokens = a.tokens, c = s.m - s.n;
  const int blind = c >= 0 ? 0 : min(-c / tokens, regular);   // units that see nothing
  const int n = regular - blind, b = c + tokens * (blind + 1) + kKeys - 1;
  Line sum = 0;   // blocks
  if (a.token_shift < 0) {
    sum += static_cast<Line>(floor_sum(n, kKeys, tokens, b));
  } else if (tokens >= kKeys) {
    sum += static_cast<Line>(static_cast<int64_t>(n) * (n - 1) / 2) * (tokens / kKeys) + static_cast<Line>(n) * (b / kKeys);
  } else {
    // tokens divides the block: floor((tokens i + b) / kKeys) = floor((i + first) / r) with
    // r = kKeys / tokens, first = floor(b / tokens); below x the quotients y / r add up to
    // r q (q - 1) / 2 + q (x mod r), q = x / r.
    constexpr int kLog = kKeys == 128 ? 7 : 6;
    static_assert(1 << kLog == kKeys, "key blocks of 64 or 128");
    const int shift = kLog - a.token_shift, first = b >> a.token_shift;
    const auto below = [&](int x) {
      const int q = x >> shift;
      return static_cast<int64_t>(q) * (q - 1) / 2 * (1 << shift) + static_cast<int64_t>(q) * (x - (q << shift));
    };
    sum += static_cast<Line>(below(first + n) - below(first));
  }
  return (sum << a.pair_shift) + static_cast<Line>(regular) * a.unit_cost + rest;
}

// ------------------------------------------------------------------------- finding a CTA's work

// Ranges of the line: the first total % ctas are one longer than the rest.
template <typename Line>
struct Ranges {
  Line quotient;
  int longer;
  __device__ __forceinline__ Ranges(Line total, int ctas) : quotient(total / ctas), longer(static_cast<int>(total - quotient * ctas)) {}
  Ranges() = default;
  __device__ __forceinline__ Line begin(int c) const { return c * quotient + min(c, longer); }
  __device__ __forceinline__ int holder(Line position) const {
    const Line boundary = longer * (quotient + 1);
    return static_cast<int>(position < boundary ? position / (quotient + 1) : longer + (position - boundary) / quotient);
  }
};

constexpr int kIdle = -1, kRefused = -2;

template <typename Line>
struct WorkStart {
  int sequence;               // kIdle: nothing to do; kRefused: in the whole call
  Sequence seq;
  int units;                  // of a head of the sequence
  int head, unit;
  Line offset;                // into the head's units, and at last into the unit
  Ranges<Line> ranges;
  Line begin, length;         // of this range
};

template <typename Line>
struct WorkScratch {
  int64_t sums[32];
  WorkStart<Line> start;
};

// Where this CTA's range starts: prefix sums over the sequences by all kThreads threads.
template <int kKeys, int kThreads, typename Line>
__device__ __forceinline__ WorkStart<Line> find_range(const AttentionArgs& a, WorkScratch<Line>* scratch) {
  const int count = sequence_count(a);
  const int chunk = (count + kThreads - 1) / kThreads;
  const int lo = min(static_cast<int>(threadIdx.x) * chunk, count), hi = min(lo + chunk, count);
  Sequence seq{};
  Line size = 0;
  int64_t mine = 0;   // sequences that overlap could make the line longer than the launcher counted on
  for (int s = lo; s < hi; ++s) {
    seq = sequence_of(a, s);
    const int units = unit_count(a, seq);
    size = a.kv_heads * length_before<kKeys, Line>(a, seq, units, units);
    mine += size;
    if (sizeof(Line) == 8) mine = min(mine, a.longest_line + 1);   // of 2^30 sequences the sum would pass 64 bits
  }
  int64_t upto = mine;   // inclusive over the warp
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
    if ((threadIdx.x & 31) >= o) upto += other;
  }
  if ((threadIdx.x & 31) == 31) scratch->sums[threadIdx.x >> 5] = upto;
  WorkStart<Line>& start = scratch->start;
  if (threadIdx.x == 0) start.sequence = kIdle;
  __syncthreads();
  int64_t ahead = upto - mine, whole = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < static_cast<int>(threadIdx.x >> 5)) ahead += scratch->sums[w];
    whole += scratch->sums[w];
  }
  const Line total = whole <= a.longest_line ? static_cast<Line>(whole) : 0;
  if (whole > a.longest_line && threadIdx.x == 0) start.sequence = kRefused;   // sequences overlap
  Line before = static_cast<Line>(min(ahead, static_cast<int64_t>(total)));
  const Ranges<Line> ranges(total, a.ctas);
  const Line begin = ranges.begin(blockIdx.x), length = ranges.begin(blockIdx.x + 1) - begin;
  if (length > 0 && begin >= before && begin < ahead + mine) {
    int s = lo;
    if (hi - lo > 1) {
      for (; s < hi; ++s) {
        seq = sequence_of(a, s);
        const int units = unit_count(a, seq);
        size = a.kv_heads * length_before<kKeys, Line>(a, seq, units, units);
        if (begin < before + size) break;
        before += size;
      }
    }
    const Line per_head = size / a.kv_heads;
    const int head = static_cast<int>((begin - before) / per_head);
    start = WorkStart<Line>{s, seq, unit_count(a, seq), head, 0, begin - before - head * per_head, ranges, begin, length};
  }
  __syncthreads();
  WorkStart<Line> found = start;
  if (found.sequence < 0) return found;
  // The last unit that does not start behind the position, by all threads at once.
  int low = 0, high = found.units;
  while (true) {
    const int step = (high - low + kThreads - 1) / kThreads;
    const int mid = low + step * static_cast<int>(threadIdx.x), end = min(mid + step, high);
    __syncthreads();
    if (mid < high) {
      const Line first = length_before<kKeys, Line>(a, found.seq, mid, found.units);
      if (first <= found.offset && (end == high || found.offset < length_before<kKeys, Line>(a, found.seq, end, found.units)))
        start.unit = mid, start.offset = found.offset - first;
    }
    __syncthreads();
    low = start.unit, high = min(low + step, high);
    if (step <= 1) return start;
  }
}

// Zeros for the rows that no sequence owns: those in front of the first one, or all of a call whose
// sequences overlap so far that their work has no bound, which is recorded. By some threads of every CTA.
static __device__ __noinline__ void clear_unowned_rows(const AttentionArgs& a, bool refused, int thread, int threads) {
  if (a.kind != kPrompt) return;
  const int64_t rows = refused ? a.q_rows : clamp_int(__ldg(a.cu_q), 0, a.q_rows);
  const int64_t granules = rows * a.heads * a.dim / (a.dtype == B200_FP32 ? 4 : 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * threads + thread; i < granules; i += static_cast<int64_t>(gridDim.x) * threads)
    static_cast<uint4*>(a.out)[i] = make_uint4(0, 0, 0, 0);
  if (refused && blockIdx.x == 0 && thread == 0) atomicOr(&g_device_status, kSiteOverlap);
}

// A contiguous run of key blocks of one unit.
struct Segment {
  Sequence seq;
  int head, unit;
  int block_begin, block_end;   // of the unit's blocks; none for rows that see no key
  bool opens, whole;            // starts at the unit's first block; is all of it
  int first_cta, last_cta;      // of an opened unit
};

// Walks the segments of a CTA's range.
template <int kKeys, typename Line>
struct SegmentWalk {
  const AttentionArgs& a;
  Ranges<Line> ranges;
  Line position, end;   // on the line
  int sequence, units;
  Sequence seq;
  int head, unit, offset;

  __device__ __forceinline__ SegmentWalk(const AttentionArgs& args, const WorkStart<Line>& start) : a(args), ranges(start.ranges) {
    position = start.begin, end = start.sequence < 0 ? start.begin : start.begin + start.length;
    sequence = start.sequence, seq = start.seq, units = start.units, head = start.head, unit = start.unit, offset = static_cast<int>(start.offset);
  }

  __device__ __forceinline__ bool next(Segment* out) {
    while (position < end) {
      const int blocks = unit_blocks<kKeys>(a, seq, unit), length = unit_length<kKeys>(a, seq, unit), shift = block_shift(a, seq, unit);
      const int from = offset, to = static_cast<int>(min(static_cast<Line>(length), offset + end - position));
      const Line unit_position = position - from;
      Segment g{seq, head, unit, max(from - a.unit_cost, 0) >> shift, max(to - a.unit_cost, 0) >> shift, false, false, 0, 0};
      position += to - from;
      offset = to;
      if (to == length) {   // on to the next unit
        offset = 0;
        if (++unit >= units) {
          unit = 0;
          if (++head >= a.kv_heads && position < end) {
            head = 0;
            do {
              seq = sequence_of(a, ++sequence);
              units = unit_count(a, seq);
            } while (units == 0);
          }
        }
      }
      // A range may end within what a unit costs beside its blocks, or within a block; a block belongs
      // to the range that holds its end. A range that holds only a piece of a block in the middle of
      // a unit leaves an empty partial result: the join counts on one from every CTA on the way.
      if (blocks > 0 ? g.block_end > 0 : length > 0 && to == length) {
        g.opens = g.block_begin == 0, g.whole = g.opens && g.block_end == blocks;   // block_end > 0 or no blocks at all
        g.first_cta = g.last_cta = blockIdx.x;
        if (g.opens && !g.whole) g.last_cta = ranges.holder(unit_position + length - 1);
        *out = g;
        return true;
      }
    }
    return false;
  }
};

// ------------------------------------------------------------------------------- partial results

// Rows in front of slots; see AttentionArgs. prefix_units: of one head.
__device__ __forceinline__ int64_t continued_slot(const AttentionArgs& a, int cta) { return static_cast<int64_t>(cta) * a.unit_rows; }
__device__ __forceinline__ int prefix_units(const AttentionArgs& a) { return (a.q_rows * a.group + a.unit_rows - 1) / a.unit_rows; }
__device__ __forceinline__ int64_t prefix_slot(const AttentionArgs& a, int unit, int head) {
  return (a.ctas + static_cast<int64_t>(unit) * a.kv_heads + head) * a.unit_rows;
}
__device__ __forceinline__ int64_t own_slot(const AttentionArgs& a, int request, int head) {
  return (a.ctas + static_cast<int64_t>(prefix_units(a)) * a.kv_heads) * a.unit_rows + (static_cast<int64_t>(request) * a.kv_heads + head) * a.group;
}
__device__ __forceinline__ int64_t prefix_record(const AttentionArgs& a, int unit, int head) { return static_cast<int64_t>(unit) * a.kv_heads + head; }
__device__ __forceinline__ int64_t own_record(const AttentionArgs& a, int request, int head) {
  return (static_cast<int64_t>(prefix_units(a)) + request) * a.kv_heads + head;
}

__device__ __forceinline__ bool is_partial(const AttentionArgs& a, const Segment& g) { return a.kind == kShared || !g.whole; }

// Slot of a segment's partial result, and the rows of the slot.
__device__ __forceinline__ int64_t slot_of(const AttentionArgs& a, const Segment& g, int* pitch) {
  *pitch = a.unit_rows;
  if (!g.opens) return continued_slot(a, blockIdx.x);
  if (a.kind == kPrompt) return continued_slot(a, a.ctas + blockIdx.x);
  if (g.seq.source == 0) return prefix_slot(a, g.unit, g.head);
  *pitch = a.group;
  return own_slot(a, g.seq.batch, g.head);
}

// The record of an opened unit. To be called by one thread of the CTA for each segment, and, in a
// prompt call, once before the first (`start`).
__device__ __forceinline__ void start_records(const AttentionArgs& a) {
  if (a.kind == kPrompt && a.cuts != nullptr) a.cuts[blockIdx.x] = CutRecord{};
}
__device__ __forceinline__ void record(const AttentionArgs& a, const Segment& g) {
  if (!g.opens || !is_partial(a, g)) return;
  const CutRecord r{g.first_cta, g.last_cta, min(a.unit_rows, g.seq.n * a.group - g.unit * a.unit_rows), g.seq.q_row, g.head, g.unit * a.unit_rows};
  if (a.kind == kPrompt) a.cuts[blockIdx.x] = r;
  else a.cuts[g.seq.source == 0 ? prefix_record(a, g.unit, g.head) : own_record(a, g.seq.batch, g.head)] = r;
}

// Output row of row `flat` of a sequence's rows of a key head.
__device__ __forceinline__ int64_t output_row(const AttentionArgs& a, int q_row, int head, int flat) {
  const int token = flat / a.group;
  return static_cast<int64_t>(q_row + token) * a.heads + head * a.group + (flat - token * a.group);
}

// The kernels: rows of a unit and CTAs that the machine holds at once, and launch. The key block of
// each is needed by the join.
constexpr int kSimtKeyBlock = 64;
constexpr int kUmmaKeyBlock = 128;
inline bool wide_line(const AttentionArgs& a) { return a.longest_line > 0x7fffffff; }
void plan_attention_umma(AttentionArgs* a, int sms);
void plan_attention_simt(AttentionArgs* a, int sms);
int launch_attention_umma(const AttentionArgs& a, cudaStream_t s);
int launch_attention_simt(const AttentionArgs& a, cudaStream_t s);

}  // namespace b200
