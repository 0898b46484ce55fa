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
// A unit is `unit_rows` such rows of one key head; its keys are cut in blocks of kKeyBlock.
//   direct : one CTA per unit, which writes finished rows.
//   split  : too few units for the machine. All blocks of all units, in the order sequence, head,
//            unit, block, are dealt out in equal contiguous ranges, one per CTA, whatever the lengths
//            are; a unit cut by a range boundary leaves one partial result (sum, maximum, denominator)
//            per CTA that worked on it, and a second launch joins them in CTA order.
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
  // split form only
  int split, ctas;
  int64_t natural_rows;              // partial rows that belong to output rows; ctas * unit_rows follow
  int64_t* plan;                     // [0] blocks per CTA, [1 + s] first block of sequence s
  float* partial_o;                  // [row][dim], not divided by the denominator
  float2* partial_ml;                // maximum (scaled, base 2), denominator
};

struct Sequence {
  int q_row, n;        // first query row, queries
  int k_row, m;        // first key row, keys
  int source, batch;   // which pair of key and value arrays
};

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
  return static_cast<int>((static_cast<int64_t>(s.n) * a.group + a.unit_rows - 1) / a.unit_rows);
}

template <int kKeyBlock>
__device__ __forceinline__ int unit_blocks(const AttentionArgs& a, const Sequence& s, int unit) {
  const int64_t last = ((static_cast<int64_t>(unit) + 1) * a.unit_rows - 1) / a.group;
  const int keys = visible_keys(a, s, static_cast<int>(last < s.n - 1 ? last : s.n - 1));
  return (keys + kKeyBlock - 1) / kKeyBlock;
}

// Blocks of one key head of the sequence.
template <int kKeyBlock>
__device__ __forceinline__ int64_t head_blocks(const AttentionArgs& a, const Sequence& s) {
  const int units = unit_count(a, s);
  if (units == 0 || s.m == 0) return 0;
  if (a.kind == kShared || a.causal == 0) return static_cast<int64_t>(units) * unit_blocks<kKeyBlock>(a, s, 0);
  int64_t sum = 0;
  for (int t = 0; t < units; ++t) sum += unit_blocks<kKeyBlock>(a, s, t);
  return sum;
}

// ------------------------------------------------------------------------- finding a CTA's work

struct WorkStart {
  int sequence;     // -1: nothing to do
  int64_t offset;   // within the sequence
  int64_t total, first;
};

struct WorkScratch {
  int64_t sums[32];
  WorkStart start;
};

// Prefix sums of weight(s) over the sequences by all kThreads threads of the CTA; then the sequence
// that holds position target(total). `record` is called once per sequence with its first position.
template <int kThreads, class Weight, class Target, class Record>
__device__ __forceinline__ WorkStart find_work(int count, WorkScratch* scratch, const Weight& weight, const Target& target,
                                               const Record& record) {
  const int chunk = (count + kThreads - 1) / kThreads;
  const int lo = min(static_cast<int>(threadIdx.x) * chunk, count), hi = min(lo + chunk, count);
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
  const int64_t wanted = target(total);
  if (threadIdx.x == 0) scratch->start = WorkStart{-1, 0, total, wanted};
  __syncthreads();
  for (int s = lo; s < hi; ++s) {
    record(s, before, total);
    const int64_t size = weight(s);
    if (wanted >= before && wanted < before + size) scratch->start = WorkStart{s, wanted - before, total, wanted};
    before += size;
  }
  __syncthreads();
  return scratch->start;
}

// A contiguous run of key blocks of one unit.
struct Segment {
  Sequence seq;
  int head, unit;
  int block_begin, block_end;   // of the unit's blocks
  bool opens;                   // starts at the unit's first block
};

// Walks the segments of a CTA: one whole unit in the direct form, a range of blocks in the split form.
// Every role of a CTA walks for itself and sees the same segments.
template <int kKeyBlock>
struct SegmentWalk {
  const AttentionArgs& a;
  int sequence;
  int64_t left;      // blocks still to be handed out (split)
  Sequence seq;
  int head, unit, block;
  bool more;

  __device__ __forceinline__ SegmentWalk(const AttentionArgs& args, const WorkStart& start) : a(args), sequence(start.sequence) {
    more = sequence >= 0;
    if (!more) return;
    seq = sequence_of(a, sequence);
    if (a.split == 0) {   // blockIdx.x % kv_heads is the head, the offset the unit
      head = blockIdx.x % a.kv_heads, unit = static_cast<int>(start.offset), block = 0, left = 0;
      return;
    }
    const int64_t per = (start.total + a.ctas - 1) / a.ctas;
    left = min(per, start.total - start.first);
    const int64_t per_head = head_blocks<kKeyBlock>(a, seq);
    head = static_cast<int>(start.offset / per_head);
    int64_t rest = start.offset - head * per_head;
    unit = 0;
    while (rest >= unit_blocks<kKeyBlock>(a, seq, unit)) rest -= unit_blocks<kKeyBlock>(a, seq, unit), ++unit;
    block = static_cast<int>(rest);
  }

  __device__ __forceinline__ bool next(Segment* out) {
    if (!more) return false;
    if (a.split == 0) {
      *out = Segment{seq, head, unit, 0, unit_blocks<kKeyBlock>(a, seq, unit), true};
      more = false;
      return true;
    }
    int blocks = unit_blocks<kKeyBlock>(a, seq, unit);
    while (block >= blocks) {   // on to the next unit that has blocks; there is one while `left` > 0
      block = 0;
      if (++unit >= unit_count(a, seq)) {
        unit = 0;
        if (++head >= a.kv_heads) {
          head = 0;
          do seq = sequence_of(a, ++sequence);
          while (unit_count(a, seq) == 0 || seq.m == 0);
        }
      }
      blocks = unit_blocks<kKeyBlock>(a, seq, unit);
    }
    const int take = static_cast<int>(min(static_cast<int64_t>(blocks - block), left));
    *out = Segment{seq, head, unit, block, block + take, block == 0};
    block += take;
    left -= take;
    more = left > 0;
    return true;
  }
};

template <int kKeyBlock, int kThreads>
__device__ __forceinline__ WorkStart find_attention_work(const AttentionArgs& a, WorkScratch* scratch) {
  const int count = sequence_count(a);
  if (a.split == 0) {
    // The units that see most keys are the last of a sequence: they go first.
    return find_work<kThreads>(
        count, scratch, [&](int s) -> int64_t { return unit_count(a, sequence_of(a, s)); },
        [&](int64_t total) -> int64_t { return total - 1 - static_cast<int64_t>(blockIdx.x / a.kv_heads); }, [](int, int64_t, int64_t) {});
  }
  return find_work<kThreads>(
      count, scratch, [&](int s) -> int64_t { return a.kv_heads * head_blocks<kKeyBlock>(a, sequence_of(a, s)); },
      [&](int64_t total) -> int64_t { return blockIdx.x * ((total + a.ctas - 1) / a.ctas); },
      [&](int s, int64_t first, int64_t total) {
        if (blockIdx.x != 0) return;
        a.plan[1 + s] = first;
        if (s == 0) a.plan[0] = (total + a.ctas - 1) / a.ctas;
      });
}

// Where row `flat` (of the sequence's rows of a key head) of a segment goes.
__device__ __forceinline__ int64_t output_row(const AttentionArgs& a, const Segment& g, int64_t flat) {
  return (g.seq.q_row + flat / a.group) * a.heads + g.head * a.group + flat % a.group;
}
__device__ __forceinline__ int64_t partial_row(const AttentionArgs& a, const Segment& g, int64_t flat) {
  if (g.opens) return output_row(a, g, flat) + (g.seq.source == 1 ? static_cast<int64_t>(a.q_rows) * a.heads : 0);
  return a.natural_rows + static_cast<int64_t>(blockIdx.x) * a.unit_rows + (flat - static_cast<int64_t>(g.unit) * a.unit_rows);
}

// Launchers of the kernels; the key block of each is needed by the join.
constexpr int kSimtKeyBlock = 64;
constexpr int kUmmaKeyBlock = 128;
int launch_attention_umma(const AttentionArgs& a, cudaStream_t s, int64_t units);
void plan_attention_umma(AttentionArgs* a, int sms);
int launch_attention_simt(const AttentionArgs& a, cudaStream_t s, int64_t units);
void plan_attention_simt(AttentionArgs* a, int sms);

}  // namespace b200
