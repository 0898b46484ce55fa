// Entry points of the attention operators: checks, workspace layout, and the passes that join partial
// results.
#include "attention.cuh"

namespace b200 {
namespace {

constexpr float kMinusInf = -__builtin_huge_valf();
constexpr int kJoinWarps = 4;

__device__ __forceinline__ void store_row4(void* out, int dtype, int64_t at, float4 v) {
  if (dtype == B200_FP32) {
    *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = v;
  } else if (dtype == B200_FP16) {
    __half2* p = reinterpret_cast<__half2*>(static_cast<__half*>(out) + at);
    p[0] = __floats2half2_rn(v.x, v.y), p[1] = __floats2half2_rn(v.z, v.w);
  } else {
    __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(out) + at);
    p[0] = __floats2bfloat162_rn(v.x, v.y), p[1] = __floats2bfloat162_rn(v.z, v.w);
  }
}

// O = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over the partial results c of a row, in CTA order.
// One with l = 0 saw no key; its O is not used. A CTA joins eight rows: lane (r, q) of warp w holds
// columns 4 (4 k + q) .. + 3, k = w and w + 4, of row r, so that slots are read and rows written in whole
// sectors, and up to four partial results of a row are on their way at a time.
struct RowJoin {
  const AttentionArgs& a;
  int quad[2];   // of four columns
  float top = kMinusInf, total = 0.f;
  float4 sum[2];

  __device__ __forceinline__ explicit RowJoin(const AttentionArgs& args) : a(args) {
    quad[0] = (threadIdx.x >> 5) * 4 + (threadIdx.x & 31) / 8, quad[1] = quad[0] + 16;
    sum[0] = sum[1] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  struct Part {
    float2 ml;
    float4 o[2];
  };
  __device__ __forceinline__ Part load(int64_t slot, int pitch, int row) const {
    Part p;
    p.ml = a.partial_ml[slot + row];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      p.o[i] = quad[i] * 4 < a.dim ? *reinterpret_cast<const float4*>(a.partial_o + slot * a.dim + (static_cast<int64_t>(quad[i]) * pitch + row) * 4)
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
    return p;
  }
  __device__ __forceinline__ void add(const Part& p) {
    if (p.ml.y == 0.f) return;
    const float next = fmaxf(top, p.ml.x);
    const float base = next == kMinusInf ? 0.f : next;   // maxima of -infinity with l != 0: NaN rows
    const float keep = exp2f(top - base), more = exp2f(p.ml.x - base);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      sum[i] = make_float4(sum[i].x * keep + p.o[i].x * more, sum[i].y * keep + p.o[i].y * more, sum[i].z * keep + p.o[i].z * more,
                           sum[i].w * keep + p.o[i].w * more);
    total = total * keep + p.ml.y * more;
    top = next;
  }
  // The opened slot, then the continued ones of CTAs first + 1 .. last.
  __device__ __forceinline__ void unit(int64_t slot, int pitch, int row, int first, int last) {
    add(load(slot, pitch, row));
    int c = first + 1;
    for (; c + 3 <= last; c += 4) {
      Part p[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = load(continued_slot(a, c + i), a.unit_rows, row);
#pragma unroll
      for (int i = 0; i < 4; ++i) add(p[i]);
    }
    for (; c <= last; ++c) add(load(continued_slot(a, c), a.unit_rows, row));
  }
  __device__ __forceinline__ void store(int64_t row) const {
    const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (quad[i] * 4 < a.dim)
        store_row4(a.out, a.dtype, row * a.dim + quad[i] * 4, make_float4(sum[i].x * inv, sum[i].y * inv, sum[i].z * inv, sum[i].w * inv));
  }
};
static_assert(kJoinWarps == 4, "columns of a row over the warps of a CTA");

// Prompt calls: block (c, y) handles rows 8 y .. 8 y + 7 of the unit that CTA c left open.
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_cuts_kernel(const __grid_constant__ AttentionArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  const CutRecord cut = a.cuts[blockIdx.x];
  const int row = blockIdx.y * 8 + (threadIdx.x & 7);
  if (row >= cut.rows) return;
  RowJoin join(a);
  join.unit(continued_slot(a, a.ctas + blockIdx.x), a.unit_rows, row, cut.first, cut.last);
  join.store(output_row(a, cut.q_row, cut.head, cut.row0 + row));
}

// Shared-prefix calls: block (x, h) handles rows 8 x .. 8 x + 7 of key head h: their part over the
// prefix, and the one over their request's own keys.
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_rows_kernel(const __grid_constant__ AttentionArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int flat = blockIdx.x * 8 + (threadIdx.x & 7), head = blockIdx.y;
  if (flat >= a.q_rows * a.group) return;
  const int request = flat / a.group, g = flat - request * a.group;
  RowJoin join(a);
  if (a.k_rows > 0) {
    const int unit = flat / a.unit_rows;
    const CutRecord cut = a.cuts[prefix_record(a, unit, head)];
    join.unit(prefix_slot(a, unit, head), a.unit_rows, flat - unit * a.unit_rows, cut.first, cut.last);
  }
  if (sequence_of(a, 1 + request).m > 0) {
    const CutRecord cut = a.cuts[own_record(a, request, head)];
    join.unit(own_slot(a, request, head), a.group, g, cut.first, cut.last);
  }
  join.store(static_cast<int64_t>(request) * a.heads + head * a.group + g);
}

// 16-bit operands lose nothing on the tensor cores. One TF32 or BF16 term of an FP32 operand holds half of
// its bits; it would take a sum of terms, and several products for one.
bool on_tensor_cores(const AttentionArgs& a) { return a.dtype != B200_FP32; }

template <typename Kernel>
int launch_join(Kernel kernel, dim3 grid, const AttentionArgs& a, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = s;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  if (cudaLaunchKernelEx(&cfg, kernel, a) != cudaSuccess) return launch_failed();
  return launch_status();
}

int join(const AttentionArgs& a, cudaStream_t s) {
  if (a.kind == kShared)
    return launch_join(attention_join_rows_kernel, dim3(static_cast<unsigned>((a.q_rows * static_cast<int64_t>(a.group) + 7) / 8), a.kv_heads), a, s);
  return launch_join(attention_join_cuts_kernel, dim3(static_cast<unsigned>(a.ctas), (a.unit_rows + 7) / 8), a, s);
}

// ------------------------------------------------------------------- arguments

size_t element_bytes(int dtype) { return dtype == B200_FP32 ? 4 : 2; }

int check_common(int dtype, int heads, int kv_heads, int dim, float scale) {
  if (dtype < B200_FP32 || dtype > B200_BF16) return B200_ERR_INVALID_ARGUMENT;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0) return B200_ERR_INVALID_ARGUMENT;
  if (!(scale > 0.f) || scale > 2.0e38f) return B200_ERR_INVALID_ARGUMENT;
  if (dim % 8 != 0 || dim > 128 || heads / kv_heads > 128) return B200_ERR_NOT_SUPPORTED;
  return B200_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// An array with rows: there, aligned, and with strides of whole 16-byte granules.
int check_view(const b200_rows_view& v, int64_t rows, size_t element) {
  if (rows == 0) return B200_OK;
  if (v.data == nullptr || v.row_stride < 0 || v.head_stride < 0) return B200_ERR_INVALID_ARGUMENT;
  const int64_t granule = static_cast<int64_t>(16 / element);
  if (!aligned16(v.data) || v.row_stride % granule != 0 || v.head_stride % granule != 0) return B200_ERR_MISALIGNED_OPERAND;
  return B200_OK;
}

// Rows of an array, and rows of a key head (tokens times group), are counted in 32 bits on the device.
constexpr int64_t kMostRows = int64_t{1} << 30;

// What launches and workspace sizes follow from; host only.
int make_args(const b200_attention_prompt_problem& q, AttentionArgs* a) {
  if (const int rc = check_common(q.dtype, q.heads, q.kv_heads, q.dim, q.scale); rc != B200_OK) return rc;
  if (q.sequences < 0 || q.q_rows < 0 || q.k_rows < 0) return B200_ERR_INVALID_ARGUMENT;
  if (q.q_rows > kMostRows || q.k_rows > kMostRows || q.sequences > kMostRows ||
      q.q_rows * (q.heads / q.kv_heads) > kMostRows)
    return B200_ERR_INVALID_PROBLEM;
  *a = AttentionArgs{};
  a->kind = kPrompt, a->dtype = q.dtype, a->sequences = q.sequences;
  a->q_rows = static_cast<int>(q.q_rows), a->k_rows = static_cast<int>(q.k_rows);
  a->heads = q.heads, a->kv_heads = q.kv_heads, a->group = q.heads / q.kv_heads, a->dim = q.dim;
  a->scale_log2 = q.scale * 1.4426950408889634f, a->causal = q.causal != 0;
  a->q = q.q.data, a->q_row = q.q.row_stride, a->q_head = q.q.head_stride;
  a->k[0] = q.k.data, a->k_row[0] = q.k.row_stride, a->k_head[0] = q.k.head_stride;
  a->v[0] = q.v.data, a->v_row[0] = q.v.row_stride, a->v_head[0] = q.v.head_stride;
  a->out = q.out, a->cu_q = q.cu_q, a->cu_k = q.cu_k;
  return B200_OK;
}

int make_args(const b200_attention_shared_problem& q, AttentionArgs* a) {
  if (const int rc = check_common(q.dtype, q.heads, q.kv_heads, q.dim, q.scale); rc != B200_OK) return rc;
  if (q.batch < 0 || q.prefix < 0 || q.room < 0 || q.k_batch_stride < 0 || q.v_batch_stride < 0) return B200_ERR_INVALID_ARGUMENT;
  if (q.batch > kMostRows || q.prefix > kMostRows || q.room > kMostRows || q.batch * (q.heads / q.kv_heads) > kMostRows)
    return B200_ERR_INVALID_PROBLEM;
  *a = AttentionArgs{};
  a->kind = kShared, a->dtype = q.dtype, a->sequences = static_cast<int>(q.batch) + 1;
  a->q_rows = static_cast<int>(q.batch), a->k_rows = static_cast<int>(q.prefix), a->room = static_cast<int>(q.room);
  a->heads = q.heads, a->kv_heads = q.kv_heads, a->group = q.heads / q.kv_heads, a->dim = q.dim;
  a->scale_log2 = q.scale * 1.4426950408889634f;
  a->q = q.q.data, a->q_row = q.q.row_stride, a->q_head = q.q.head_stride;
  a->k[0] = q.k_prefix.data, a->k_row[0] = q.k_prefix.row_stride, a->k_head[0] = q.k_prefix.head_stride;
  a->v[0] = q.v_prefix.data, a->v_row[0] = q.v_prefix.row_stride, a->v_head[0] = q.v_prefix.head_stride;
  a->k[1] = q.k_cache.data, a->k_row[1] = q.k_cache.row_stride, a->k_head[1] = q.k_cache.head_stride, a->k_batch = q.k_batch_stride;
  a->v[1] = q.v_cache.data, a->v_row[1] = q.v_cache.row_stride, a->v_head[1] = q.v_cache.head_stride, a->v_batch = q.v_batch_stride;
  a->out = q.out, a->lengths = q.lengths;
  return B200_OK;
}

// Decomposition, as far as it does not depend on the lengths.
struct Plan {
  int status;
  bool partial;   // there may be partial results
};
Plan plan(AttentionArgs* a) {
  const int sms = sm_count() > 0 ? sm_count() : 1;
  on_tensor_cores(*a) ? plan_attention_umma(a, sms) : plan_attention_simt(a, sms);
  a->token_shift = log2_or_minus_one(a->tokens);
  const int64_t keys = on_tensor_cores(*a) ? kUmmaKeyBlock : kSimtKeyBlock;
  const auto blocks = [&](int64_t rows) { return (rows + keys - 1) / keys; };
  const auto units = [&](int64_t rows) { return (rows + a->unit_rows - 1) / a->unit_rows; };
  const int64_t longest = blocks(a->k_rows);
  __int128 most;       // length of the line
  __int128 ranges;     // more CTAs than this would have nothing to do
  if (a->kind == kShared) {
    if (a->kv_heads > 65535) return {B200_ERR_INVALID_PROBLEM, false};   // a dimension of the join's grid
    const __int128 prefix = units(static_cast<int64_t>(a->q_rows) * a->group), own = a->q_rows;
    ranges = (prefix * longest + own * blocks(a->room)) * a->kv_heads;
    most = (ranges << a->pair_shift) + (prefix + own) * a->kv_heads * a->unit_cost;
  } else {
    // Each sequence, and the rows behind them, rounds up once.
    const __int128 whole = a->q_rows / a->tokens, all = whole + a->sequences + 1;
    ranges = all * a->kv_heads * (longest > 0 ? longest : 1);
    // A sequence of n queries and m keys has at most n / tokens + 1 units of m / keys + 1 blocks. Summed
    // over sequences that do not overlap: n m to at most all queries by all keys, n and m to all of them.
    const __int128 all_keys = a->k_rows / keys + 1;
    most = ((((whole + 1) * all_keys + whole + 1 + all_keys + a->sequences) << a->pair_shift) + all * a->unit_cost) * a->kv_heads;
  }
  // On the device the line is counted in 64 bits, with room for a sum per thread. It would take years to
  // work through.
  if (most >= __int128{1} << 54) return {B200_ERR_INVALID_PROBLEM, false};
  a->longest_line = static_cast<int64_t>(most);
  if (ranges < a->ctas) a->ctas = static_cast<int>(ranges > 0 ? ranges : 1);
  return {B200_OK, a->kind == kShared || longest > 1};   // units of one block are never cut
}

struct Workspace {
  size_t cuts, o, total;   // maxima and denominators first
};
Workspace workspace_of(const AttentionArgs& a) {
  const auto round = [](size_t v) { return (v + 255) & ~size_t{255}; };
  const auto units = [&](size_t rows) { return (rows + a.unit_rows - 1) / a.unit_rows; };
  size_t rows = static_cast<size_t>(a.ctas) * a.unit_rows, records = a.ctas;
  if (a.kind == kPrompt) {
    rows *= 2;
  } else {
    const size_t prefix = units(static_cast<size_t>(a.q_rows) * a.group) * a.kv_heads;
    rows += prefix * a.unit_rows + static_cast<size_t>(a.q_rows) * a.heads;
    records = prefix + static_cast<size_t>(a.q_rows) * a.kv_heads;
  }
  Workspace w{};
  w.cuts = round(rows * sizeof(float2));
  w.o = w.cuts + round(records * sizeof(CutRecord));
  w.total = w.o + round(rows * a.dim * sizeof(float));
  return w;
}

int run(AttentionArgs& a, void* workspace, size_t bytes, cudaStream_t s) {
  const Plan planned = plan(&a);
  if (planned.status != B200_OK) return planned.status;
  if (planned.partial) {
    const Workspace w = workspace_of(a);
    if (workspace == nullptr || bytes < w.total) return B200_ERR_INVALID_ARGUMENT;
    if (!aligned16(workspace)) return B200_ERR_MISALIGNED_OPERAND;
    uint8_t* base = static_cast<uint8_t*>(workspace);
    a.partial_ml = reinterpret_cast<float2*>(base);
    a.cuts = reinterpret_cast<CutRecord*>(base + w.cuts);
    a.partial_o = reinterpret_cast<float*>(base + w.o);
  }
  const int rc = on_tensor_cores(a) ? launch_attention_umma(a, s) : launch_attention_simt(a, s);
  return rc != B200_OK || !planned.partial ? rc : join(a, s);
}

template <class Problem>
size_t workspace_bytes(const Problem* problem) {
  AttentionArgs a;
  if (problem == nullptr || make_args(*problem, &a) != B200_OK) return 0;
  const Plan planned = plan(&a);
  return planned.status == B200_OK && planned.partial ? workspace_of(a).total : 0;
}

}  // namespace
}  // namespace b200

extern "C" {

size_t b200_attention_prompt_workspace_bytes(const b200_attention_prompt_problem* problem) { return b200::workspace_bytes(problem); }
size_t b200_attention_shared_workspace_bytes(const b200_attention_shared_problem* problem) { return b200::workspace_bytes(problem); }

int b200_attention_prompt(const b200_attention_prompt_problem* problem, void* workspace, size_t workspace_bytes, b200_stream_t stream) {
  if (problem == nullptr) return B200_ERR_INVALID_ARGUMENT;
  const b200_attention_prompt_problem& q = *problem;
  b200::AttentionArgs a;
  if (const int rc = b200::make_args(q, &a); rc != B200_OK) return rc;
  if (q.q_rows == 0) return B200_OK;
  if (q.out == nullptr || q.cu_q == nullptr || q.cu_k == nullptr) return B200_ERR_INVALID_ARGUMENT;
  const size_t element = b200::element_bytes(q.dtype);
  if (const int rc = b200::check_view(q.q, q.q_rows, element); rc != B200_OK) return rc;
  if (const int rc = b200::check_view(q.k, q.k_rows, element); rc != B200_OK) return rc;
  if (const int rc = b200::check_view(q.v, q.k_rows, element); rc != B200_OK) return rc;
  if (!b200::aligned16(q.out)) return B200_ERR_MISALIGNED_OPERAND;
  return b200::run(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int b200_attention_shared(const b200_attention_shared_problem* problem, void* workspace, size_t workspace_bytes, b200_stream_t stream) {
  if (problem == nullptr) return B200_ERR_INVALID_ARGUMENT;
  const b200_attention_shared_problem& q = *problem;
  b200::AttentionArgs a;
  if (const int rc = b200::make_args(q, &a); rc != B200_OK) return rc;
  if (q.batch == 0) return B200_OK;
  if (q.out == nullptr || q.lengths == nullptr) return B200_ERR_INVALID_ARGUMENT;
  const size_t element = b200::element_bytes(q.dtype);
  if (const int rc = b200::check_view(q.q, q.batch, element); rc != B200_OK) return rc;
  if (const int rc = b200::check_view(q.k_prefix, q.prefix, element); rc != B200_OK) return rc;
  if (const int rc = b200::check_view(q.v_prefix, q.prefix, element); rc != B200_OK) return rc;
  if (const int rc = b200::check_view(q.k_cache, q.room, element); rc != B200_OK) return rc;
  if (const int rc = b200::check_view(q.v_cache, q.room, element); rc != B200_OK) return rc;
  const int64_t granule = static_cast<int64_t>(16 / element);
  if (!b200::aligned16(q.out) || q.k_batch_stride % granule != 0 || q.v_batch_stride % granule != 0) return B200_ERR_MISALIGNED_OPERAND;
  return b200::run(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
