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

// Joins the partial results c of one row, a warp per row, in CTA order:
// O = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c. One with l = 0 saw no key; its O is not read.
struct RowJoin {
  float top = kMinusInf, total = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);

  __device__ __forceinline__ void add(const AttentionArgs& a, int64_t at, int lane) {
    const float2 ml = a.partial_ml[at];
    if (ml.y == 0.f) return;
    const float next = fmaxf(top, ml.x);
    const float base = next == kMinusInf ? 0.f : next;   // maxima of -infinity with l != 0: NaN rows
    const float keep = exp2f(top - base), more = exp2f(ml.x - base);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (lane * 4 < a.dim) v = *reinterpret_cast<const float4*>(a.partial_o + at * a.dim + lane * 4);
    sum = make_float4(sum.x * keep + v.x * more, sum.y * keep + v.y * more, sum.z * keep + v.z * more, sum.w * keep + v.w * more);
    total = total * keep + ml.y * more;
    top = next;
  }
  __device__ __forceinline__ void store(const AttentionArgs& a, int64_t row, int lane) const {
    const float inv = total == 0.f ? 0.f : 1.f / total;
    if (lane * 4 < a.dim) store_row4(a.out, a.dtype, row * a.dim + lane * 4, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
  }
};

// Prompt calls: block (c, y) handles rows y, y + gridDim.y, ... (in groups of a warp each) of the unit
// that boundary c cuts, if c is the first that does.
template <int kKeys>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_cuts_kernel(const AttentionArgs a) {
  __shared__ WorkScratch scratch;
  grid_launch_dependents();
  grid_dependency_wait();
  const int cta = blockIdx.x + 1;
  const WorkStart start = find_range<kKeys, kJoinWarps * 32>(a, &scratch, cta);
  if (start.sequence < 0 || start.block == 0 || start.before / start.per != cta - 1) return;
  const Sequence seq = sequence_of(a, start.sequence);
  const int last = static_cast<int>((start.before + unit_weight<kKeys>(a, seq, start.unit) - 1) / start.per);
  const int row0 = start.unit * a.unit_rows;
  const int rows = min(a.unit_rows, seq.n * a.group - row0);
  const int lane = threadIdx.x & 31;
  for (int r = blockIdx.y * kJoinWarps + (threadIdx.x >> 5); r < rows; r += gridDim.y * kJoinWarps) {
    RowJoin join;
    const int64_t out = output_row(a, seq, start.head, row0 + r);
    join.add(a, opened_row(a, seq, out, cta - 1, r), lane);
    for (int c = cta; c <= last; ++c) join.add(a, continued_row(a, c, r), lane);
    join.store(a, out, lane);
  }
}

// Shared-prefix calls: a warp per row, which has a part over the prefix and one over its own keys. All
// rows of a block belong to one request (blockIdx.x); the block finds the requests' first blocks by
// itself.
template <int kKeys>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_rows_kernel(const AttentionArgs a) {
  __shared__ int64_t sums[2][kJoinWarps];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, request = blockIdx.x;
  const auto head_size = [&](int s) { return head_weight<kKeys>(a, sequence_of(a, s)); };
  int64_t all = 0, before = 0;   // blocks of a key head: of all sequences, and of those ahead of this request
  for (int s = threadIdx.x; s < a.sequences; s += kJoinWarps * 32) {
    const int64_t size = head_size(s);
    all += size;
    if (s < request + 1) before += size;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o), before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) sums[0][threadIdx.x >> 5] = all, sums[1][threadIdx.x >> 5] = before;
  __syncthreads();
  all = before = 0;
  for (int w = 0; w < kJoinWarps; ++w) all += sums[0][w], before += sums[1][w];
  const int64_t per = quotient(a.kv_heads * all + a.ctas - 1, a.ctas);
  const Sequence prefix = sequence_of(a, 0), own = sequence_of(a, 1 + request);
  for (int h = blockIdx.y * kJoinWarps + (threadIdx.x >> 5); h < a.heads; h += gridDim.y * kJoinWarps) {
    const int head = h / a.group, g = h - head * a.group;
    RowJoin join;
    const int64_t out = static_cast<int64_t>(request) * a.heads + h;
    const auto part = [&](const Sequence& seq, int64_t first_of_sequence, int flat) {
      const int unit = flat / a.unit_rows, row = flat - unit * a.unit_rows;
      const int blocks = unit_blocks<kKeys>(a, seq, unit);
      if (blocks == 0) return;
      const int64_t first = first_of_sequence + head * head_weight<kKeys>(a, seq) + weight_before<kKeys>(a, seq, unit);
      const int c0 = static_cast<int>(quotient(first, per)), c1 = static_cast<int>(quotient(first + blocks - 1, per));
      join.add(a, opened_row(a, seq, out, c0, row), lane);
      for (int c = c0 + 1; c <= c1; ++c) join.add(a, continued_row(a, c, row), lane);
    };
    part(prefix, 0, request * a.group + g);
    part(own, a.kv_heads * before, g);
    join.store(a, out, lane);
  }
}

// FP32 operands would lose half their bits on the tensor cores; 16-bit ones lose nothing.
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

template <int kKeys>
int join(const AttentionArgs& a, cudaStream_t s) {
  if (a.kind == kShared) {
    const unsigned share = static_cast<unsigned>((a.heads + kJoinWarps - 1) / kJoinWarps);
    return launch_join(attention_join_rows_kernel<kKeys>, dim3(static_cast<unsigned>(a.q_rows), share < 32 ? share : 32), a, s);
  }
  return a.ctas < 2 ? B200_OK : launch_join(attention_join_cuts_kernel<kKeys>, dim3(static_cast<unsigned>(a.ctas) - 1, 8), a, s);
}

// ------------------------------------------------------------------- arguments

size_t element_bytes(int dtype) { return dtype == B200_FP32 ? 4 : 2; }

int check_common(int dtype, int heads, int kv_heads, int dim, float scale) {
  if (dtype < B200_FP32 || dtype > B200_BF16) return B200_ERR_INVALID_ARGUMENT;
  if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0) return B200_ERR_INVALID_ARGUMENT;
  if (!(scale > 0.f) || scale > 3.0e38f) return B200_ERR_INVALID_ARGUMENT;
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

// Decomposition, without the lengths: returns whether there may be partial results.
bool plan(AttentionArgs* a) {
  const int sms = sm_count() > 0 ? sm_count() : 1;
  on_tensor_cores(*a) ? plan_attention_umma(a, sms) : plan_attention_simt(a, sms);
  a->token_shift = log2_or_minus_one(a->tokens);
  const int64_t keys = on_tensor_cores(*a) ? kUmmaKeyBlock : kSimtKeyBlock;
  const auto blocks = [&](int64_t rows) { return (rows + keys - 1) / keys; };
  if (a->kind == kShared) {
    // Never more ranges than blocks.
    const int64_t own = (a->group + a->unit_rows - 1) / a->unit_rows * static_cast<int64_t>(a->q_rows) * blocks(a->room);
    const int64_t prefix = (static_cast<int64_t>(a->q_rows) * a->group + a->unit_rows - 1) / a->unit_rows * blocks(a->k_rows);
    const int64_t most = (own + prefix) * a->kv_heads;
    if (most < a->ctas) a->ctas = static_cast<int>(most > 0 ? most : 1);
    return true;
  }
  // Each sequence, and the rows behind them, rounds up once.
  const int64_t units = (static_cast<int64_t>(a->q_rows) * a->group / a->unit_rows + a->sequences + 1) * a->kv_heads;
  const int64_t longest = blocks(a->k_rows) > 0 ? blocks(a->k_rows) : 1;
  if (units < a->ctas && units * longest < a->ctas) a->ctas = static_cast<int>(units * longest);
  return longest > 1;   // units of one block are never cut
}

struct Workspace {
  size_t o, total;   // maxima and denominators first
};
Workspace workspace_of(const AttentionArgs& a) {
  const auto round = [](size_t v) { return (v + 255) & ~size_t{255}; };
  const size_t cuts = static_cast<size_t>(a.ctas) * a.unit_rows;
  const size_t rows = cuts + (a.kind == kShared ? 2 * static_cast<size_t>(a.q_rows) * a.heads : cuts);
  Workspace w{};
  w.o = round(rows * sizeof(float2));
  w.total = w.o + round(rows * a.dim * sizeof(float));
  return w;
}

int run(AttentionArgs& a, void* workspace, size_t bytes, cudaStream_t s) {
  const bool partial = plan(&a);
  if (partial) {
    const Workspace w = workspace_of(a);
    if (workspace == nullptr || bytes < w.total) return B200_ERR_INVALID_ARGUMENT;
    if (!aligned16(workspace)) return B200_ERR_MISALIGNED_OPERAND;
    a.partial_ml = static_cast<float2*>(workspace);
    a.partial_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + w.o);
  }
  const int rc = on_tensor_cores(a) ? launch_attention_umma(a, s) : launch_attention_simt(a, s);
  if (rc != B200_OK || !partial) return rc;
  return on_tensor_cores(a) ? join<kUmmaKeyBlock>(a, s) : join<kSimtKeyBlock>(a, s);
}

template <class Problem>
size_t workspace_bytes(const Problem* problem) {
  AttentionArgs a;
  if (problem == nullptr || make_args(*problem, &a) != B200_OK) return 0;
  return plan(&a) ? workspace_of(a).total : 0;
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
