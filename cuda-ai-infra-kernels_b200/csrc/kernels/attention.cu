// Entry points of the attention operators: checks, choice of the form (direct or split), workspace
// layout, and the pass that joins the partial results of the split form.
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

// One warp per output row: O = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c over the partial results
// c of the row, in a fixed order. A partial result with l = 0 saw no key; its O is not read.
template <int kKeyBlock>
__global__ void __launch_bounds__(kJoinWarps * 32) attention_join_kernel(const AttentionArgs a) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kJoinWarps + (threadIdx.x >> 5);
  if (row >= static_cast<int64_t>(a.q_rows) * a.heads) return;
  const int q_row = static_cast<int>(row / a.heads), head = static_cast<int>(row % a.heads) / a.group;
  const int g = static_cast<int>(row % a.heads) - head * a.group;

  float top = kMinusInf, total = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  const int64_t per = a.plan[0];
  const auto join = [&](int s) {
    const Sequence seq = sequence_of(a, s);
    const int64_t flat = static_cast<int64_t>(q_row - seq.q_row) * a.group + g;
    const int unit = static_cast<int>(flat / a.unit_rows);
    if (q_row < seq.q_row || q_row - seq.q_row >= seq.n || seq.m == 0) return;
    const int blocks = unit_blocks<kKeyBlock>(a, seq, unit);
    if (blocks == 0) return;
    int64_t first = a.plan[1 + s] + head * head_blocks<kKeyBlock>(a, seq);
    for (int t = 0; t < unit; ++t) first += unit_blocks<kKeyBlock>(a, seq, t);
    const int c0 = static_cast<int>(first / per), c1 = static_cast<int>((first + blocks - 1) / per);
    for (int c = c0; c <= c1; ++c) {
      const int64_t at = c == c0 ? row + (seq.source == 1 ? static_cast<int64_t>(a.q_rows) * a.heads : 0)
                                 : a.natural_rows + static_cast<int64_t>(c) * a.unit_rows + (flat - static_cast<int64_t>(unit) * a.unit_rows);
      const float2 ml = a.partial_ml[at];
      if (ml.y == 0.f) continue;
      const float next = fmaxf(top, ml.x);
      const float base = next == kMinusInf ? 0.f : next;   // maxima of -infinity with l != 0: NaN rows
      const float keep = exp2f(top - base), add = exp2f(ml.x - base);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane * 4 < a.dim) v = *reinterpret_cast<const float4*>(a.partial_o + at * a.dim + lane * 4);
      sum = make_float4(sum.x * keep + v.x * add, sum.y * keep + v.y * add, sum.z * keep + v.z * add, sum.w * keep + v.w * add);
      total = total * keep + ml.y * add;
      top = next;
    }
  };
  if (a.kind == kShared) {
    join(0);
    join(1 + q_row);
  } else {
    int lo = 0, hi = a.sequences + 1;   // the last offset that is not behind the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (__ldg(a.cu_q + mid) <= q_row) lo = mid;
      else hi = mid;
    }
    if (lo < a.sequences) join(lo);
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (lane * 4 < a.dim) store_row4(a.out, a.dtype, row * a.dim + lane * 4, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
}

// FP32 operands would lose half their bits on the tensor cores; 16-bit ones lose nothing.
bool on_tensor_cores(const AttentionArgs& a) { return a.dtype != B200_FP32; }

int launch_join(const AttentionArgs& a, cudaStream_t s) {
  const int64_t blocks = (static_cast<int64_t>(a.q_rows) * a.heads + kJoinWarps - 1) / kJoinWarps;
  if (blocks > 0x7fffffffLL) return B200_ERR_INVALID_PROBLEM;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = s;
  const GemmLaunchAttributes attrs = gemm_launch_attributes(1);
  cfg.attrs = const_cast<cudaLaunchAttribute*>(attrs.list);
  cfg.numAttrs = attrs.count;
  const cudaError_t rc = on_tensor_cores(a) ? cudaLaunchKernelEx(&cfg, attention_join_kernel<kUmmaKeyBlock>, a)
                                            : cudaLaunchKernelEx(&cfg, attention_join_kernel<kSimtKeyBlock>, a);
  if (rc != cudaSuccess) return launch_failed();
  return launch_status();
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

constexpr int64_t kMostRows = int64_t{1} << 30;   // rows are counted in 32 bits on the device

// What launches and workspace sizes follow from; host only.
int make_args(const b200_attention_prompt_problem& q, AttentionArgs* a) {
  if (const int rc = check_common(q.dtype, q.heads, q.kv_heads, q.dim, q.scale); rc != B200_OK) return rc;
  if (q.sequences < 0 || q.q_rows < 0 || q.k_rows < 0) return B200_ERR_INVALID_ARGUMENT;
  if (q.q_rows > kMostRows || q.k_rows > kMostRows || q.sequences > kMostRows) return B200_ERR_INVALID_PROBLEM;
  *a = AttentionArgs{};
  a->kind = kPrompt, a->dtype = q.dtype, a->sequences = q.sequences;
  a->q_rows = static_cast<int>(q.q_rows), a->k_rows = static_cast<int>(q.k_rows);
  a->heads = q.heads, a->kv_heads = q.kv_heads, a->group = q.heads / q.kv_heads, a->dim = q.dim;
  a->scale_log2 = q.scale * 1.4426950408889634f, a->causal = q.causal != 0;
  a->q = q.q.data, a->q_row = q.q.row_stride, a->q_head = q.q.head_stride;
  a->k[0] = q.k.data, a->k_row[0] = q.k.row_stride, a->k_head[0] = q.k.head_stride;
  a->v[0] = q.v.data, a->v_row[0] = q.v.row_stride, a->v_head[0] = q.v.head_stride;
  a->out = q.out, a->cu_q = q.cu_q, a->cu_k = q.cu_k;
  a->natural_rows = static_cast<int64_t>(a->q_rows) * a->heads;
  return B200_OK;
}

int make_args(const b200_attention_shared_problem& q, AttentionArgs* a) {
  if (const int rc = check_common(q.dtype, q.heads, q.kv_heads, q.dim, q.scale); rc != B200_OK) return rc;
  if (q.batch < 0 || q.prefix < 0 || q.room < 0 || q.k_batch_stride < 0 || q.v_batch_stride < 0) return B200_ERR_INVALID_ARGUMENT;
  if (q.batch > kMostRows || q.prefix > kMostRows || q.room > kMostRows) return B200_ERR_INVALID_PROBLEM;
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
  a->natural_rows = 2 * static_cast<int64_t>(a->q_rows) * a->heads;   // prefix parts, own parts
  return B200_OK;
}

// Upper bound of the units of one key head of a prompt call: each sequence, and the rows behind
// them, rounds up once.
int64_t unit_bound(const AttentionArgs& a) {
  return static_cast<int64_t>(a.q_rows) * a.group / a.unit_rows + a.sequences + 1;
}

void choose_form(AttentionArgs* a) {
  const int sms = sm_count() > 0 ? sm_count() : 1;
  on_tensor_cores(*a) ? plan_attention_umma(a, sms) : plan_attention_simt(a, sms);
  // A prompt is split when its rows alone would leave SMs without work; a decoding step always.
  const int64_t busy = (static_cast<int64_t>(a->q_rows) * a->group + a->unit_rows - 1) / a->unit_rows * a->kv_heads;
  a->split = a->kind == kShared || (busy < sms && a->k_rows > 4 * kSimtKeyBlock);
}

struct Workspace {
  size_t plan, ml, o, total;
};
Workspace workspace_of(const AttentionArgs& a) {
  const auto round = [](size_t v) { return (v + 255) & ~size_t{255}; };
  if (a.split == 0) return Workspace{0, 0, 0, 0};
  const size_t rows = static_cast<size_t>(a.natural_rows) + static_cast<size_t>(a.ctas) * a.unit_rows;
  Workspace w{};
  w.ml = round((static_cast<size_t>(a.sequences) + 3) * sizeof(int64_t));
  w.o = w.ml + round(rows * sizeof(float2));
  w.total = w.o + round(rows * a.dim * sizeof(float));
  return w;
}

int run(AttentionArgs& a, void* workspace, size_t bytes, cudaStream_t s) {
  choose_form(&a);
  const Workspace w = workspace_of(a);
  if (w.total > 0) {
    if (workspace == nullptr || bytes < w.total) return B200_ERR_INVALID_ARGUMENT;
    if (!aligned16(workspace)) return B200_ERR_MISALIGNED_OPERAND;
    uint8_t* base = static_cast<uint8_t*>(workspace);
    a.plan = reinterpret_cast<int64_t*>(base);
    a.partial_ml = reinterpret_cast<float2*>(base + w.ml);
    a.partial_o = reinterpret_cast<float*>(base + w.o);
  }
  const int64_t units = a.kind == kPrompt ? unit_bound(a) : 0;
  const int rc = on_tensor_cores(a) ? launch_attention_umma(a, s, units) : launch_attention_simt(a, s, units);
  if (rc != B200_OK) return rc;
  return a.split != 0 ? launch_join(a, s) : B200_OK;
}

template <class Problem>
size_t workspace_bytes(const Problem* problem) {
  AttentionArgs a;
  if (problem == nullptr || make_args(*problem, &a) != B200_OK) return 0;
  choose_form(&a);
  return workspace_of(a).total;
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
