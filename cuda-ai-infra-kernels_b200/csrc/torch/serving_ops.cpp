// PyTorch-facing launchers of the serving operators: attention over packed prompts and over a shared
// prefix, the 4-bit matrix-vector product, and the processing of logits. The reference has none of
// them; argument rules and message style are those of the other launchers here.
#include <c10/core/AutogradState.h>

#include <cmath>

#include "op_common.h"
#include "ops.h"

namespace {

using b200_torch::check_status;
using b200_torch::current_stream;

int dtype_of(const torch::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return B200_FP32;
    case torch::kFloat16: return B200_FP16;
    case torch::kBFloat16: return B200_BF16;
    default: TORCH_CHECK(false, name, " must be float32, float16 or bfloat16");
  }
}

// These operators compute no gradient: a graph that would need one, backward or forward, is refused
// instead of being cut. (torch.no_grad() does not switch tangents off.)
void check_no_gradient(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name,
              " requires a gradient, which this operator does not compute; call it under torch.no_grad()");
  TORCH_CHECK(!(c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()), name,
              " carries a forward-mode tangent, which this operator does not propagate; pass its primal");
}

void check_same(const torch::Tensor& t, const char* name, const torch::Tensor& first, const char* first_name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == first.device(), name, " and ", first_name, " must be on the same CUDA device");
}

void check_array(const torch::Tensor& t, const char* name, int64_t dims, const torch::Tensor& first, const char* first_name) {
  check_same(t, name, first, first_name);
  TORCH_CHECK(t.scalar_type() == first.scalar_type(), name, " and ", first_name, " must have the same dtype");
  TORCH_CHECK(t.dim() == dims, name, " must be ", dims, "-dimensional");
  check_no_gradient(t, name);
}

void check_limit(int64_t rows, const char* name, const char* what = "rows") {
  TORCH_CHECK(rows <= int64_t{1} << 30, name, " has too many ", what);
}

torch::Tensor int32_vector(const torch::Tensor& t, const char* name, const torch::Tensor& first, const char* first_name) {
  check_same(t, name, first, first_name);
  TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.dim() == 1, name, " must be 1-dimensional");
  check_limit(t.size(0) - 1, name, "entries");   // sequences and requests are counted in 32 bits
  return t.contiguous();
}

// The kernels take strided arrays as they are while the last dimension is dense and everything else
// sits on 16-byte granules (slices of a fused projection, head-major caches); other layouts are copied.
torch::Tensor granular(const torch::Tensor& t) {
  const int64_t granule = 16 / t.element_size();
  bool ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (t.stride(-1) == 1 || t.size(-1) == 1);
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && (t.size(d) <= 1 || (t.stride(d) > 0 && t.stride(d) % granule == 0));
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A stride of a dimension with at most one entry may be anything; it is never used.
int64_t stride_of(const torch::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

b200_rows_view rows_view(const torch::Tensor& t, int64_t row_dim) {
  return b200_rows_view{t.data_ptr(), stride_of(t, row_dim), stride_of(t, row_dim + 1)};
}

float scale_or_default(const c10::optional<double>& scale, int64_t dim) {
  const float s = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(dim)));
  TORCH_CHECK(s > 0.f && s <= 2.0e38f, "scale must be positive and finite");
  return s;
}

void check_heads(const torch::Tensor& q, int64_t kv_heads) {
  const int64_t heads = q.size(1), dim = q.size(2);
  TORCH_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "the number of query heads must be a multiple of the number of key heads");
  check_limit(heads, "q", "heads");
  TORCH_CHECK(heads / kv_heads <= 128, "at most 128 query heads per key head are supported");
  TORCH_CHECK(dim > 0 && dim % 8 == 0 && dim <= 128, "head dimension must be a multiple of 8 up to 128");
}

}  // namespace

torch::Tensor attention_prompt(const torch::Tensor& q_in, const torch::Tensor& k_in, const torch::Tensor& v_in,
                               const torch::Tensor& cu_q_in, const c10::optional<at::Tensor>& cu_k_in, bool causal,
                               c10::optional<double> scale) {
  B200_CHECK_CUDA(q_in);
  const int dtype = dtype_of(q_in, "q");
  check_array(q_in, "q", 3, q_in, "q");
  check_array(k_in, "k", 3, q_in, "q");
  check_array(v_in, "v", 3, q_in, "q");
  TORCH_CHECK(k_in.size(2) == q_in.size(2) && v_in.sizes() == k_in.sizes(), "q, k and v must be [rows, heads, dim] with k and v of one shape");
  check_heads(q_in, k_in.size(1));
  const auto cu_q = int32_vector(cu_q_in, "cu_seqlens_q", q_in, "q");
  const auto cu_k = cu_k_in.has_value() ? int32_vector(*cu_k_in, "cu_seqlens_k", q_in, "q") : cu_q;
  TORCH_CHECK(cu_q.size(0) >= 1 && cu_k.size(0) == cu_q.size(0), "cu_seqlens_q and cu_seqlens_k must hold one more offset than there are sequences");
  TORCH_CHECK(cu_k_in.has_value() || k_in.size(0) == q_in.size(0), "cu_seqlens_k is required when k has other rows than q");
  check_limit(q_in.size(0) * (q_in.size(1) / k_in.size(1)), "q");
  check_limit(k_in.size(0), "k");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const auto q = granular(q_in), k = granular(k_in), v = granular(v_in);
  auto out = torch::empty(q.sizes(), q.options());
  b200_attention_prompt_problem p{};
  p.dtype = dtype;
  p.heads = static_cast<int>(q.size(1)), p.kv_heads = static_cast<int>(k.size(1)), p.dim = static_cast<int>(q.size(2));
  p.sequences = static_cast<int>(cu_q.size(0) - 1);
  p.q_rows = q.size(0), p.k_rows = k.size(0);
  p.q = rows_view(q, 0), p.k = rows_view(k, 0), p.v = rows_view(v, 0);
  p.out = out.data_ptr();
  p.cu_q = cu_q.data_ptr<int32_t>(), p.cu_k = cu_k.data_ptr<int32_t>();
  p.scale = scale_or_default(scale, q.size(2));
  p.causal = causal;
  const size_t bytes = b200_attention_prompt_workspace_bytes(&p);
  torch::Tensor workspace;
  if (bytes > 0) workspace = torch::empty({static_cast<int64_t>(bytes)}, q.options().dtype(torch::kUInt8));
  check_status(b200_attention_prompt(&p, bytes > 0 ? workspace.data_ptr() : nullptr, bytes, current_stream(q)), "attention_prompt");
  return out;
}

torch::Tensor attention_shared_prefix(const torch::Tensor& q_in, const torch::Tensor& k_prefix_in, const torch::Tensor& v_prefix_in,
                                      const torch::Tensor& k_cache_in, const torch::Tensor& v_cache_in, const torch::Tensor& lengths_in,
                                      c10::optional<double> scale) {
  B200_CHECK_CUDA(q_in);
  const int dtype = dtype_of(q_in, "q");
  check_array(q_in, "q", 3, q_in, "q");
  check_array(k_prefix_in, "k_prefix", 3, q_in, "q");
  check_array(v_prefix_in, "v_prefix", 3, q_in, "q");
  check_array(k_cache_in, "k_cache", 4, q_in, "q");
  check_array(v_cache_in, "v_cache", 4, q_in, "q");
  const int64_t batch = q_in.size(0), kv_heads = k_prefix_in.size(1), dim = q_in.size(2);
  TORCH_CHECK(k_prefix_in.size(2) == dim && v_prefix_in.sizes() == k_prefix_in.sizes(), "k_prefix and v_prefix must be [prefix, kv_heads, dim]");
  TORCH_CHECK(k_cache_in.size(0) == batch && k_cache_in.size(2) == kv_heads && k_cache_in.size(3) == dim && v_cache_in.sizes() == k_cache_in.sizes(),
              "k_cache and v_cache must be [batch, room, kv_heads, dim]");
  check_heads(q_in, kv_heads);
  const auto lengths = int32_vector(lengths_in, "lengths", q_in, "q");
  TORCH_CHECK(lengths.size(0) == batch, "lengths must have one entry per request");
  check_limit(batch * (q_in.size(1) / kv_heads), "q");
  check_limit(k_prefix_in.size(0), "k_prefix");
  check_limit(k_cache_in.size(1), "k_cache");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const auto q = granular(q_in), k_prefix = granular(k_prefix_in), v_prefix = granular(v_prefix_in), k_cache = granular(k_cache_in),
             v_cache = granular(v_cache_in);
  auto out = torch::empty(q.sizes(), q.options());
  b200_attention_shared_problem p{};
  p.dtype = dtype;
  p.heads = static_cast<int>(q.size(1)), p.kv_heads = static_cast<int>(kv_heads), p.dim = static_cast<int>(dim);
  p.batch = batch, p.prefix = k_prefix.size(0), p.room = k_cache.size(1);
  p.q = rows_view(q, 0), p.k_prefix = rows_view(k_prefix, 0), p.v_prefix = rows_view(v_prefix, 0);
  p.k_cache = rows_view(k_cache, 1), p.v_cache = rows_view(v_cache, 1);
  p.k_batch_stride = stride_of(k_cache, 0), p.v_batch_stride = stride_of(v_cache, 0);
  p.out = out.data_ptr();
  p.lengths = lengths.data_ptr<int32_t>();
  p.scale = scale_or_default(scale, dim);
  const size_t bytes = b200_attention_shared_workspace_bytes(&p);
  const auto workspace = torch::empty({static_cast<int64_t>(bytes)}, q.options().dtype(torch::kUInt8));
  check_status(b200_attention_shared(&p, workspace.data_ptr(), bytes, current_stream(q)), "attention_shared_prefix");
  return out;
}

torch::Tensor matvec_w4(const torch::Tensor& x_in, const torch::Tensor& qweight_in, const torch::Tensor& scales_in,
                        const c10::optional<at::Tensor>& zeros_in) {
  B200_CHECK_CUDA(x_in);
  const int dtype = dtype_of(x_in, "x");
  TORCH_CHECK(x_in.dim() == 2, "x must be [rows, k]");
  check_no_gradient(x_in, "x");
  check_same(qweight_in, "qweight", x_in, "x");
  TORCH_CHECK(qweight_in.scalar_type() == torch::kUInt8 && qweight_in.dim() == 2, "qweight must be uint8 [n, k / 2]");
  check_same(scales_in, "scales", x_in, "x");
  TORCH_CHECK(scales_in.dim() == 2 && scales_in.size(0) == qweight_in.size(0), "scales must be [n, k / group]");
  TORCH_CHECK(scales_in.scalar_type() == x_in.scalar_type() || scales_in.scalar_type() == torch::kFloat32, "scales must be float32 or of x's dtype");
  check_no_gradient(scales_in, "scales");
  const int64_t rows = x_in.size(0), k = x_in.size(1), n = qweight_in.size(0), groups = scales_in.size(1);
  TORCH_CHECK(qweight_in.size(1) * 2 == k, "qweight must be [n, k / 2]");
  TORCH_CHECK(rows <= 16, "matvec_w4 takes at most 16 rows");
  TORCH_CHECK(groups > 0 && k > 0 && k % groups == 0 && (k / groups) % 32 == 0, "k / scales.size(1), the group size, must be a multiple of 32");
  TORCH_CHECK(n <= 0x7fffffff - 16 && k <= 0x7fffffff, "qweight is too large");
  const c10::cuda::CUDAGuard guard(x_in.device());
  const auto aligned = [](const torch::Tensor& t) {
    const auto c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
  };
  const auto x = aligned(x_in), qweight = aligned(qweight_in);
  const auto scales = scales_in.contiguous();
  torch::Tensor zeros;
  if (zeros_in.has_value()) {
    check_same(*zeros_in, "zeros", x_in, "x");
    TORCH_CHECK(zeros_in->scalar_type() == torch::kUInt8 && zeros_in->sizes() == scales_in.sizes(), "zeros must be uint8 of the shape of scales");
    zeros = zeros_in->contiguous();
  }
  auto y = torch::empty({rows, n}, x.options());
  b200_matvec_w4_problem p{};
  p.dtype = dtype, p.scale_dtype = dtype_of(scales, "scales");
  p.rows = static_cast<int>(rows), p.n = static_cast<int>(n), p.k = static_cast<int>(k), p.group = static_cast<int>(k / groups);
  p.x = x.data_ptr(), p.qweight = qweight.data_ptr<uint8_t>(), p.scales = scales.data_ptr();
  p.zeros = zeros.defined() ? zeros.data_ptr<uint8_t>() : nullptr;
  p.y = y.data_ptr();
  check_status(b200_matvec_w4(&p, current_stream(x)), "matvec_w4");
  return y;
}

torch::Tensor process_logits(const torch::Tensor& logits_in, const c10::optional<at::Tensor>& prompt_tokens_in,
                             const c10::optional<at::Tensor>& output_tokens_in, const c10::optional<at::Tensor>& repetition_in,
                             const c10::optional<at::Tensor>& frequency_in, const c10::optional<at::Tensor>& presence_in,
                             const c10::optional<at::Tensor>& bias_ids_in, const c10::optional<at::Tensor>& bias_values_in,
                             const c10::optional<at::Tensor>& allowed_in) {
  B200_CHECK_CUDA(logits_in);
  b200_logits_problem p{};
  p.dtype = dtype_of(logits_in, "logits");
  TORCH_CHECK(logits_in.dim() == 2, "logits must be [rows, vocab]");
  check_no_gradient(logits_in, "logits");
  const int64_t rows = logits_in.size(0), vocab = logits_in.size(1);
  TORCH_CHECK(vocab <= int64_t{1} << 30, "logits have too many columns");
  const c10::cuda::CUDAGuard guard(logits_in.device());
  std::vector<torch::Tensor> keep;   // contiguous copies live until the launch
  const auto table = [&](const c10::optional<at::Tensor>& in, const char* name, at::ScalarType type, const char* type_name) -> const torch::Tensor* {
    if (!in.has_value()) return nullptr;
    check_same(*in, name, logits_in, "logits");
    TORCH_CHECK(in->scalar_type() == type, name, " must be ", type_name);
    TORCH_CHECK(in->dim() == 2 && in->size(0) == rows, name, " must have one row per row of logits");
    check_no_gradient(*in, name);
    keep.push_back(in->contiguous());
    return &keep.back();
  };
  const auto per_row = [&](const c10::optional<at::Tensor>& in, const char* name) -> const float* {
    if (!in.has_value()) return nullptr;
    check_same(*in, name, logits_in, "logits");
    TORCH_CHECK(in->scalar_type() == torch::kFloat32 && in->dim() == 1 && in->size(0) == rows, name, " must be float32 [rows]");
    check_no_gradient(*in, name);
    keep.push_back(in->contiguous());
    return keep.back().data_ptr<float>();
  };
  keep.reserve(16);
  if (const auto* t = table(prompt_tokens_in, "prompt_tokens", torch::kInt32, "int32")) p.prompt_tokens = t->data_ptr<int32_t>(), p.prompt_length = t->size(1);
  if (const auto* t = table(output_tokens_in, "output_tokens", torch::kInt32, "int32")) p.output_tokens = t->data_ptr<int32_t>(), p.output_length = t->size(1);
  p.repetition = per_row(repetition_in, "repetition_penalty");
  p.frequency = per_row(frequency_in, "frequency_penalty");
  p.presence = per_row(presence_in, "presence_penalty");
  TORCH_CHECK(bias_ids_in.has_value() == bias_values_in.has_value(), "bias_ids and bias_values go together");
  if (const auto* t = table(bias_ids_in, "bias_ids", torch::kInt32, "int32")) p.bias_ids = t->data_ptr<int32_t>(), p.bias_length = t->size(1);
  if (const auto* t = table(bias_values_in, "bias_values", torch::kFloat32, "float32")) {
    TORCH_CHECK(t->size(1) == p.bias_length, "bias_ids and bias_values must have the same shape");
    p.bias_values = t->data_ptr<float>();
  }
  if (allowed_in.has_value()) {
    check_same(*allowed_in, "allowed", logits_in, "logits");
    TORCH_CHECK(allowed_in->scalar_type() == torch::kInt32 && allowed_in->dim() == 2 && (allowed_in->size(0) == rows || allowed_in->size(0) == 1) &&
                    allowed_in->size(1) == (vocab + 31) / 32,
                "allowed must be int32 [rows or 1, (vocab + 31) / 32]");
    keep.push_back(allowed_in->contiguous());
    p.allowed = keep.back().data_ptr<int32_t>();
    p.allowed_stride = allowed_in->size(0) == 1 ? 0 : keep.back().size(1);
  }
  auto x = logits_in.contiguous();
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0) x = x.clone();
  auto out = torch::empty_like(x);
  p.rows = rows, p.vocab = vocab, p.logits = x.data_ptr(), p.out = out.data_ptr();
  // Empty tables have no address; they say nothing.
  if (p.prompt_length == 0) p.prompt_tokens = nullptr;
  if (p.output_length == 0) p.output_tokens = nullptr;
  if (p.bias_length == 0) p.bias_ids = nullptr, p.bias_values = nullptr;
  check_status(b200_process_logits(&p, current_stream(x)), "process_logits");
  return out;
}
