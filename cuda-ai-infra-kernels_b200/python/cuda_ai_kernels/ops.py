"""Python operator wrappers over the native module ``cuda_ai_kernels._C``.

Behaviour mirrors python/cuda_ai_kernels/ops.py:9-101 of the reference: string
selected implementations, ``ValueError`` for unknown names, ladder GEMMs receive
the caller's tensors as they are (no copy, no transpose, no fallback), every
other operator makes its arguments contiguous first.
"""
from typing import Optional

import torch

from cuda_ai_kernels import _C
from cuda_ai_kernels.gemm_stages import COLUMN_MAJOR_IMPLS

_GEMM_IMPLS = {
    "cublas": _C.gemm_cublas,
    "naive": _C.gemm_naive,
    "block_tile": _C.gemm_block_tile,
    "thread_tile": _C.gemm_thread_tile,
    "block_tile_float4_16x16": _C.gemm_block_tile_float4_16x16,
    "block_tile_float4_16x32": _C.gemm_block_tile_float4_16x32,
    "block_tile_float4_32x32": _C.gemm_block_tile_float4_32x32,
    "thread_tile_4x4": _C.gemm_thread_tile_4x4,
    "thread_tile_4x8": _C.gemm_thread_tile_4x8,
    "thread_tile_8x8": _C.gemm_thread_tile_8x8,
    "thread_tile_8x8_warp4x8": _C.gemm_thread_tile_8x8_warp4x8,
    "warp_tile": _C.gemm_warp_tile,
    "tensor_core": _C.gemm_tensor_core,
    "prefetch_smem": _C.gemm_prefetch_smem,
    "prefetch_reg": _C.gemm_prefetch_reg,
    "split_k": _C.gemm_split_k,
    "cutlass": _C.gemm_cutlass,
}

_RMSNORM_IMPLS = {
    "naive": _C.rmsnorm_naive,
    "cache_x": _C.rmsnorm_cache_x,
}

_SOFTMAX_IMPLS = {
    "naive": _C.softmax_naive,
}


def gemm(a: torch.Tensor, b: torch.Tensor, impl: str = "naive") -> torch.Tensor:
    """FP32 ``A[M,K] @ B[K,N]``.

    Ladder implementations (``gemm_stages.GEMM_STAGES`` and the alias
    ``thread_tile``) need A as a column-major view (strides ``(1, M)``), B
    row-major, and M, N, K positive multiples of the entry's tile; nothing is
    converted on the caller's behalf. ``cublas`` also takes a row-major A.
    ``tensor_core`` and ``cutlass`` are row-major TF32 entries for any shape.
    """
    if impl not in _GEMM_IMPLS:
        raise ValueError(f"unknown GEMM impl: {impl}")
    fn = _GEMM_IMPLS[impl]
    if impl in COLUMN_MAJOR_IMPLS:
        return fn(a, b)
    return fn(a.contiguous(), b.contiguous())


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, impl: str = "naive") -> torch.Tensor:
    """``x * rsqrt(mean(x**2, -1) + eps) * weight`` for a 2-D FP32 ``x``."""
    if impl not in _RMSNORM_IMPLS:
        raise ValueError(f"unknown RMSNorm impl: {impl}")
    return _RMSNORM_IMPLS[impl](x.contiguous(), weight.contiguous(), eps)


def softmax(x: torch.Tensor, impl: str = "naive") -> torch.Tensor:
    """Softmax over the last dimension of a 2-D FP32 tensor."""
    if impl not in _SOFTMAX_IMPLS:
        raise ValueError(f"unknown softmax impl: {impl}")
    return _SOFTMAX_IMPLS[impl](x.contiguous())


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """Declared by the reference, not implemented there or here (raises)."""
    return _C.rope_forward(x.contiguous(), cos.contiguous(), sin.contiguous())


def attention_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor) -> torch.Tensor:
    """Declared by the reference, not implemented there or here (raises)."""
    return _C.attention_decode_forward(q.contiguous(), k_cache.contiguous(), v_cache.contiguous())


def adaptive_gemm(
    a: torch.Tensor,
    b: torch.Tensor,
    c: Optional[torch.Tensor] = None,
    bias: Optional[torch.Tensor] = None,
    alpha: float = 1.0,
    beta: float = 0.0,
    epilogue: str = "linear",
    kernel: str = "auto",
) -> torch.Tensor:
    """``act(alpha * A @ B + beta * C [+ bias])`` on the tensor cores (TF32).

    ``epilogue``: ``"linear"``, ``"relu"``, ``"gelu"`` (exact, erf-based), or
    ``"bias"``, ``"bias_relu"``, ``"bias_gelu"``, which add the length-N vector
    ``bias`` to every row before the activation (the reference declares the last
    four and refuses them at run time). ``kernel``: ``"auto"`` (first compatible
    registry entry), ``"cublas"`` (library baseline, linear only), ``"cublaslt"``
    (library baseline with the ReLU / bias epilogue fused by the library) or a registry
    name such as ``"fast"``, ``"fallback"``, ``"fast_relu"``, ``"pair"``. A
    forced kernel that cannot run the problem raises instead of falling back.
    """
    return _C.adaptive_gemm(
        a.contiguous(),
        b.contiguous(),
        c.contiguous() if c is not None else None,
        bias.contiguous() if bias is not None else None,
        alpha,
        beta,
        epilogue,
        kernel,
    )


# ---------------------------------------------------------------- serving operators
# What one serving step of a decoder needs next to the products and row operators above. The
# reference has none of them. They compute no gradient (inputs that require one are refused outside
# ``torch.no_grad()``, inputs with a forward-mode tangent always), run on the inputs' device and its current stream, read lengths and offsets on
# the device only, and may be captured in CUDA graphs.


def attention_prompt(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: Optional[torch.Tensor] = None,
    causal: bool = True,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """Attention over packed prompts; ``[rows, heads, dim]`` in and out.

    Sequence ``s`` owns the rows ``cu_seqlens_q[s]:cu_seqlens_q[s + 1]`` of ``q`` and
    ``cu_seqlens_k[s]:cu_seqlens_k[s + 1]`` of ``k`` and ``v`` (int32 offsets; those of
    ``q`` serve for both when ``cu_seqlens_k`` is left out). Query head ``h`` reads key
    head ``h // (heads / kv_heads)``. Of ``m`` keys, query ``i`` of ``n`` sees the first
    ``m - n + i + 1`` when ``causal`` (a chunk of a prompt, or a single token, at the end
    of its cached keys), else all. ``scale`` defaults to ``dim ** -0.5``.

    Rows that see no key, and rows in front of the first sequence or behind the last, are
    zero. Types: float32 (FP32 arithmetic), float16, bfloat16 (tensor cores: probabilities
    are rounded to the type before they meet ``v``, which about doubles the variance of the
    result's own rounding; maxima and sums are FP32).
    ``dim`` is a multiple of 8 up to 128. Strided views are taken as they are where their
    rows sit on 16-byte granules, and copied otherwise. Keys and values outside a sequence
    may hold anything; inside one, ``v`` must be finite.
    """
    return _C.attention_prompt(q, k, v, cu_seqlens_q, cu_seqlens_k, causal, scale)


def attention_shared_prefix(
    q: torch.Tensor,
    k_prefix: torch.Tensor,
    v_prefix: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    lengths: torch.Tensor,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """One decoding step of a batch whose requests share a prefix.

    ``q`` is ``[batch, heads, dim]``, one token per request. Request ``b`` sees all of
    ``k_prefix`` / ``v_prefix`` ``[prefix, kv_heads, dim]``, which are read once for up to
    256 rows (request, query head of a key head; 16 to 128 in float32), and the first ``lengths[b]`` rows of ``k_cache[b]`` / ``v_cache[b]``
    (``[batch, room, kv_heads, dim]``); the rows behind may hold anything. Types, head
    dimensions, strides and ``scale`` as for :func:`attention_prompt`. A request that
    sees no key gets zeros.
    """
    return _C.attention_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, lengths, scale)


def matvec_w4(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ W.T`` for 1 to 16 rows ``x`` ``[rows, k]`` and 4-bit weights.

    ``W[n, j] = (code[n, j] - zeros[n, j // group]) * scales[n, j // group]``, with the
    codes packed two to a byte in ``qweight`` (uint8 ``[n, k / 2]``, the even ``j`` in the
    low half), ``scales`` ``[n, k / group]`` in float32 or ``x``'s type, and ``zeros`` uint8
    of the same shape (0 .. 15; 8 throughout when left out). The group size is
    ``k / scales.shape[1]`` and a multiple of 32. ``x`` is float32, float16 or bfloat16;
    products are exact in the codes, sums are FP32.
    """
    return _C.matvec_w4(x, qweight, scales, zeros)


def process_logits(
    logits: torch.Tensor,
    prompt_tokens: Optional[torch.Tensor] = None,
    output_tokens: Optional[torch.Tensor] = None,
    repetition_penalty: Optional[torch.Tensor] = None,
    frequency_penalty: Optional[torch.Tensor] = None,
    presence_penalty: Optional[torch.Tensor] = None,
    bias_ids: Optional[torch.Tensor] = None,
    bias_values: Optional[torch.Tensor] = None,
    allowed: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Logits ``[rows, vocab]`` made ready for :func:`softmax`, as a new tensor.

    In this order, for row ``r`` and token ``t``: a token in the row's ``prompt_tokens`` or
    ``output_tokens`` is divided by ``repetition_penalty[r]`` where positive and multiplied
    by it otherwise; ``frequency_penalty[r]`` is subtracted once per occurrence in
    ``output_tokens`` and ``presence_penalty[r]`` once if there is any; each entry ``i``
    with ``bias_ids[r, i] == t`` adds ``bias_values[r, i]``; a token whose bit
    ``t % 32`` of word ``t // 32`` of ``allowed`` is clear becomes minus infinity, whatever
    it was. Token and bias ids are int32 ``[rows, length]``, and ids outside the vocabulary
    are padding; penalties and bias values are float32; ``allowed`` is int32
    ``[rows or 1, (vocab + 31) // 32]``. Arithmetic is FP32, rounded once.
    """
    return _C.process_logits(logits, prompt_tokens, output_tokens, repetition_penalty, frequency_penalty, presence_penalty,
                             bias_ids, bias_values, allowed)
