"""The serving operators where their callers come to the edges of what is documented: rows in front of the
first sequence, offsets that overlap, probabilities far below a row's largest, gradients of either mode.
Helpers and the derivation of the tolerances: test_serving_gpu.py."""
import ctypes
import math

import pytest
import torch

import cuda_ai_kernels as K
from conftest import assert_device_clean, current_stream_ptr
from test_serving_gpu import (TYPES, NAN, attention_bound, check_prompt, check_w4, logits_inputs, offsets, prompt_inputs, shared_inputs,
                              w4_inputs, within)

pytestmark = pytest.mark.gpu


def leave_nan_in_the_allocator(like):
    """The next tensor of this size starts out as NaN where nobody writes it."""
    torch.cuda.synchronize()
    torch.full_like(like, NAN)


# ------------------------------------------------------------------- rows in front of the first sequence

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("front_q,front_k,q_lens,k_lens,heads,kv_heads,dim", [
    (1, 0, [1], [1], 4, 4, 64),
    (5, 7, [33, 1], [33, 1], 8, 2, 64),
    (300, 3, [200], [200], 4, 2, 128),
    (70, 0, [2, 17], [3000, 2500], 14, 2, 80),       # keys split over CTAs
    (11, 200, [0, 40], [5, 0], 6, 6, 96),
    (9, 0, [], [], 4, 2, 64)], ids=str)
def test_rows_in_front_of_the_first_sequence_are_zero(front_q, front_k, q_lens, k_lens, heads, kv_heads, dim, causal, dtype, abi):
    tail = 3
    q, k, v = prompt_inputs(40, [front_q, *q_lens], [front_k, *k_lens], heads, kv_heads, dim, dtype, tail)
    q[:front_q], k[:front_k], v[:front_k] = NAN, NAN, NAN
    cu_q, cu_k = offsets([front_q, *q_lens])[1:], offsets([front_k, *k_lens])[1:]
    leave_nan_in_the_allocator(q)
    out = K.attention_prompt(q, k, v, cu_q, cu_k, causal=causal)
    check_prompt(out, q, k, v, q_lens, k_lens, causal=causal, first_q=front_q, first_k=front_k)
    assert_device_clean(abi)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_is_in_front_of_the_first_sequence(dtype):
    q, k, v = prompt_inputs(41, [150], [20], 8, 2, 64, dtype)
    for first in (150, 1000):    # all rows; and an offset behind the array
        cu = torch.tensor([first], dtype=torch.int32, device="cuda")
        leave_nan_in_the_allocator(q)
        assert bool((K.attention_prompt(q, k, v, cu, cu) == 0).all())


# ------------------------------------------------------------------------------ very many sequences

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sequences,keys,heads", [(20000, 511, 1), (3000, 4000, 4)])
def test_many_single_tokens_at_the_end_of_long_keys(sequences, keys, heads, dtype, abi):
    # Units of all sequences times blocks of all keys would be more than 2^31: each sees its own only.
    dim = 8
    q, k, v = prompt_inputs(42, [sequences], [sequences * keys], heads, 1, dim, dtype)
    cu_q = torch.arange(sequences + 1, dtype=torch.int32, device="cuda")
    out = K.attention_prompt(q, k, v, cu_q, cu_q * keys)
    scale = float(torch.tensor(dim ** -0.5, dtype=torch.float32))
    q64, k64, v64 = q.double(), k.double().view(sequences, keys, dim), v.double().view(sequences, keys, dim)
    p = torch.softmax(torch.bmm(q64, k64.transpose(1, 2)) * scale, dim=-1)
    size = (torch.bmm(q64.abs(), k64.abs().transpose(1, 2)) * scale).amax(-1, keepdim=True)
    within(out, torch.bmm(p, v64), attention_bound(torch.bmm(p, v64), torch.bmm(p, v64.abs()), size, dim, keys, dtype))
    assert_device_clean(abi)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q_rows,k_rows,heads,kv_heads", [(1 << 20, 1 << 20, 32, 32), (400000, 1 << 20, 96, 32)])
def test_arrays_large_enough_for_positions_of_64_bits(q_rows, k_rows, heads, kv_heads, causal, dtype, abi):
    # All queries over all keys would pass 32 bits; these sequences use a corner of the arrays.
    q_lens, k_lens, dim = [300, 0, 5, 1, 1100], [700, 9, 5, 3000, 1100], 8
    q, k, v = prompt_inputs(43, [q_rows], [k_rows], heads, kv_heads, dim, dtype)
    out = K.attention_prompt(q, k, v, offsets(q_lens), offsets(k_lens), causal=causal)
    check_prompt(out, q, k, v, q_lens, k_lens, causal=causal)
    assert torch.equal(out, K.attention_prompt(q, k, v, offsets(q_lens), offsets(k_lens), causal=causal))
    assert_device_clean(abi)


# ------------------------------------------------------------------------------- overlapping offsets

@pytest.mark.parametrize("dtype", TYPES)
def test_offsets_that_overlap_too_much_give_zeros_and_a_status(dtype, abi):
    # Twenty sequences that all claim all rows, with falling offsets between them.
    rows = 4096
    q, k, v = prompt_inputs(44, [rows], [rows], 4, 2, 64, dtype)
    cu = torch.tensor([0, rows] * 20, dtype=torch.int32, device="cuda")
    assert_device_clean(abi)
    leave_nan_in_the_allocator(q)
    out = K.attention_prompt(q, k, v, cu)
    word = ctypes.c_uint32(0)
    assert abi.b200_device_status_read(ctypes.byref(word), ctypes.c_void_p(current_stream_ptr())) == 4   # invalid argument
    assert word.value == 1 << 12
    assert bool((out == 0).all())
    check_prompt(K.attention_prompt(q, k, v, offsets([rows])), q, k, v, [rows], [rows])
    assert_device_clean(abi)


def test_falling_offsets_still_define_every_row(abi):
    q, k, v = prompt_inputs(45, [64], [64], 4, 2, 64, torch.bfloat16)
    for bad in ([0, 1000], [-50, 64], [0, 40, 20, 64], [70, 90], [50, 20], [30, 10, 64, 0]):
        leave_nan_in_the_allocator(q)
        assert bool(torch.isfinite(K.attention_prompt(q, k, v, torch.tensor(bad, dtype=torch.int32, device="cuda"))).all())
    assert_device_clean(abi)


# ------------------------------------------------------- probabilities far below a row's largest

def sink(rows, keys, gap, dtype, place, dim=64):
    """One key whose score is `gap` above all others', and its value zero where theirs are one."""
    q, k = torch.zeros(rows, 2, dim, device="cuda"), torch.zeros(keys, 2, dim, device="cuda")
    q[..., 0], k[place, :, 0] = 1.0, gap
    v = torch.ones(keys, 2, dim, device="cuda")
    v[place] = 0.0
    return q.to(dtype), k.to(dtype), v.to(dtype)


def check_sink(out, keys, gap, dtype):
    # Others weigh w = (keys - 1) 2^(-gap log2 e) against one. What test_serving_gpu.py derives holds while a
    # probability rounds relative to itself. FP16 holds it times 2^7 (at most 2^15), so that below 2^-21 of the
    # largest it rounds to multiples of 2^-24 instead: half of that, 2^-32 of the largest, for each key.
    w = (keys - 1) * math.exp(-gap)
    expected = torch.full(out.shape, w / (1 + w), dtype=torch.float64, device="cuda")
    far = keys * 2.0 ** -32 if dtype == torch.float16 else 0.0
    within(out, expected, attention_bound(expected, expected, torch.full_like(expected[..., :1], gap), out.shape[-1], keys, dtype) + far)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gap", [17.546875, 16.5, 12.0, 19.0])   # 2^-25.3, 2^-23.8, 2^-17.3, 2^-27.4; exact in the types but BF16's 17.5
@pytest.mark.parametrize("keys", [32768, 131072])
@pytest.mark.parametrize("place", [0, -1, 5000])
def test_many_keys_far_below_the_largest_still_count(keys, gap, place, dtype):
    gap = float(torch.tensor(gap, dtype=dtype))
    # One row, whose keys are dealt out over all CTAs, and so many that a CTA meets all keys of its rows.
    rows = 20000
    q, k, v = sink(rows, keys, gap, dtype, place)
    check_sink(K.attention_prompt(q[:1], k, v, offsets([1]), offsets([keys]), scale=1.0), keys, gap, dtype)
    check_sink(K.attention_prompt(q, k, v, offsets([rows]), offsets([keys]), causal=False, scale=1.0), keys, gap, dtype)
    # The same keys as a prefix and a request's own part.
    own = 16
    cut = keys - own
    cache = [t[cut:].expand(rows, own, 2, 64).contiguous() for t in (k, v)]
    lengths = torch.full((rows,), own, dtype=torch.int32, device="cuda")
    check_sink(K.attention_shared_prefix(q, k[:cut], v[:cut], *cache, lengths, scale=1.0), keys, gap, dtype)


def test_fp16_probabilities_stay_in_range_while_the_maximum_grows():
    # The maximum is followed lazily: a row's scores may be 2^8 above the base of its exponentials.
    keys = 640
    steps = torch.arange(keys, device="cuda") // 64                        # a block of scores after the other,
    for each in (5.0, 5.5, 5.6, 2.75):                                     # 2^7.2, 2^7.9, 2^8.1 and 2^4 apart
        q, k = torch.zeros(300, 2, 64, device="cuda").half(), torch.zeros(keys, 2, 64, device="cuda").half()
        q[..., 0] = 1.0
        k[:, :, 0] = (steps * each).half()[:, None]
        v = torch.full((keys, 2, 64), 60000.0, device="cuda").half()
        out = K.attention_prompt(q, k, v, offsets([300]), offsets([keys]), causal=False, scale=1.0)
        check_prompt(out, q, k, v, [300], [keys], scale=1.0, causal=False)


# ------------------------------------------------------------------------------ forward-mode tangents

def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as forward

    half = torch.float16
    q, k, v = prompt_inputs(46, [5], [5], 4, 2, 64, half)
    shared = shared_inputs(47, 2, 10, 4, 4, 2, 64, half)
    lengths, cu = torch.ones(2, dtype=torch.int32, device="cuda"), offsets([5])
    x, qweight, scales, _ = w4_inputs(48, 2, 8, 128, 64, half, False)
    logits = logits_inputs(49, 2, 100, 5, 5, 2, half)
    with forward.dual_level():
        dual = lambda t: forward.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda i=i: K.attention_prompt(*[dual(t) if j == i else t for j, t in enumerate((q, k, v))], cu) for i in range(3)]
        calls += [lambda i=i: K.attention_shared_prefix(*[dual(t) if j == i else t for j, t in enumerate(shared)], lengths) for i in range(5)]
        calls += [lambda: K.matvec_w4(dual(x), qweight, scales), lambda: K.matvec_w4(x, qweight, dual(scales))]
        calls += [lambda n=n: K.process_logits(**{**logits, n: dual(logits[n])})
                  for n in ("logits", "repetition_penalty", "frequency_penalty", "presence_penalty", "bias_values")]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward-mode tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode tangent"):
                call()
        expected = K.attention_prompt(q, k, v, cu)
        assert torch.equal(K.attention_prompt(forward.unpack_dual(dual(q)).primal, k, v, cu), expected)
        with forward._set_fwd_grad_enabled(False):
            assert torch.equal(K.attention_prompt(dual(q), k, v, cu), expected)


# ------------------------------------------------------------------------------- FP32 4-bit product

@pytest.mark.parametrize("bits", [0x7f800001, 0x7f80ffff, 0x7fbf0000, 0x7fc00000, 0xff800001 - (1 << 32), 0xffc00000 - (1 << 32)], ids=hex)
@pytest.mark.parametrize("rows", [1, 4, 16])
def test_matvec_w4_every_nan_stays_one(rows, bits):
    x, qweight, scales, _ = w4_inputs(50, rows, 40, 256, 64, torch.float32, False)
    qweight[:] = 0x99   # all weights one step above zero
    clean = K.matvec_w4(x, qweight, scales)
    x.view(torch.int32)[rows - 1, 77] = bits
    out = K.matvec_w4(x, qweight, scales)
    assert bool(torch.isnan(out[rows - 1]).all()) and torch.equal(out[:rows - 1], clean[:rows - 1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 6, 9, 16])
@pytest.mark.parametrize("ctas,height", [(1, 16), (2, 16), (2, 32)])
def test_matvec_w4_around_the_sizes_at_which_a_cta_changes(ctas, height, rows, dtype):
    # Rows of weights that make one or two CTAs per multiprocessor of this machine, one less and one more.
    here = ctas * height * torch.cuda.get_device_properties(0).multi_processor_count
    for n in (here - 1, here, here + 1):
        x, qweight, scales, z = w4_inputs(51, rows, n, 256, 128, dtype, True)
        check_w4(K.matvec_w4(x, qweight, scales, z), x, qweight, scales, z)


# ------------------------------------------------------------------------- counts that pass 32 bits

def test_more_sequences_or_heads_than_32_bits_count_are_refused():
    q, k, v = prompt_inputs(52, [5], [5], 1, 1, 64, torch.float16)
    many = torch.zeros(1, dtype=torch.int32, device="cuda").expand(2 ** 32 + 2)   # would read as one sequence
    with pytest.raises(RuntimeError, match="too many entries"):
        K.attention_prompt(q, k, v, many)
    with pytest.raises(RuntimeError, match="too many entries"):
        K.attention_prompt(q, k, v, offsets([5]), many)
    none, heads = q[:0], 2 ** 32 + 1                                              # would read as one head
    with pytest.raises(RuntimeError, match="too many heads"):
        K.attention_prompt(*[t[:0].expand(0, heads, 64) for t in (q, k, v)], offsets([]))
    assert K.attention_prompt(none, none, none, offsets([])).shape == none.shape
