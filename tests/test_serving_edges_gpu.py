"""The serving operators where their callers come to the edges of what is documented: rows in front of the
first sequence, offsets that overlap, probabilities far below a row's largest, gradients of either mode.
Helpers and the derivation of the tolerances: test_serving_gpu.py."""
import ctypes

import pytest
import torch

import cuda_ai_kernels as K
from conftest import assert_device_clean, current_stream_ptr
from test_serving_gpu import TYPES, NAN, attention_bound, check_prompt, offsets, prompt_inputs, within

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
