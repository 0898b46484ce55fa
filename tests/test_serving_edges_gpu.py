"""The serving operators where their callers come to the edges of what is documented: rows in front of the
first sequence, offsets that overlap, probabilities far below a row's largest, gradients of either mode.
Helpers and the derivation of the tolerances: test_serving_gpu.py."""
import pytest
import torch

import cuda_ai_kernels as K
from conftest import assert_device_clean
from test_serving_gpu import TYPES, NAN, check_prompt, offsets, prompt_inputs

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
