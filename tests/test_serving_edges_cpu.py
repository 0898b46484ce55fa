"""What the C ABI of the serving operators accepts at its edges; no call here touches a device."""
import ctypes

import pytest

from test_serving_cpu import INVALID_ARGUMENT, INVALID_PROBLEM, lib, prompt, shared  # noqa: F401  (lib: fixture)


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("sequences,q_rows,k_rows,heads,kv_heads", [
    (2048, 2048, 2048 * 4096, 32, 8),             # single tokens, each at the end of its own keys
    (1024, 1024, 1024 * 16384, 32, 8),
    (8192, 8192 * 100, 8192 * 100, 32, 8),        # many short prompts
    (16, 16 * 65536, 16 * 65536, 32, 8),
    (1, 1 << 20, 1 << 20, 32, 8),                 # one long document
    (1, 1 << 22, 1 << 22, 64, 64),                # whose work passes 32 bits
    (1 << 20, 1 << 20, 1 << 24, 8, 1)], ids=str)
def test_prompt_calls_of_many_sequences_or_keys_are_accepted(lib, dtype, sequences, q_rows, k_rows, heads, kv_heads):  # noqa: F811
    p = prompt(dtype=dtype, sequences=sequences, q_rows=q_rows, k_rows=k_rows, heads=heads, kv_heads=kv_heads)
    need = lib.b200_attention_prompt_workspace_bytes(ctypes.byref(p))
    assert need > 0
    # The last check before anything is launched; a problem that is refused is refused earlier.
    assert lib.b200_attention_prompt(ctypes.byref(p), None, 0, None) == INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", [0, 2])
def test_work_without_end_is_refused(lib, dtype):  # noqa: F811
    most = 1 << 30
    p = prompt(dtype=dtype, q_rows=most, k_rows=most, heads=1 << 20, kv_heads=1 << 20)
    assert lib.b200_attention_prompt_workspace_bytes(ctypes.byref(p)) == 0
    assert lib.b200_attention_prompt(ctypes.byref(p), None, 0, None) == INVALID_PROBLEM
    p = shared(dtype=dtype, batch=most, prefix=most, room=most, heads=60000, kv_heads=60000)
    assert lib.b200_attention_shared_workspace_bytes(ctypes.byref(p)) == 0
    assert lib.b200_attention_shared(ctypes.byref(p), None, 0, None) == INVALID_PROBLEM
