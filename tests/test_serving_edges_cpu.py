"""What the C ABI of the serving operators accepts at its edges; no call here touches a device."""
import ctypes
import warnings
from types import SimpleNamespace

import pytest
import torch

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


@pytest.mark.parametrize("word,status,outcome", [(0, 0, None), (1 << 12, 4, RuntimeWarning), (1 << 8, 6, "never reached the barrier"),
                                                 (1 << 11, 6, "wait gave up"), (1 << 12 | 1 << 8, 6, "never reached the barrier"), (0, 5, "wait gave up")])
def test_a_gather_is_not_blamed_for_refused_offsets(monkeypatch, word, status, outcome):
    from cuda_ai_kernels import sharded

    def read(out, stream):
        ctypes.cast(out, ctypes.POINTER(ctypes.c_uint32))[0] = word
        return status

    monkeypatch.setattr(sharded, "_abi", lambda: SimpleNamespace(b200_device_status_read=read))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=0))
    gathered = sharded.GatheredOutput.__new__(sharded.GatheredOutput)
    gathered.full = torch.zeros(1)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        if outcome is None:
            gathered.check()
        elif outcome is RuntimeWarning:
            with pytest.warns(RuntimeWarning, match="overlap"):
                gathered.check()
        else:
            with pytest.raises(RuntimeError, match=outcome):
                gathered.check()
