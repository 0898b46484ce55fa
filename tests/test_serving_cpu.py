"""The serving operators on a machine without a GPU: the names they are reached by, what the wrappers
hand on, and the refusals of the C ABI, which come before anything touches the device."""
import ctypes

import pytest
import torch

from conftest import load_serving_abi, LogitsProblem, MatvecProblem, PromptProblem, RowsView, SharedProblem
from test_python_api_cpu import stub_ops  # noqa: F401  (fixture)

OK, MISALIGNED, INVALID_PROBLEM, NOT_SUPPORTED, INVALID_ARGUMENT = 0, 1, 2, 3, 4
NAMES = ["attention_prompt", "attention_shared_prefix", "matvec_w4", "process_logits"]


@pytest.fixture(scope="module")
def lib():
    return load_serving_abi()


def test_names_are_reached_like_the_other_operators():
    import cuda_ai_kernels

    assert cuda_ai_kernels.SERVING_OPERATORS == NAMES
    for name in NAMES:
        assert callable(getattr(cuda_ai_kernels, name)) and name in dir(cuda_ai_kernels)


def test_wrappers_hand_the_callers_tensors_on(stub_ops, monkeypatch):  # noqa: F811
    ops, _ = stub_ops
    seen = {}
    for name in NAMES:
        monkeypatch.setattr(ops._C, name, lambda *args, _n=name: seen.setdefault(_n, args), raising=False)
    a, b, c, d, e, f = (torch.zeros(1) for _ in range(6))
    ops.attention_prompt(a, b, c, d)
    assert seen["attention_prompt"][0] is a and seen["attention_prompt"][4:] == (None, True, None)
    ops.attention_shared_prefix(a, b, c, d, e, f)
    assert seen["attention_shared_prefix"][5] is f and seen["attention_shared_prefix"][6] is None
    ops.matvec_w4(a, b, c)
    assert seen["matvec_w4"] == (a, b, c, None)
    ops.process_logits(a, allowed=b)
    assert seen["process_logits"] == (a, *[None] * 7, b)


def test_cpu_tensors_are_refused():
    from cuda_ai_kernels import _C

    x = torch.zeros(4, 2, 8)
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        _C.attention_prompt(x, x, x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        _C.attention_shared_prefix(x, x, x, x, x, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        _C.matvec_w4(x[0], x[0], x[0])
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        _C.process_logits(x[0])


# Addresses below are never dereferenced: every call is refused, or has nothing to do.
HERE = 1 << 20


def prompt(**changes):
    view = RowsView(HERE, 1024, 128)
    p = PromptProblem(dtype=2, heads=8, kv_heads=2, dim=128, sequences=1, q_rows=16, k_rows=16, q=view, k=view, v=view, out=HERE,
                      cu_q=HERE, cu_k=HERE, scale=0.1, causal=1)
    for name, value in changes.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("changes,status", [
    (dict(dtype=3), INVALID_ARGUMENT), (dict(dtype=-1), INVALID_ARGUMENT), (dict(heads=0), INVALID_ARGUMENT),
    (dict(heads=7), INVALID_ARGUMENT), (dict(kv_heads=0), INVALID_ARGUMENT), (dict(dim=0), INVALID_ARGUMENT),
    (dict(dim=36), NOT_SUPPORTED), (dict(dim=136), NOT_SUPPORTED), (dict(heads=258), NOT_SUPPORTED),
    (dict(scale=0.0), INVALID_ARGUMENT), (dict(scale=-1.0), INVALID_ARGUMENT), (dict(scale=float("nan")), INVALID_ARGUMENT),
    (dict(scale=float("inf")), INVALID_ARGUMENT), (dict(sequences=-1), INVALID_ARGUMENT), (dict(q_rows=-1), INVALID_ARGUMENT),
    (dict(q_rows=(1 << 30) + 1), INVALID_PROBLEM), (dict(k_rows=1 << 31), INVALID_PROBLEM),
    (dict(cu_q=None), INVALID_ARGUMENT), (dict(cu_k=None), INVALID_ARGUMENT), (dict(out=None), INVALID_ARGUMENT),
    (dict(out=HERE + 8), MISALIGNED), (dict(q=RowsView(None, 1024, 128)), INVALID_ARGUMENT),
    (dict(q=RowsView(HERE + 2, 1024, 128)), MISALIGNED), (dict(k=RowsView(HERE, 1020, 128)), MISALIGNED),
    (dict(v=RowsView(HERE, 1024, 4)), MISALIGNED), (dict(v=RowsView(HERE, -8, 8)), INVALID_ARGUMENT), (dict(q_rows=0), OK)])
def test_prompt_refusals(lib, changes, status):
    assert lib.b200_attention_prompt(ctypes.byref(prompt(**changes)), None, 0, None) == status


def test_prompt_split_needs_its_workspace(lib):
    p = prompt(q_rows=1, k_rows=100000)
    need = lib.b200_attention_prompt_workspace_bytes(ctypes.byref(p))
    assert lib.b200_attention_prompt_workspace_bytes(None) == 0
    if need:   # one SM is assumed where there is no device: one unit fills it
        assert lib.b200_attention_prompt(ctypes.byref(p), HERE, need - 1, None) == INVALID_ARGUMENT
        assert lib.b200_attention_prompt(ctypes.byref(p), HERE + 8, need, None) == MISALIGNED


def shared(**changes):
    view = RowsView(HERE, 1024, 128)
    p = SharedProblem(dtype=1, heads=8, kv_heads=8, dim=64, batch=3, prefix=100, room=50, q=view, k_prefix=view, v_prefix=view,
                      k_cache=view, v_cache=view, k_batch_stride=51200, v_batch_stride=51200, out=HERE, lengths=HERE, scale=0.1)
    for name, value in changes.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("changes,status", [
    (dict(dtype=9), INVALID_ARGUMENT), (dict(heads=12), INVALID_ARGUMENT), (dict(dim=65), NOT_SUPPORTED),
    (dict(batch=-1), INVALID_ARGUMENT), (dict(prefix=-1), INVALID_ARGUMENT), (dict(room=-1), INVALID_ARGUMENT),
    (dict(room=1 << 31), INVALID_PROBLEM), (dict(lengths=None), INVALID_ARGUMENT), (dict(out=HERE + 4), MISALIGNED),
    (dict(k_batch_stride=-8), INVALID_ARGUMENT), (dict(k_batch_stride=51204), MISALIGNED), (dict(v_batch_stride=1), MISALIGNED),
    (dict(k_cache=RowsView(None, 1024, 128)), INVALID_ARGUMENT), (dict(v_prefix=RowsView(HERE, 1024, 100)), MISALIGNED),
    (dict(scale=0.0), INVALID_ARGUMENT), (dict(batch=0), OK)])
def test_shared_refusals(lib, changes, status):
    assert lib.b200_attention_shared(ctypes.byref(shared(**changes)), None, 0, None) == status


def test_shared_always_needs_its_workspace(lib):
    need = lib.b200_attention_shared_workspace_bytes(ctypes.byref(shared()))
    assert need > 0
    assert lib.b200_attention_shared(ctypes.byref(shared()), None, 0, None) == INVALID_ARGUMENT
    assert lib.b200_attention_shared(ctypes.byref(shared()), HERE, need - 1, None) == INVALID_ARGUMENT
    assert lib.b200_attention_shared(ctypes.byref(shared()), HERE + 4, need, None) == MISALIGNED


@pytest.mark.parametrize("changes,status", [
    (dict(dtype=3), INVALID_ARGUMENT), (dict(scale_dtype=2), INVALID_ARGUMENT), (dict(rows=17), NOT_SUPPORTED),
    (dict(rows=-1), INVALID_ARGUMENT), (dict(k=0), INVALID_ARGUMENT), (dict(group=0), INVALID_ARGUMENT),
    (dict(group=48), INVALID_PROBLEM), (dict(k=96), INVALID_PROBLEM), (dict(x=None), INVALID_ARGUMENT),
    (dict(qweight=None), INVALID_ARGUMENT), (dict(scales=None), INVALID_ARGUMENT), (dict(y=None), INVALID_ARGUMENT),
    (dict(x=HERE + 2), MISALIGNED), (dict(qweight=HERE + 1), MISALIGNED), (dict(rows=0), OK), (dict(n=0), OK)])
def test_matvec_refusals(lib, changes, status):
    p = MatvecProblem(dtype=1, scale_dtype=0, rows=1, n=8, k=128, group=64, x=HERE, qweight=HERE, scales=HERE, zeros=None, y=HERE)
    for name, value in changes.items():
        setattr(p, name, value)
    assert lib.b200_matvec_w4(ctypes.byref(p), None) == status


@pytest.mark.parametrize("changes,status", [
    (dict(dtype=5), INVALID_ARGUMENT), (dict(rows=-1), INVALID_ARGUMENT), (dict(vocab=-1), INVALID_ARGUMENT),
    (dict(vocab=(1 << 30) + 1), INVALID_PROBLEM), (dict(prompt_length=-1), INVALID_ARGUMENT), (dict(bias_ids=HERE), INVALID_ARGUMENT),
    (dict(allowed=HERE, allowed_stride=3), INVALID_ARGUMENT), (dict(logits=None), INVALID_ARGUMENT), (dict(out=None), INVALID_ARGUMENT),
    (dict(logits=HERE + 4), MISALIGNED), (dict(out=HERE + 4), MISALIGNED), (dict(rows=0), OK), (dict(vocab=0), OK)])
def test_logits_refusals(lib, changes, status):
    p = LogitsProblem(dtype=0, rows=2, vocab=100, logits=HERE, out=HERE)
    for name, value in changes.items():
        setattr(p, name, value)
    assert lib.b200_process_logits(ctypes.byref(p), None) == status


def test_null_problems_are_refused(lib):
    assert lib.b200_attention_prompt(None, None, 0, None) == INVALID_ARGUMENT
    assert lib.b200_attention_shared(None, None, 0, None) == INVALID_ARGUMENT
    assert lib.b200_matvec_w4(None, None) == INVALID_ARGUMENT
    assert lib.b200_process_logits(None, None) == INVALID_ARGUMENT
