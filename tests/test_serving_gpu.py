"""The serving operators against their formulas in 64 bits.

Tolerances follow from the arithmetic. With u the rounding of the type (half a step relative to the
value), e = 2^-24 that of FP32, and A = sum_j p_j |v_j|:
  attention: a score of `dim` products is off by at most (dim + 4) e S, S = scale sum_d |q_d k_d|, and
  the subtraction of the maximum and the change to base 2 by a few e S more; a probability by the
  exponential of that and 8 e; sums over n keys by n e (2 e per term on the tensor cores, whose adder
  truncates). The denominator carries the same again. The tensor-core path rounds probabilities to the
  type, another u A, and the result is rounded once: u |out| (plus half the smallest subnormal).
  4-bit product: x and the codes are exact; K sums and one product per group: (k + 4) 2 e sum |x w|.
  logits: at most six FP32 operations on terms of size `size`: 6 e size, and one rounding.
"""
import math

import pytest
import torch

import cuda_ai_kernels as K
from conftest import assert_device_clean
from oracle import oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
E = 2.0 ** -24
NAN = float("nan")


def rounding(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def within(actual, expected, bound):
    actual = actual.double()
    assert actual.shape == expected.shape
    assert bool(torch.isfinite(actual).all())
    excess = (actual - expected).abs() - bound
    assert float(excess.max()) <= 0 if excess.numel() else True, f"off by {float((actual - expected).abs().max()):.3e}, too far by {float(excess.max()):.3e}"


def attention_bound(expected, absolute, score_size, dim, keys, dtype):
    u = rounding(dtype)
    wide = dtype == torch.float32
    term = 2 * (dim + 16) * E * score_size + 8 * E + (1 if wide else 2) * keys * E   # one of numerator and denominator
    return absolute * (2 * term + 16 * E + (0 if wide else u)) * 1.01 + u * expected.abs() + smallest(dtype)


# ------------------------------------------------------------------------------------- prompts

def offsets(lens):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist() if lens else [0], dtype=torch.int32, device="cuda")


def check_prompt(out, q, k, v, q_lens, k_lens, scale=None, causal=True, first_q=0, first_k=0):
    dim = q.shape[2]
    scale = float(torch.tensor(dim ** -0.5 if scale is None else scale, dtype=torch.float32))
    a, b = first_q, first_k
    for n, m in zip(q_lens, k_lens):
        if n:
            expected, absolute, size = oracle.attention_fp64(q[a:a + n], k[b:b + m], v[b:b + m], scale, causal)
            within(out[a:a + n], expected, attention_bound(expected, absolute, size, dim, m, q.dtype))
        a, b = a + n, b + m
    assert bool((out[a:] == 0).all()) and bool((out[:first_q] == 0).all())


def prompt_inputs(seed, q_lens, k_lens, heads, kv_heads, dim, dtype, tail=0):
    g = generator(seed)
    rows_q, rows_k = sum(q_lens) + tail, sum(k_lens)
    return (normal(g, rows_q, heads, dim, dtype=dtype, scale=1.5), normal(g, rows_k, kv_heads, dim, dtype=dtype),
            normal(g, rows_k, kv_heads, dim, dtype=dtype))


PROMPTS = [
    # queries, keys (None: the same), heads, kv_heads, dim, tail
    ([1], None, 1, 1, 8, 0),
    ([1], [1], 4, 4, 64, 3),
    ([2], [1], 2, 1, 64, 0),                             # the first query sees nothing
    ([300], [100], 4, 2, 64, 5),                         # most queries see nothing
    ([5, 0, 1, 0, 33], None, 8, 2, 64, 0),               # empty sequences
    ([0, 0], [7, 9], 4, 4, 64, 4),                       # keys without queries
    ([3, 4], [0, 6], 4, 1, 40, 0),                       # queries without keys
    ([63, 64, 65, 127, 128, 129], None, 4, 2, 64, 1),
    ([255, 256, 257], None, 3, 3, 128, 0),
    ([130], [1000], 8, 8, 128, 0),
    ([1, 1, 1], [129, 1, 640], 32, 4, 128, 2),           # single tokens at the end of their keys
    ([1], [5000], 8, 1, 128, 0),                         # split over the keys
    ([17, 3], [3000, 2500], 14, 2, 80, 0),
    ([40], [4096], 128, 1, 64, 0),                       # the widest group
    ([70], None, 127, 1, 72, 0),
    ([90], None, 65, 1, 32, 0),
    ([1100], None, 6, 2, 96, 0),
    ([400, 30], None, 5, 1, 120, 0),
    ([700], None, 16, 16, 16, 0),
    ([600, 500, 1], [900, 500, 1300], 24, 8, 112, 9),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", PROMPTS, ids=str)
def test_prompt(case, causal, dtype):
    q_lens, k_lens, heads, kv_heads, dim, tail = case
    k_lens = q_lens if k_lens is None else k_lens
    q, k, v = prompt_inputs(1, q_lens, k_lens, heads, kv_heads, dim, dtype, tail)
    out = K.attention_prompt(q, k, v, offsets(q_lens), offsets(k_lens), causal=causal)
    check_prompt(out, q, k, v, q_lens, k_lens, causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_many_sequences(dtype):
    lens = [(7 * i * i) % 61 for i in range(700)]
    q, k, v = prompt_inputs(2, lens, lens, 4, 2, 64, dtype, 3)
    check_prompt(K.attention_prompt(q, k, v, offsets(lens), offsets(lens)), q, k, v, lens, lens)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [1e-3, 0.3, 4.0])
def test_prompt_scale_and_growing_maxima(dtype, scale):
    # Scores that grow along the keys: the running maximum moves in every block.
    lens = [500]
    q, k, v = prompt_inputs(3, lens, lens, 2, 2, 64, dtype)
    k = (k.float() * torch.linspace(0.1, 3.0, 500, device="cuda")[:, None, None]).to(dtype)
    check_prompt(K.attention_prompt(q, k, v, offsets(lens), scale=scale), q, k, v, lens, lens, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens", [([5, 200, 66], [130, 200, 70]), ([2, 1], [3000, 2000])], ids=str)
def test_prompt_ignores_what_lies_outside_a_sequence(dtype, lens):
    # Rows before, between (a sequence without queries) and behind the sequences hold NaN and infinities.
    q_lens, k_lens = lens
    q_all, k_all = [11, *q_lens[:1], 0, *q_lens[1:], 6], [13, *k_lens[:1], 50, *k_lens[1:], 300]
    q, k, v = prompt_inputs(4, q_all, k_all, 8, 2, 128, dtype)
    cu_q, cu_k = offsets(q_all), offsets(k_all)
    for t, cu, rows in ((q, cu_q, len(q_all)), (k, cu_k, len(k_all)), (v, cu_k, len(k_all))):
        for s in (0, 2, rows - 1):
            t[int(cu[s]):int(cu[s + 1])] = NAN if s != 2 else float("inf")
    out = K.attention_prompt(q, k, v, cu_q[1:-1].contiguous(), cu_k[1:-1].contiguous())[int(cu_q[1]):]
    clean = [t.clone() for t in (q, k, v)]
    a = int(cu_q[1])
    for i, s in enumerate((1, 3) if len(q_lens) == 2 else (1, 3, 4)):
        n, m, b = q_all[s], k_all[s], int(cu_k[s])
        start = int(cu_q[s])
        expected, absolute, size = oracle.attention_fp64(clean[0][start:start + n], clean[1][b:b + m], clean[2][b:b + m],
                                                         float(torch.tensor(128 ** -0.5)), True)
        within(out[start - a:start - a + n], expected, attention_bound(expected, absolute, size, 128, m, dtype))
    assert bool((out[int(cu_q[-2]) - a:] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_masked_keys_may_hold_anything(dtype):
    # Keys (not values) that only later queries see: a NaN or an infinity there reaches those only.
    lens = [200]
    q, k, v = prompt_inputs(5, lens, lens, 4, 2, 64, dtype)
    expected = K.attention_prompt(q, k, v, offsets(lens))
    k[150] = NAN
    k[151] = float("inf")
    out = K.attention_prompt(q, k, v, offsets(lens))
    assert torch.equal(out[:150], expected[:150]) and bool(torch.isnan(out[150:]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_takes_strided_views(dtype):
    g = generator(6)
    lens = [100, 57]
    heads, kv_heads, dim = 6, 2, 64
    fused = normal(g, 157, heads + 2 * kv_heads, dim, dtype=dtype)                # one projection for all three
    q, k, v = fused.split([heads, kv_heads, kv_heads], dim=1)
    out = K.attention_prompt(q, k, v, offsets(lens))
    check_prompt(out, q, k, v, lens, lens)
    assert out.is_contiguous()
    head_major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(K.attention_prompt(*head_major, offsets(lens)), out)
    shifted = [torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (q, k, v)]
    assert torch.equal(K.attention_prompt(*shifted, offsets(lens)), out)          # off the granule: copied
    loose = [torch.empty(157, t.shape[1], dim + 1, dtype=dtype, device="cuda")[..., :dim].copy_(t) for t in (q, k, v)]
    assert torch.equal(K.attention_prompt(*loose, offsets(lens)), out)
    one = k[:, :1].expand(157, heads, dim)                                        # a broadcast key head
    assert torch.equal(K.attention_prompt(q, one, v[:, :1].expand(157, heads, dim), offsets(lens)),
                       K.attention_prompt(q, one.contiguous(), v[:, :1].expand(157, heads, dim).contiguous(), offsets(lens)))


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_without_rows(dtype):
    empty = torch.empty(0, 4, 64, dtype=dtype, device="cuda")
    some = torch.ones(5, 4, 64, dtype=dtype, device="cuda")
    assert K.attention_prompt(empty, some, some, offsets([0]), offsets([5])).shape == empty.shape
    assert bool((K.attention_prompt(some, empty, empty, offsets([5]), offsets([0])) == 0).all())
    assert bool((K.attention_prompt(some, some, some, offsets([])) == 0).all())


def test_prompt_offsets_outside_the_arrays_stay_inside():
    q, k, v = prompt_inputs(7, [64], [64], 4, 2, 64, torch.bfloat16)
    for bad in ([0, 1000], [-50, 64], [0, 40, 20, 64], [70, 90]):
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        assert K.attention_prompt(q, k, v, cu).shape == q.shape
    torch.cuda.synchronize()


def test_prompt_refusals():
    q = torch.zeros(4, 4, 64, device="cuda")
    cu = offsets([4])
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        K.attention_prompt(q.double(), q.double(), q.double(), cu)
    with pytest.raises(RuntimeError, match="same dtype"):
        K.attention_prompt(q, q.half(), q.half(), cu)
    with pytest.raises(RuntimeError, match="3-dimensional"):
        K.attention_prompt(q[0], q, q, cu)
    with pytest.raises(RuntimeError, match="one shape"):
        K.attention_prompt(q, q, q[:, :2], cu)
    with pytest.raises(RuntimeError, match="multiple of the number of key heads"):
        K.attention_prompt(q, q[:, :3], q[:, :3], cu)
    with pytest.raises(RuntimeError, match="multiple of 8 up to 128"):
        K.attention_prompt(q[..., :60], q[..., :60], q[..., :60], cu)
    with pytest.raises(RuntimeError, match="multiple of 8 up to 128"):
        K.attention_prompt(*[torch.zeros(4, 4, 256, device="cuda")] * 3, cu)
    with pytest.raises(RuntimeError, match="must be int32"):
        K.attention_prompt(q, q, q, cu.long())
    with pytest.raises(RuntimeError, match="one more offset"):
        K.attention_prompt(q, q, q, cu, offsets([2, 2]))
    with pytest.raises(RuntimeError, match="cu_seqlens_k is required"):
        K.attention_prompt(q, q[:2], q[:2], cu)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        K.attention_prompt(q, q, q, cu.cpu())
    for scale in (0.0, -1.0, NAN, float("inf")):
        with pytest.raises(RuntimeError, match="scale must be positive"):
            K.attention_prompt(q, q, q, cu, scale=scale)
    needs = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="requires a gradient"):
        K.attention_prompt(q, needs, q, cu)
    with torch.no_grad():
        K.attention_prompt(q, needs, q, cu)


# -------------------------------------------------------------------------------- shared prefix

def shared_inputs(seed, batch, prefix, room, heads, kv_heads, dim, dtype):
    g = generator(seed)
    return (normal(g, batch, heads, dim, dtype=dtype, scale=1.5), normal(g, prefix, kv_heads, dim, dtype=dtype),
            normal(g, prefix, kv_heads, dim, dtype=dtype), normal(g, batch, room, kv_heads, dim, dtype=dtype),
            normal(g, batch, room, kv_heads, dim, dtype=dtype))


def check_shared(out, q, k_prefix, v_prefix, k_cache, v_cache, lengths, scale=None):
    dim, room = q.shape[2], k_cache.shape[1]
    scale = float(torch.tensor(dim ** -0.5 if scale is None else scale, dtype=torch.float32))
    for b in range(q.shape[0]):
        length = min(max(int(lengths[b]), 0), room)
        k, v = torch.cat([k_prefix, k_cache[b, :length]]), torch.cat([v_prefix, v_cache[b, :length]])
        expected, absolute, size = oracle.attention_fp64(q[b:b + 1], k, v, scale, False)
        within(out[b:b + 1], expected, attention_bound(expected, absolute, size, dim, k.shape[0], q.dtype))


SHARED = [
    # batch, prefix, room, heads, kv_heads, dim, lengths (None: from empty to full)
    (1, 1, 1, 1, 1, 8, [0]),
    (1, 0, 5, 4, 2, 64, [3]),
    (2, 0, 4, 4, 2, 64, [0, 4]),              # one request sees nothing at all
    (3, 200, 0, 8, 2, 128, [0, 0, 0]),        # only the prefix
    (4, 1000, 64, 16, 4, 128, None),
    (5, 129, 300, 6, 2, 80, [0, 1, 300, 128, 129]),
    (33, 4097, 70, 14, 2, 64, None),
    (7, 64, 900, 8, 8, 96, None),
    (70, 300, 20, 32, 8, 128, None),          # more rows than one tile
    (300, 50, 9, 7, 1, 40, None),
    (2, 20000, 5000, 8, 1, 128, [5000, 17]),  # one long continuation beside a short one
    (3, 500, 130, 128, 1, 64, None),
    (4, 70, 9, 66, 1, 128, [-3, 9, 100, 1]),  # lengths outside the room are clamped
    (500, 0, 3, 2, 2, 64, None),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", SHARED, ids=str)
def test_shared_prefix(case, dtype):
    batch, prefix, room, heads, kv_heads, dim, lengths = case
    q, k_prefix, v_prefix, k_cache, v_cache = shared_inputs(8, batch, prefix, room, heads, kv_heads, dim, dtype)
    lengths = lengths or [(b * room) // max(1, batch - 1) for b in range(batch)]
    t = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for b in range(batch):   # behind a request's rows the cache holds anything
        k_cache[b, max(lengths[b], 0):] = NAN
        v_cache[b, max(lengths[b], 0):] = float("inf") if b % 2 else NAN
    out = K.attention_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, t)
    check_shared(out, q, k_prefix, v_prefix, k_cache, v_cache, lengths)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_prefix_is_the_prompt_operator_over_joined_keys(dtype):
    # The same tokens two ways: keys of prefix and continuation joined per request, one query each.
    batch, prefix, room, heads, kv_heads, dim = 6, 700, 40, 8, 2, 64
    q, k_prefix, v_prefix, k_cache, v_cache = shared_inputs(9, batch, prefix, room, heads, kv_heads, dim, dtype)
    lengths = torch.full((batch,), room, dtype=torch.int32, device="cuda")
    out = K.attention_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, lengths)
    k = torch.cat([torch.cat([k_prefix, k_cache[b]]) for b in range(batch)])
    v = torch.cat([torch.cat([v_prefix, v_cache[b]]) for b in range(batch)])
    joined = K.attention_prompt(q, k, v, offsets([1] * batch), offsets([prefix + room] * batch))
    torch.testing.assert_close(out.float(), joined.float(), atol=4 * rounding(dtype) if dtype != torch.float32 else 1e-5, rtol=0)


def test_shared_prefix_head_major_cache():
    dtype = torch.bfloat16
    q, k_prefix, v_prefix, k_cache, v_cache = shared_inputs(10, 5, 300, 200, 8, 2, 128, dtype)
    lengths = torch.tensor([200, 3, 0, 77, 128], dtype=torch.int32, device="cuda")
    out = K.attention_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, lengths)
    caches = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k_cache, v_cache)]
    prefixes = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k_prefix, v_prefix)]
    assert torch.equal(K.attention_shared_prefix(q, *prefixes, *caches, lengths), out)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_shared_prefix_offsets_beyond_32_bits(dtype):
    # A cache of more than 2^31 elements; the request that has rows is the last one.
    batch, room, heads, kv_heads, dim = 34, 65536, 8, 8, 128
    g = generator(11)
    q, k_prefix, v_prefix = normal(g, batch, heads, dim, dtype=dtype), normal(g, 20, kv_heads, dim, dtype=dtype), normal(g, 20, kv_heads, dim, dtype=dtype)
    k_cache = torch.empty(batch, room, kv_heads, dim, dtype=dtype, device="cuda")
    v_cache = torch.empty_like(k_cache)
    lengths = [0] * (batch - 1) + [room]
    assert k_cache.numel() > 2 ** 31
    k_cache[-1], v_cache[-1] = normal(g, room, kv_heads, dim, dtype=dtype), normal(g, room, kv_heads, dim, dtype=dtype)
    out = K.attention_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    check_shared(out, q, k_prefix, v_prefix, k_cache, v_cache, lengths)


def test_shared_prefix_refusals():
    q, k_prefix, v_prefix, k_cache, v_cache = shared_inputs(12, 2, 10, 4, 4, 2, 64, torch.float16)
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="kv_heads, dim"):
        K.attention_shared_prefix(q, k_prefix, v_prefix[:5], k_cache, v_cache, lengths)
    with pytest.raises(RuntimeError, match="batch, room, kv_heads, dim"):
        K.attention_shared_prefix(q, k_prefix, v_prefix, k_cache[:1], v_cache[:1], lengths)
    with pytest.raises(RuntimeError, match="one entry per request"):
        K.attention_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, lengths[:1])
    with pytest.raises(RuntimeError, match="int32"):
        K.attention_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, lengths.long())
    with pytest.raises(RuntimeError, match="same dtype"):
        K.attention_shared_prefix(q, k_prefix, v_prefix, k_cache.float(), v_cache.float(), lengths)
    with pytest.raises(RuntimeError, match="multiple of the number of key heads"):
        K.attention_shared_prefix(q[:, :3], k_prefix, v_prefix, k_cache, v_cache, lengths)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        K.attention_shared_prefix(q.clone().requires_grad_(), k_prefix, v_prefix, k_cache, v_cache, lengths)


# --------------------------------------------------------------------------------- 4-bit product

def w4_inputs(seed, rows, n, k, group, dtype, zeros, scale_dtype=None):
    g = generator(seed)
    x = normal(g, rows, k, dtype=dtype)
    qweight = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(n, k // group, generator=g, device="cuda") * 0.02 - 0.01).to(scale_dtype or dtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return x, qweight, scales, z


def check_w4(y, x, qweight, scales, zeros):
    expected, absolute = oracle.matvec_w4_fp64(x, qweight, scales, zeros)
    within(y, expected, absolute * (x.shape[1] + 4) * 2 * E + rounding(x.dtype) * expected.abs() + smallest(x.dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k,group,zeros", [
    (1, 1, 32, 32, False), (1, 16, 128, 128, True), (2, 17, 64, 64, True), (1, 1000, 1024, 64, True), (3, 33, 480, 96, True),
    (8, 100, 1152, 128, False), (9, 100, 1152, 32, True), (16, 257, 2048, 256, True), (5, 50, 4096, 4096, False), (1, 4099, 8192, 128, True),
    (7, 640, 11008, 128, False), (16, 31, 96, 32, False), (6, 15, 192, 192, True)])
def test_matvec_w4(dtype, rows, n, k, group, zeros):
    x, qweight, scales, z = w4_inputs(13, rows, n, k, group, dtype, zeros)
    check_w4(K.matvec_w4(x, qweight, scales, z), x, qweight, scales, z)
    check_w4(K.matvec_w4(x, qweight, scales.float(), z), x, qweight, scales, z)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k,group,zeros", [(6, 9472, 256, 128, True), (8, 9473, 384, 128, True), (16, 10001, 128, 128, False),
                                                  (5, 9999, 192, 64, True), (2, 9503, 1152, 128, False), (9, 9488, 96, 32, True),
                                                  # around the sizes from which a CTA has fewer warps
                                                  (1, 4736, 2176, 128, True), (8, 4737, 192, 64, False), (3, 2368, 160, 32, True),
                                                  (16, 2369, 384, 128, True), (7, 4725, 2048, 256, False), (12, 2300, 1088, 64, True)])
def test_matvec_w4_many_weight_rows(dtype, rows, n, k, group, zeros):
    x, qweight, scales, z = w4_inputs(19, rows, n, k, group, dtype, zeros)
    check_w4(K.matvec_w4(x, qweight, scales, z), x, qweight, scales, z)


@pytest.mark.parametrize("dtype", TYPES)
def test_matvec_w4_every_code_and_position(dtype):
    # Unit rows of x read single weights: every nibble has to come out where it was put in.
    k, n = 128, 16
    codes = (torch.arange(n, device="cuda")[:, None] * 7 + torch.arange(k, device="cuda")[None] * 3) % 16
    qweight = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8)
    scales = torch.ones(n, 1, dtype=dtype, device="cuda")
    for first in range(0, k, 16):
        x = torch.zeros(16, k, dtype=dtype, device="cuda")
        x[torch.arange(16), first + torch.arange(16)] = 1
        assert torch.equal(K.matvec_w4(x, qweight, scales).double(), (codes[:, first:first + 16].t() - 8).double())


def test_matvec_w4_fp32_is_as_exact_as_fp32():
    # Numbers whose low bits matter: BF16 or FP16 operands would lose them.
    x, qweight, scales, z = w4_inputs(14, 2, 64, 1024, 128, torch.float32, True)
    x = 1.0 + x * 2.0 ** -12
    check_w4(K.matvec_w4(x, qweight, scales, z), x, qweight, scales, z)
    big = torch.full((1, 128), 3.4e38, device="cuda")   # above BF16's largest number, and finite
    q = torch.full((1, 64), 0x88, dtype=torch.uint8, device="cuda")
    q[0, 0] = 0x89
    out = K.matvec_w4(big, q, torch.ones(1, 1, device="cuda"))
    assert float(out) == float(big[0, 0])


def test_matvec_w4_infinities_and_nan():
    x, qweight, scales, z = w4_inputs(15, 4, 64, 256, 64, torch.float32, False)
    qweight[:] = 0x99   # all weights positive
    scales = scales.abs() + 1e-3
    x[1, 17], x[2, 200] = float("inf"), NAN
    out = K.matvec_w4(x, qweight, scales)
    assert bool(torch.isfinite(out[[0, 3]]).all()) and bool((out[1] == float("inf")).all()) and bool(torch.isnan(out[2]).all())


def test_matvec_w4_views_and_empty_calls():
    x, qweight, scales, z = w4_inputs(16, 3, 40, 256, 64, torch.bfloat16, True)
    y = K.matvec_w4(x, qweight, scales, z)
    wide = torch.zeros(3, 512, dtype=torch.bfloat16, device="cuda")
    wide[:, ::2] = x
    assert torch.equal(K.matvec_w4(wide[:, ::2], qweight, scales, z), y)
    shifted = torch.empty(qweight.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view(qweight.shape).copy_(qweight)
    assert torch.equal(K.matvec_w4(x, shifted, scales, z), y)
    assert torch.equal(K.matvec_w4(x, qweight[8:], scales[8:], z[8:]), y[:, 8:])
    assert K.matvec_w4(x[:0], qweight, scales, z).shape == (0, 40) and K.matvec_w4(x, qweight[:0], scales[:0], z[:0]).shape == (3, 0)


def test_matvec_w4_refusals():
    x, qweight, scales, z = w4_inputs(17, 2, 8, 128, 64, torch.float16, True)
    with pytest.raises(RuntimeError, match="at most 16 rows"):
        K.matvec_w4(x[:1].expand(17, 128), qweight, scales)
    with pytest.raises(RuntimeError, match="k / 2"):
        K.matvec_w4(x[:, :64], qweight, scales)
    with pytest.raises(RuntimeError, match="multiple of 32"):
        K.matvec_w4(x, qweight, scales[:, :1].expand(8, 8))
    with pytest.raises(RuntimeError, match="multiple of 32"):
        K.matvec_w4(x, qweight, scales[:, :0])
    with pytest.raises(RuntimeError, match="uint8"):
        K.matvec_w4(x, qweight.to(torch.int8), scales)
    with pytest.raises(RuntimeError, match="scales must be float32 or"):
        K.matvec_w4(x, qweight, scales.bfloat16())
    with pytest.raises(RuntimeError, match="shape of scales"):
        K.matvec_w4(x, qweight, scales, z[:, :1])
    with pytest.raises(RuntimeError, match="requires a gradient"):
        K.matvec_w4(x.clone().requires_grad_(), qweight, scales)


# -------------------------------------------------------------------------------------- logits

def logits_inputs(seed, rows, vocab, prompt, output, bias, dtype):
    g = generator(seed)
    some = min(vocab, 40)   # few different tokens, so that histories repeat them; and padding on both sides
    tokens = lambda n: torch.randint(-2, some + 1, (rows, n), generator=g, device="cuda", dtype=torch.int32) * (vocab // some)  # noqa: E731
    uniform = lambda low, high, *shape: torch.rand(*shape, generator=g, device="cuda") * (high - low) + low  # noqa: E731
    words = (vocab + 31) // 32
    allowed = torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    return dict(logits=normal(g, rows, vocab, dtype=dtype, scale=3.0), prompt_tokens=tokens(prompt), output_tokens=tokens(output),
                repetition_penalty=uniform(0.7, 1.5, rows), frequency_penalty=uniform(-0.5, 0.5, rows),
                presence_penalty=uniform(-1.0, 1.0, rows), bias_ids=tokens(bias), bias_values=uniform(-5, 5, rows, bias), allowed=allowed)


def check_logits(out, inputs):
    expected, size = oracle.process_logits_fp64(**inputs)
    dtype = inputs["logits"].dtype
    out = out.cpu().double()
    gone = torch.isinf(expected)
    assert torch.equal(gone, torch.isinf(out)) and bool((out[gone] < 0).all())
    bound = 6 * E * size + rounding(dtype) * (expected.abs() + 6 * E * size) + smallest(dtype)
    excess = torch.where(gone, 0.0, (out - expected).abs() - bound)
    assert float(excess.max()) <= 0 if excess.numel() else True


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,prompt,output,bias", [
    (1, 1, 1, 1, 1), (3, 7, 5, 0, 2), (2, 1000, 50, 300, 9), (5, 1001, 0, 77, 0), (9, 4099, 700, 10, 33), (4, 20003, 100, 100, 5),
    (130, 517, 20, 30, 3), (700, 65, 9, 9, 1)])
def test_process_logits(dtype, rows, vocab, prompt, output, bias):
    inputs = logits_inputs(18, rows, vocab, prompt, output, bias, dtype)
    before = inputs["logits"].clone()
    check_logits(K.process_logits(**inputs), inputs)
    assert torch.equal(inputs["logits"], before)


@pytest.mark.parametrize("left", ["prompt_tokens", "output_tokens", "repetition_penalty", "frequency_penalty", "presence_penalty", "bias", "allowed"])
def test_process_logits_steps_stand_alone(left):
    inputs = logits_inputs(19, 3, 333, 20, 20, 4, torch.float32)
    without = {name: (None if name.startswith(left) else t) for name, t in inputs.items()}
    check_logits(K.process_logits(**without), without)
    history = ("prompt_tokens", "output_tokens")
    alone = {name: (t if name.startswith(left) or name == "logits" or (name in history and "penalty" in left) else None) for name, t in inputs.items()}
    check_logits(K.process_logits(**alone), alone)
    assert torch.equal(K.process_logits(inputs["logits"]), inputs["logits"])


def test_process_logits_masks():
    inputs = logits_inputs(20, 4, 100, 5, 5, 2, torch.bfloat16)
    inputs["allowed"][0] = 0                                   # nothing is left of the first row
    inputs["allowed"][1] = -1
    inputs["logits"][2, ::3], inputs["logits"][3, ::5] = NAN, float("inf")
    allowed = ((inputs["allowed"][..., None] >> torch.arange(32, device="cuda")) & 1).view(4, -1)[:, :100] != 0
    inputs["logits"][2] = torch.where(allowed[2], 1.0, inputs["logits"][2])   # NaN and infinities in masked places only
    inputs["logits"][3] = torch.where(allowed[3], 1.0, inputs["logits"][3])
    out = K.process_logits(**inputs)
    assert bool((out[0] == float("-inf")).all()) and not bool(torch.isnan(out).any())
    check_logits(out, inputs)
    one = dict(inputs, allowed=inputs["allowed"][2:3])         # one mask for all rows
    all_rows = dict(inputs, allowed=inputs["allowed"][2:3].expand(4, -1))
    a, b = K.process_logits(**one), K.process_logits(**all_rows)
    assert torch.equal(a.nan_to_num(), b.nan_to_num())
    lowest = torch.full((2, 50), torch.finfo(torch.float16).min, dtype=torch.float16, device="cuda")
    assert torch.equal(K.process_logits(lowest), lowest)


def test_process_logits_counts_long_repetitions():
    logits = torch.zeros(1, 64, device="cuda")
    tokens = torch.full((1, 100000), 5, dtype=torch.int32, device="cuda")
    out = K.process_logits(logits, output_tokens=tokens, frequency_penalty=torch.ones(1, device="cuda"))
    assert float(out[0, 5]) == -100000.0 and int((out != 0).sum()) == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [255, 257, 700])
def test_process_logits_long_bias_lists(dtype, bias):
    inputs = logits_inputs(31, 2, 3000, 30, 40000 if bias == 700 else 60, bias, dtype)   # many entries of few tokens; counters of both widths
    check_logits(K.process_logits(**inputs), inputs)


def test_process_logits_refusals():
    inputs = logits_inputs(21, 3, 100, 5, 5, 2, torch.float32)
    for change, match in ((dict(prompt_tokens=inputs["prompt_tokens"].long()), "int32"), (dict(output_tokens=inputs["output_tokens"][:2]), "one row per row"),
                          (dict(repetition_penalty=inputs["repetition_penalty"][:2]), "float32 \\[rows\\]"), (dict(bias_values=None), "go together"),
                          (dict(bias_values=inputs["bias_values"][:, :1]), "same shape"), (dict(allowed=inputs["allowed"][:, :2]), "allowed must be"),
                          (dict(allowed=inputs["allowed"][:2]), "allowed must be"), (dict(logits=inputs["logits"][0]), "rows, vocab"),
                          (dict(logits=inputs["logits"].double()), "float32, float16 or bfloat16"),
                          (dict(logits=inputs["logits"].clone().requires_grad_()), "requires a gradient"),
                          (dict(prompt_tokens=inputs["prompt_tokens"].cpu()), "CUDA tensor")):
        with pytest.raises(RuntimeError, match=match):
            K.process_logits(**{**inputs, **change})


# ------------------------------------------------------------------- streams, graphs, a whole step

def calls(dtype):
    q, k, v = prompt_inputs(22, [200, 61], [200, 61], 8, 2, 64, dtype)
    single = prompt_inputs(23, [1, 2], [3000, 1700], 8, 2, 64, dtype)
    shared = shared_inputs(24, 5, 900, 120, 8, 2, 128, dtype)
    lengths = torch.tensor([0, 120, 5, 64, 99], dtype=torch.int32, device="cuda")
    w4 = w4_inputs(25, 5, 500, 1024, 128, dtype, True)
    logits = logits_inputs(26, 5, 3001, 60, 60, 5, dtype)
    lens, one, many = offsets([200, 61]), offsets([1, 2]), offsets([3000, 1700])
    return [lambda: K.attention_prompt(q, k, v, lens), lambda: K.attention_prompt(*single, one, many),
            lambda: K.attention_shared_prefix(*shared, lengths), lambda: K.matvec_w4(*w4), lambda: K.process_logits(**logits)], (q, single[0], shared[0], w4[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_repeated_side_stream_and_captured_calls_agree(dtype, abi):
    functions, inputs = calls(dtype)
    first = [f() for f in functions]
    for f, y in zip(functions, first):
        assert all(torch.equal(f(), y) for _ in range(3))     # the same bits every time
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = [f() for f in functions]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graphs, outs = [], []
    for _ in range(2):                                          # two graphs of the same calls, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([f() for f in functions])
        graphs.append(graph)
    for t in inputs:
        t.mul_(0.5)
    expected = [f() for f in functions]
    for _ in range(2):
        for graph, out in zip(graphs, outs):
            for y in out:
                y.fill_(1)
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, expected))
    assert_device_clean(abi)


@pytest.mark.parametrize("dtype", TYPES)
def test_calls_on_two_streams_at_once(dtype):
    functions, _ = calls(dtype)
    expected = [f() for f in functions]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                results[i].append([f() for f in functions])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for per in results for ys in per for a, b in zip(ys, expected))


def test_lengths_are_read_when_the_graph_runs():
    q, k_prefix, v_prefix, k_cache, v_cache = shared_inputs(27, 4, 300, 200, 8, 2, 64, torch.bfloat16)
    lengths = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    args = (q, k_prefix, v_prefix, k_cache, v_cache, lengths)
    K.attention_shared_prefix(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.attention_shared_prefix(*args)
    for new in ([200, 0, 100, 7], [5, 6, 7, 8]):
        lengths.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        check_shared(out, *args[:5], new)


@pytest.mark.parametrize("dtype", TYPES)
def test_another_device(dtype):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two CUDA devices")
    q, k, v = (t.to("cuda:1") for t in prompt_inputs(28, [70], [70], 4, 2, 64, dtype))
    with torch.cuda.device(0):
        out = K.attention_prompt(q, k, v, offsets([70]).to("cuda:1"))
        assert torch.cuda.current_device() == 0 and out.device == q.device


@pytest.mark.parametrize("dtype", TYPES)
def test_a_serving_step(dtype):
    """Prompt attention fills a cache, a batch decodes over it, its output goes through a 4-bit projection,
    and the logits through penalties and mask into the package's softmax."""
    g = generator(29)
    prefix, batch, heads, kv_heads, dim, vocab = 333, 6, 8, 2, 64, 2050
    q, k, v = normal(g, prefix, heads, dim, dtype=dtype), normal(g, prefix, kv_heads, dim, dtype=dtype), normal(g, prefix, kv_heads, dim, dtype=dtype)
    hidden = K.attention_prompt(q, k, v, offsets([prefix]))
    check_prompt(hidden, q, k, v, [prefix], [prefix])
    k_cache, v_cache = (torch.full((batch, 16, kv_heads, dim), NAN, dtype=dtype, device="cuda") for _ in range(2))
    lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
    _, qweight, scales, zeros = w4_inputs(30, 1, vocab, heads * dim, 128, dtype, True)
    history = torch.full((batch, 4), -1, dtype=torch.int32, device="cuda")
    ones = torch.ones(batch, device="cuda")
    allowed = torch.full((1, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
    allowed[0, 0] = 0
    for step in range(4):
        k_cache[:, step], v_cache[:, step] = normal(g, batch, kv_heads, dim, dtype=dtype), normal(g, batch, kv_heads, dim, dtype=dtype)
        lengths += 1
        token = normal(g, batch, heads, dim, dtype=dtype)
        seen = K.attention_shared_prefix(token, k, v, k_cache, v_cache, lengths)
        check_shared(seen, token, k, v, k_cache, v_cache, [step + 1] * batch)
        logits = K.matvec_w4(seen.view(batch, -1), qweight, scales, zeros)
        check_w4(logits, seen.view(batch, -1), qweight, scales, zeros)
        settings = dict(logits=logits, output_tokens=history, repetition_penalty=1.2 * ones, frequency_penalty=0.3 * ones,
                        presence_penalty=0.1 * ones, allowed=allowed)
        ready = K.process_logits(**settings)
        check_logits(ready, settings)
        p = K.softmax(ready.float())
        torch.testing.assert_close(p, torch.softmax(ready.double(), -1).float(), atol=1e-5, rtol=1e-5)
        assert bool((p[:, :32] == 0).all())
        history[:, step] = p.argmax(-1).int()
