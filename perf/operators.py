"""The serving operators as they are measured: their calls, their plain forms, and their definitions in 64 bits.

Four operators of one serving step of a decoder: attention over packed prompts, attention of a decoding batch
that shares a prefix, the matrix-vector product with 4-bit weights, and the processing of logits before the
softmax. `own` chooses between the calls of the package (true) and elementary torch operations (false).
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # Four very short requests admitted together (one of them a single token): latency of one call.
        {"name": "prompt_tiny", "op": "prompt", "dtype": "bf16", "q_lens": "1 17 33 5", "k_lens": "1 17 33 5",
         "heads": 8, "kv_heads": 2, "dim": 64, "tail": 0},
        # An ordinary admission batch: ragged prompts packed end to end, with a few spare rows behind them.
        {"name": "prompt_ragged", "op": "prompt", "dtype": "bf16",
         "q_lens": "771 64 1023 412 897 130 1 655 999 288 510 745 33 1024 601 350",
         "k_lens": "771 64 1023 412 897 130 1 655 999 288 510 745 33 1024 601 350",
         "heads": 32, "kv_heads": 8, "dim": 128, "tail": 11},
        # One long document.
        {"name": "prompt_long", "op": "prompt", "dtype": "bf16", "q_lens": "16384", "k_lens": "16384",
         "heads": 16, "kv_heads": 4, "dim": 128, "tail": 0},
        # Chunks of prompts whose first part is in the cache already: more keys than queries.
        {"name": "prompt_chunks", "op": "prompt", "dtype": "fp16", "q_lens": "257 512 96", "k_lens": "4353 2048 7001",
         "heads": 14, "kv_heads": 2, "dim": 80, "tail": 0},
        # Single precision end to end, as the package's matrix products have it.
        {"name": "prompt_fp32", "op": "prompt", "dtype": "fp32", "q_lens": "2048 1000", "k_lens": "2048 1000",
         "heads": 16, "kv_heads": 4, "dim": 64, "tail": 0},
        # A handful of samples of one short conversation.
        {"name": "shared_small", "op": "shared", "dtype": "bf16", "batch": 4, "prefix": 1000, "room": 64,
         "heads": 16, "kv_heads": 4, "dim": 128},
        # A full batch behind a long common context, each request with its own continuation.
        {"name": "shared_large", "op": "shared", "dtype": "bf16", "batch": 64, "prefix": 32768, "room": 2048,
         "heads": 32, "kv_heads": 8, "dim": 128},
        # Single precision cache, one query head per key head.
        {"name": "shared_fp32", "op": "shared", "dtype": "fp32", "batch": 13, "prefix": 4100, "room": 333,
         "heads": 8, "kv_heads": 8, "dim": 64},
        # One token through a small projection.
        {"name": "matvec_small", "op": "matvec", "dtype": "fp16", "rows": 1, "n": 1000, "k": 1024, "group": 64, "zeros": True},
        # One token through a large one: the stream over the weights.
        {"name": "matvec_large", "op": "matvec", "dtype": "bf16", "rows": 1, "n": 28672, "k": 8192, "group": 128, "zeros": False},
        # One row of logits with a short history.
        {"name": "logits_small", "op": "logits", "dtype": "fp32", "rows": 1, "vocab": 32000, "prompt": 300, "output": 100,
         "bias": 0, "grammar": False},
        # A large batch over a large vocabulary of odd size, everything switched on.
        {"name": "logits_large", "op": "logits", "dtype": "bf16", "rows": 256, "vocab": 100003, "prompt": 4000, "output": 2000,
         "bias": 64, "grammar": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["prompt", "shared", "matvec", "logits"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("prompt", "shared"):
        kv_heads, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8])
        heads = {"heads": kv_heads * group, "kv_heads": kv_heads, "dim": rng.choice([40, 64, 80, 96, 128])}
    if op == "prompt":
        count = _spread(rng, 1, 24)
        top = _spread(rng, 16, min(8192, 16384 / math.sqrt(count)))
        q_lens = [rng.randint(1, top) for _ in range(count)]
        k_lens = [n + rng.choice([0, 0, rng.randint(0, top)]) for n in q_lens]
        # The scores of the padded batch stay within the longest listed case's, and so does the work.
        room = 2.0e9 if dtype == "fp32" else 4.0e9
        while count * heads["heads"] * max(q_lens) * max(k_lens) > room:
            q_lens, k_lens = [(n + 1) // 2 for n in q_lens], [(n + 1) // 2 for n in k_lens]
        text = lambda lens: " ".join(str(n) for n in lens)  # noqa: E731
        return {"op": op, "dtype": dtype, "q_lens": text(q_lens), "k_lens": text(k_lens), "tail": rng.choice([0, 0, rng.randint(1, 40)]), **heads}
    if op == "shared":
        return {"op": op, "dtype": dtype, "batch": _spread(rng, 1, 64), "prefix": _spread(rng, 1, 24000),
                "room": _spread(rng, 1, 1500), **heads}
    if op == "matvec":
        group = rng.choice([32, 64, 128])
        return {"op": op, "dtype": dtype, "rows": _spread(rng, 1, 16), "n": _spread(rng, 100, 20000),
                "k": group * _spread(rng, 4, 10000 // group), "group": group, "zeros": rng.random() < 0.5}
    return {"op": op, "dtype": dtype, "rows": _spread(rng, 1, 128), "vocab": _spread(rng, 1000, 150000),
            "prompt": _spread(rng, 1, 6000), "output": _spread(rng, 1, 3000), "bias": rng.choice([0, _spread(rng, 1, 256)]),
            "grammar": rng.random() < 0.5}


# ----------------------------------------------------------------------------------------------- inputs

def _lens(case):
    """The queries and the keys of each sequence."""
    return [int(n) for n in case["q_lens"].split()], [int(n) for n in case["k_lens"].split()]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def uniform(low, high, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") * (high - low) + low

    state = {"case": case}
    if case["op"] == "prompt":
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        offsets = lambda lens: torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")  # noqa: E731
        q_lens, k_lens = _lens(case)
        state["cu_q"], state["cu_k"] = offsets(q_lens), offsets(k_lens)
        state["q"] = normal(sum(q_lens) + case["tail"], heads, dim, scale=1.5)
        state["k"], state["v"] = normal(sum(k_lens), kv_heads, dim), normal(sum(k_lens), kv_heads, dim)
        state["most_q"], state["most_k"] = max(q_lens), max(k_lens)
    elif case["op"] == "shared":
        heads, kv_heads, dim, batch, room = case["heads"], case["kv_heads"], case["dim"], case["batch"], case["room"]
        state["q"] = normal(batch, heads, dim, scale=1.5)
        state["k_prefix"], state["v_prefix"] = normal(case["prefix"], kv_heads, dim), normal(case["prefix"], kv_heads, dim)
        state["k_cache"], state["v_cache"] = normal(batch, room, kv_heads, dim), normal(batch, room, kv_heads, dim)
        state["lengths"] = torch.randint(0, room + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
    elif case["op"] == "matvec":
        rows, n, k, groups = case["rows"], case["n"], case["k"], case["k"] // case["group"]
        state["x"] = normal(rows, k)
        state["qweight"] = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        state["scales"] = uniform(0.005, 0.015, n, groups).to(dtype)
        state["zeros"] = torch.randint(4, 12, (n, groups), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    else:
        rows, vocab = case["rows"], case["vocab"]

        def tokens(length):  # frequent tokens have low numbers; the end of some histories is padding
            t = torch.exp(uniform(0.0, math.log(vocab), rows, length)).to(torch.int32) - 1
            live = torch.randint(0, length + 1, (rows, 1), generator=gen, device="cuda")
            return torch.where(torch.arange(length, device="cuda") < live, t.clamp(0, vocab - 1), -1)

        state["logits"] = normal(rows, vocab, scale=2.0)
        state["prompt_tokens"], state["output_tokens"] = tokens(case["prompt"]), tokens(case["output"])
        state["repetition"], state["frequency"] = uniform(1.0, 1.3, rows), uniform(0.0, 0.5, rows)
        state["presence"] = uniform(0.0, 0.5, rows)
        state["bias_ids"] = state["bias_values"] = state["allowed"] = None
        if case["bias"]:
            state["bias_ids"] = torch.randint(0, vocab, (rows, case["bias"]), generator=gen, device="cuda", dtype=torch.int32)
            state["bias_values"] = uniform(-5.0, 5.0, rows, case["bias"])
        if case["grammar"]:  # from rows in which nearly all is allowed to rows in which nearly nothing is
            words = (vocab + 31) // 32
            share = uniform(0.0, 1.0, rows, 1, 1) ** 2
            bits = (torch.rand(rows, words, 32, generator=gen, device="cuda") < share).to(torch.int64)
            packed = (bits << torch.arange(32, device="cuda")).sum(-1)
            state["allowed"] = torch.where(packed >= 2 ** 31, packed - 2 ** 32, packed).to(torch.int32)
    return state


def _visible_pairs(case):
    """Pairs of a query and a key that it sees: query i of n, with m keys, sees the first m - n + i + 1."""
    return sum(sum(max(0, min(m, m - n + i + 1)) for i in range(n)) for n, m in zip(*_lens(case)))


def work(case):
    size = BYTES[case["dtype"]]
    if case["op"] == "prompt":
        q_rows, k_rows = sum(_lens(case)[0]) + case["tail"], sum(_lens(case)[1])
        return {"bytes": size * case["dim"] * (2 * q_rows * case["heads"] + 2 * k_rows * case["kv_heads"]),
                "flops": 4 * case["dim"] * case["heads"] * _visible_pairs(case)}
    if case["op"] == "shared":
        # A continuation is half the room long on average.
        keys = case["prefix"] + case["batch"] * case["room"] / 2
        seen = case["batch"] * (case["prefix"] + case["room"] / 2)
        return {"bytes": size * case["dim"] * (2 * case["batch"] * case["heads"] + 2 * keys * case["kv_heads"]),
                "flops": 4 * case["dim"] * case["heads"] * seen}
    if case["op"] == "matvec":
        groups = case["k"] // case["group"]
        return {"bytes": case["n"] * (case["k"] // 2 + groups * (size + case["zeros"])) + size * case["rows"] * (case["k"] + case["n"]),
                "flops": 2 * case["rows"] * case["n"] * case["k"]}
    rows, vocab = case["rows"], case["vocab"]
    history = 4 * (case["prompt"] + case["output"] + 2 * case["bias"])
    return {"bytes": rows * (2 * size * vocab + history + (vocab + 31) // 32 * 4 * case["grammar"]), "flops": 6 * rows * vocab}


# --------------------------------------------------------------------------------- one pass of an operator

def run(state):
    if own:
        return _own(state)
    return {"prompt": _plain_prompt, "shared": _plain_shared, "matvec": _plain_matvec, "logits": _plain_logits}[state["case"]["op"]](state)


def _own(s):
    package = str(Path(__file__).resolve().parents[1] / "cuda-ai-infra-kernels_b200" / "python")
    if package not in sys.path:
        sys.path.insert(0, package)
    import cuda_ai_kernels as K

    op = s["case"]["op"]
    if op == "prompt":
        return K.attention_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])
    if op == "shared":
        return K.attention_shared_prefix(s["q"], s["k_prefix"], s["v_prefix"], s["k_cache"], s["v_cache"], s["lengths"])
    if op == "matvec":
        return K.matvec_w4(s["x"], s["qweight"], s["scales"], s["zeros"])
    return K.process_logits(s["logits"], prompt_tokens=s["prompt_tokens"], output_tokens=s["output_tokens"],
                            repetition_penalty=s["repetition"], frequency_penalty=s["frequency"], presence_penalty=s["presence"],
                            bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed=s["allowed"])


def _plain_prompt(s):
    """The packed rows are gathered into a padded batch, attended, and put back."""
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"].long(), s["cu_k"].long()
    heads, kv_heads, dim = q.shape[1], k.shape[1], q.shape[2]
    most_q, most_k, count = s["most_q"], s["most_k"], cu_q.numel() - 1
    i, j = torch.arange(most_q, device=q.device), torch.arange(most_k, device=q.device)
    n, m = cu_q.diff(), cu_k.diff()
    rows_q = (cu_q[:-1, None] + i).clamp(max=q.shape[0] - 1)
    rows_k = (cu_k[:-1, None] + j).clamp(max=k.shape[0] - 1)
    qb = q[rows_q].float().view(count, most_q, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    kb = k[rows_k].float().permute(0, 2, 1, 3)
    vb = v[rows_k].float().permute(0, 2, 1, 3)
    scores = torch.matmul(qb.reshape(count, kv_heads, -1, dim), kb.transpose(-1, -2)).view(count, kv_heads, -1, most_q, most_k)
    seen = j[None, None, :] < torch.minimum(m[:, None], m[:, None] - n[:, None] + i[None] + 1)[:, :, None]
    scores.mul_(1.0 / math.sqrt(dim)).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(count, kv_heads, -1, most_k), vb).view(count, kv_heads, -1, most_q, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(count, most_q, heads, dim)
    result = torch.zeros_like(q)
    live = i[None] < n[:, None]
    result[rows_q[live]] = out[live].to(q.dtype)
    return result


def _plain_shared(s):
    q, k_prefix, v_prefix, k_cache, v_cache, lengths = (s[x] for x in ("q", "k_prefix", "v_prefix", "k_cache", "v_cache", "lengths"))
    batch, heads, dim = q.shape
    prefix, kv_heads = k_prefix.shape[:2]
    room = k_cache.shape[1]
    qg = q.float().view(batch, kv_heads, heads // kv_heads, dim)
    before = torch.matmul(qg.permute(1, 0, 2, 3).reshape(kv_heads, -1, dim), k_prefix.float().permute(1, 2, 0))
    before = before.view(kv_heads, batch, -1, prefix).permute(1, 0, 2, 3)
    after = torch.matmul(qg, k_cache.float().permute(0, 2, 3, 1))
    after = after.masked_fill((torch.arange(room, device=q.device) >= lengths[:, None])[:, None, None], -math.inf)
    scores = torch.cat([before, after], -1) / math.sqrt(dim)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    total = weights.sum(-1, keepdim=True)
    ahead = weights[..., :prefix].permute(1, 0, 2, 3).reshape(kv_heads, -1, prefix)
    out = torch.matmul(ahead, v_prefix.float().permute(1, 0, 2)).view(kv_heads, batch, -1, dim).permute(1, 0, 2, 3)
    out = out + torch.matmul(weights[..., prefix:], v_cache.float().permute(0, 2, 1, 3))
    return (out / total).reshape(batch, heads, dim).to(q.dtype)


def _plain_matvec(s):
    x, qweight, scales, zeros = s["x"], s["qweight"], s["scales"], s["zeros"]
    n, groups = scales.shape
    q = torch.stack([qweight & 15, qweight >> 4], -1).view(n, groups, -1).float()
    q = q - (zeros.float()[..., None] if zeros is not None else 8.0)
    weight = (q * scales.float()[..., None]).view(n, -1)
    return torch.matmul(x.float(), weight.t()).to(x.dtype)


def _counts(tokens, rows, vocab):
    live = (tokens >= 0) & (tokens < vocab)
    counts = torch.zeros(rows, vocab, device=tokens.device)
    return counts.scatter_add_(1, torch.where(live, tokens, 0).long(), live.float())


def _plain_logits(s):
    rows, vocab = s["logits"].shape
    x = s["logits"].float()
    given, made = _counts(s["prompt_tokens"], rows, vocab), _counts(s["output_tokens"], rows, vocab)
    repeat = s["repetition"][:, None]
    x = torch.where((given + made) > 0, torch.where(x > 0, x / repeat, x * repeat), x)
    x = x - s["frequency"][:, None] * made - s["presence"][:, None] * (made > 0).float()
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias_values"])
    if s["allowed"] is not None:
        bits = (s["allowed"][..., None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(rows, -1)[:, :vocab] == 0, -math.inf)
    return x.to(s["logits"].dtype)


# ------------------------------------------------------------------------------- the definitions in 64 bits

def _attend(q, keys, values):
    """One query head's rows over the keys that it sees: softmax(q k^T / sqrt(d)) v."""
    weights = torch.softmax(q @ keys.T / math.sqrt(q.shape[-1]), dim=-1)
    return weights @ values


def exact(case, seed):
    s = {name: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for name, t in prepare(case, seed).items()}
    if case["op"] == "prompt":
        out, group, a, b = torch.zeros_like(s["q"]), case["heads"] // case["kv_heads"], 0, 0
        for n, m in zip(*_lens(case)):
            for h in range(case["heads"]):
                keys, values = s["k"][b:b + m, h // group], s["v"][b:b + m, h // group]
                for first in range(0, n, 4096):
                    last = min(first + 4096, n)
                    scores = s["q"][a + first:a + last, h] @ keys.T / math.sqrt(case["dim"])
                    scores += torch.full_like(scores, -math.inf).triu(m - n + first + 1)
                    out[a + first:a + last, h] = torch.softmax(scores, -1) @ values
            a, b = a + n, b + m
        return out
    if case["op"] == "shared":
        out, group = torch.empty_like(s["q"]), case["heads"] // case["kv_heads"]
        for b, length in enumerate(s["lengths"].tolist()):
            for g in range(case["kv_heads"]):
                keys = torch.cat([s["k_prefix"][:, g], s["k_cache"][b, :length, g]])
                values = torch.cat([s["v_prefix"][:, g], s["v_cache"][b, :length, g]])
                out[b, g * group:(g + 1) * group] = _attend(s["q"][b, g * group:(g + 1) * group], keys, values)
        return out
    if case["op"] == "matvec":
        codes = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = s["qweight"].remainder(16).double(), s["qweight"].div(16, rounding_mode="floor").double()
        per = lambda t: t.double().repeat_interleave(case["group"], dim=1)  # noqa: E731
        return s["x"] @ ((codes - (per(s["zeros"]) if case["zeros"] else 8)) * per(s["scales"])).T
    out = s["logits"].clone()
    for r in range(case["rows"]):
        row = out[r]
        made, times = torch.unique(s["output_tokens"][r][s["output_tokens"][r] >= 0].long(), return_counts=True)
        known = torch.unique(torch.cat([made, s["prompt_tokens"][r][s["prompt_tokens"][r] >= 0].long()]))
        row[known] = torch.where(row[known] > 0, row[known] / s["repetition"][r], row[known] * s["repetition"][r])
        row[made] -= s["frequency"][r] * times + s["presence"][r]
        if case["bias"]:
            row.index_add_(0, s["bias_ids"][r].long(), s["bias_values"][r])
        if case["grammar"]:
            token = torch.arange(case["vocab"], device="cuda")
            row[s["allowed"][r].long()[token // 32] >> (token % 32) & 1 == 0] = -math.inf
    return out
