"""Attention over voxel features and the rotary positions that go into it, as measured work.

``own`` false computes them in elementary torch operations in 32 bits (angles in 64); ``own`` true
makes the calls a user makes of ``sparseconv.ops``. ``exact`` is the definition in 64 bits, sample
by sample, its gradients from autograd (the plain form's come from the written-out formulas).

Sizes follow the benchmark's voxel workloads (indoor: 2.0 M voxels in 8 scenes, lidar: 883,771,
cube: 168,546) and the deeper stages that a network builds on them (84,000 voxels of 512 channels).
"""
import functools
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


@functools.cache
def _ops():
    """The framework's package (it lives one folder below the repository's root)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-conv_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from sparseconv.ops import attention, rotary
    return attention, rotary


# ---------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # one scene's bottleneck tokens, every one attending to all: latency
        attention_case("attention_small", 1, 512, 512, 16, 16, 64, "bfloat16"),
        # one pooling query a scene over all of its voxels, eight heads that share one key and value:
        # the single-token form, bound by reading keys and values
        attention_case("attention_pool_indoor", 8, 8, 2_000_000, 8, 1, 64, "float16"),
        # voxels in spatial windows of about 130: many short samples, a narrow head
        attention_case("attention_windows", 1301, 168_546, 168_546, 4, 4, 32, "float16"),
        # a deep stage's voxels, full attention within each of sixteen scenes
        attention_case("attention_deep", 16, 84_000, 84_000, 8, 8, 64, "bfloat16"),
        # its training step
        attention_case("attention_deep_train", 16, 84_000, 84_000, 8, 8, 64, "bfloat16", train=True),
        # voxels in serialised order, each seeing those before it, four query heads to a key head
        attention_case("attention_causal_train", 4, 20_000, 20_000, 16, 4, 128, "bfloat16", causal=True, train=True),
        # voxels attending to a few hundred conditioning tokens of their scene
        attention_case("attention_cross_train", 16, 168_546, 4_111, 8, 8, 64, "float16", cross=True, train=True),
        # full precision at a head size that is no multiple of eight
        attention_case("attention_fp32_train", 2, 6_001, 6_001, 4, 4, 35, "float32", train=True),
        # the next token of eight sequences at far positions, past the trained length
        rotary_case("rotary_token", 8, 16, 4, 128, 128, 1, 1 << 20, "bfloat16", "half", "yarn"),
        # queries and keys of a deep stage, three coordinates a voxel (30 of the 32 pairs turn)
        rotary_case("rotary_deep", 84_000, 8, 8, 64, 64, 3, 64, "bfloat16", "half", "none"),
        # a training step over eight indoor scenes
        rotary_case("rotary_indoor_train", 2_000_000, 2, 2, 32, 32, 3, 512, "float16", "interleaved", "linear", train=True),
        # a part of an odd-sized head, in full precision
        rotary_case("rotary_part_fp32_train", 168_546, 3, 1, 35, 24, 3, 128, "float32", "half", "ntk", train=True),
    ]


def attention_case(name, samples, queries, keys, heads, key_heads, size, dtype, causal=False, cross=False, train=False):
    """`queries` and `keys` are rows over all samples; `cross`: keys are other rows than the queries."""
    return {"name": name, "op": "attention", "samples": samples, "queries": queries, "keys": keys, "heads": heads,
            "key_heads": key_heads, "size": size, "dtype": dtype, "causal": causal,
            "cross": cross or queries != keys, "train": train}


def rotary_case(name, rows, heads, key_heads, size, rotary_dim, axes, extent, dtype, layout, scaling, train=False):
    return {"name": name, "op": "rotary", "rows": rows, "heads": heads, "key_heads": key_heads, "size": size,
            "rotary_dim": rotary_dim, "axes": axes, "extent": extent, "dtype": dtype, "layout": layout,
            "scaling": scaling, "train": train}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    """A case of the same ranges: samples of one row to tens of thousands, heads of 8 to 128."""
    train = rng.random() < 0.5
    dtype = rng.choice(["float16", "float16", "bfloat16", "bfloat16", "float32"])
    heads = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    key_heads = rng.choice([h for h in (1, 2, 3, 4, 6, 8, 12, 16) if heads % h == 0] + [heads] * 2)
    if rng.random() < 0.7:
        size = rng.choice([16, 32, 32, 64, 64, 64, 128, 128])
    else:
        size = rng.randint(1, 16) * 8 if rng.random() < 0.7 else _log_int(rng, 8, 128)
    if rng.random() < 0.4:
        most = min(2_000_000, int((1 << 29) / (heads + key_heads) / size / (2 if train else 1)))
        axes = rng.choice([1, 3, 3])
        if size < 2 * axes:
            size = 8
        dim = size // 2 * 2 if rng.random() < 0.6 else rng.randint(axes, size // 2) * 2
        case = rotary_case("", _log_int(rng, 1, most // 4 if dtype == "float32" else most // 2), heads, key_heads, size,
                           dim, axes, _log_int(rng, 16, 1 << (20 if axes == 1 else 10)), dtype,
                           rng.choice(["half", "interleaved"]), rng.choice(["none", "linear", "ntk", "yarn"]), train=train)
        del case["name"]
        return case
    # 32-bit and odd-sized heads have the CUDA cores only: less work, so that a draw stays under the largest case
    slow = dtype == "float32" or size % 8 != 0
    macs = 3e11 / (4 if train else 1) / (16 if slow else 1)
    kind = rng.choice(["self", "self", "causal", "few", "cross", "windows"])
    pairs = macs / (heads * size)                              # sum over samples of queries times keys
    if kind == "windows":
        length = _log_int(rng, 4, 600)
        samples = _log_int(rng, 2, max(2, min(2000, int(pairs / (2 * length * length)))))
        queries = keys = samples * length + rng.randint(0, samples)
    elif kind == "few":                                        # one to a few queries a sample, many keys
        samples = rng.randint(1, 16)
        queries = samples * _log_int(rng, 1, 16)
        keys = samples * _log_int(rng, 1, min(200_000, pairs / (2 * queries), 4e8 / (samples * key_heads * size)))
        keys += rng.randint(0, samples)
    elif kind == "cross":
        samples = rng.randint(1, 16)
        keys = samples * _log_int(rng, 1, 1000) + rng.randint(0, samples)
        queries = samples * _log_int(rng, 1, min(40_000, pairs * samples / (2 * keys) / samples, 1e8 / (samples * heads * size)))
        queries += rng.randint(0, samples)
    else:
        samples = rng.randint(1, 16)
        queries = keys = samples * _log_int(rng, 1, min(30_000, math.sqrt(pairs / (2 * samples)))) + rng.randint(0, samples)
    case = attention_case("", samples, queries, keys, heads, key_heads, size, dtype, causal=kind == "causal",
                          cross=kind in ("few", "cross"), train=train)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def _ends(rows, samples, rng):
    """First row of each sample and their end: of uneven size, as voxelised scenes are."""
    share = [0.5 + rng.random() for _ in range(samples)]
    total, at, ends = sum(share), 0.0, [0]
    for s in share:
        at += s
        ends.append(round(at / total * rows))
    ends[-1] = rows
    return ends


def _longest(ends):
    return max(b - a for a, b in zip(ends, ends[1:]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    H, K, D = case["heads"], case["key_heads"], case["size"]
    if case["op"] == "rotary":
        M = case["rows"]
        state = {"query": randn(M, H, D), "key": randn(M, K, D),
                 "positions": torch.randint(0, case["extent"], (M, case["axes"]), generator=g, device="cuda",
                                            dtype=torch.int32)}
        state["leaves"] = ["query", "key"]
        grads = {"grad_query": (M, H, D), "grad_key": (M, K, D)}
    else:
        ends = _ends(case["queries"], case["samples"], rng)
        key_ends = _ends(case["keys"], case["samples"], rng) if case["cross"] else ends
        # normalised queries and keys with a learned gain: scores of deviation 1.5 or so
        state = {"query": randn(case["queries"], H, D, scale=1.5), "key": randn(case["keys"], K, D),
                 "value": randn(case["keys"], K, D),
                 "offsets": torch.tensor(ends, device="cuda", dtype=torch.int32),
                 "key_offsets": torch.tensor(key_ends, device="cuda", dtype=torch.int32) if case["cross"] else None,
                 "longest": _longest(ends), "longest_key": _longest(key_ends)}
        state["leaves"] = ["query", "key", "value"]
        grads = {"grad": (case["queries"], H, D)}
    if case["train"]:
        for k in state["leaves"]:
            state[k].requires_grad_(True)
        for k, shape in grads.items():
            state[k] = randn(*shape)
    state["case"] = case
    return state


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return (_own_rotary if case["op"] == "rotary" else _own_attention)(state, case)
    with torch.no_grad():
        return (_plain_rotary if case["op"] == "rotary" else _plain_attention)(state, case)


def _own_attention(s, case):
    out = _ops()[0].sparse_attention(s["query"], s["key"], s["value"], s["offsets"], s["key_offsets"],
                                     causal=case["causal"])
    if not case["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, [s[k] for k in s["leaves"]], s["grad"])
    return {"out": out, **dict(zip(s["leaves"], grads))}


def _own_rotary(s, case):
    query, key = _ops()[1].sparse_rotary(s["query"], s["key"], s["positions"], layout=case["layout"],
                                         rotary_dim=case["rotary_dim"], scaling=case["scaling"],
                                         factor=_factor(case), trained_size=_trained(case))
    if not case["train"]:
        return {"rotated_query": query, "rotated_key": key}
    grads = torch.autograd.grad([query, key], [s["query"], s["key"]], [s["grad_query"], s["grad_key"]])
    return {"rotated_query": query, "rotated_key": key, "query": grads[0], "key": grads[1]}


def _padded_rows(offsets, longest):
    """Rows of each sample, [B, longest], and which of them there are."""
    rows = offsets[:-1, None].long() + torch.arange(longest, device=offsets.device)
    there = rows < offsets[1:, None]
    return torch.where(there, rows, 0), there


def _plain_attention(s, case):
    """Samples padded to the longest one, heads a few at a time where the scores would not fit."""
    dtype, H, K, D = s["query"].dtype, case["heads"], case["key_heads"], case["size"]
    rows, there = _padded_rows(s["offsets"], s["longest"])
    key_rows, key_there = rows, there
    if case["cross"]:
        key_rows, key_there = _padded_rows(s["key_offsets"], s["longest_key"])
    B, n, m, G, scale = rows.shape[0], rows.shape[1], key_rows.shape[1], H // K, D ** -0.5
    seen = key_there[:, None, None, None, :]
    if case["causal"]:                                         # the last query sees the last key
        lengths, key_lengths = there.sum(1), key_there.sum(1)
        last = torch.arange(n, device=rows.device) + (key_lengths - lengths)[:, None]
        seen = seen & (torch.arange(m, device=rows.device) <= last[..., None])[:, None, None]
    out = torch.zeros(case["queries"], H, D, device=rows.device)
    res = {"out": out}
    if case["train"]:
        res |= {"query": torch.zeros_like(out), "key": torch.zeros(case["keys"], K, D, device=rows.device),
                "value": torch.zeros(case["keys"], K, D, device=rows.device)}
    at_once = max(1, int(1.5e9 / (B * G * n * m)))
    for k0 in range(0, K, at_once):
        kv, qh = slice(k0, k0 + at_once), slice(k0 * G, (k0 + at_once) * G)

        def batched(t, index, heads, groups):                  # [B, key heads, groups, rows, D]
            t = t[:, heads].float()[index]
            return t.view(*index.shape, -1, groups, D).permute(0, 2, 3, 1, 4)

        def rows_of(t, present):                               # back to the rows that there are
            return t.permute(0, 3, 1, 2, 4).flatten(2, 3)[present]

        q = batched(s["query"], rows, qh, G)
        k = batched(s["key"], key_rows, kv, 1)
        v = batched(s["value"], key_rows, kv, 1)
        p = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -math.inf)
        top = p.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)          # a row that sees nothing
        p = p.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        p = p.div_(torch.where(total == 0.0, 1.0, total))
        out[rows[there], qh] = rows_of(p @ v, there)
        if not case["train"]:
            continue
        grad = batched(s["grad"], rows, qh, G) * there[:, None, None, :, None]
        res["value"][key_rows[key_there], kv] = rows_of((p.transpose(-1, -2) @ grad).sum(2, keepdim=True), key_there)
        d = grad @ v.transpose(-1, -2)
        d = d.sub_((d * p).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        res["query"][rows[there], qh] = rows_of(d @ k, there)
        res["key"][key_rows[key_there], kv] = rows_of((d.transpose(-1, -2) @ q).sum(2, keepdim=True), key_there)
    return {k: t.to(dtype) for k, t in res.items()}


def _factor(case):
    return 1.0 if case["scaling"] == "none" else 4.0


def _trained(case):
    return max(1, case["extent"] // 4) if case["scaling"] == "yarn" else None


def _frequencies(case):
    """Angle per unit of position of an axis's pairs, in 64 bits, and the amplitude of the rotation."""
    n, base, factor = case["rotary_dim"] // 2 // case["axes"], 10000.0, _factor(case)
    i = torch.arange(n, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk" and n > 1:
        base = base * factor ** (n / (n - 1))
    theta = base ** (-i / n)
    if case["scaling"] == "linear":
        return theta / factor, 1.0
    if case["scaling"] == "yarn":
        turns = _trained(case) * theta / (2.0 * math.pi)       # full turns within the trained size
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        return theta * keep + theta / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0
    return theta, 1.0


def _pair_columns(case):
    """Columns of each pair's two values."""
    half = case["rotary_dim"] // 2
    i = torch.arange(half // case["axes"] * case["axes"], device="cuda")
    return (i, i + half) if case["layout"] == "half" else (2 * i, 2 * i + 1)


def _plain_rotary(s, case):
    theta, amplitude = _frequencies(case)
    angle = (s["positions"].double()[:, :, None] * theta).flatten(1)[:, None]      # [M, 1, pairs]
    cos, sin = (angle.cos() * amplitude).float(), (angle.sin() * amplitude).float()
    a, b = _pair_columns(case)

    def turn(x, sin):
        y = x.float()
        first, second = y[..., a], y[..., b]
        if y.data_ptr() == x.data_ptr():
            y = y.clone()
        y[..., a], y[..., b] = first * cos - second * sin, first * sin + second * cos
        return y.to(x.dtype)

    res = {"rotated_query": turn(s["query"], sin), "rotated_key": turn(s["key"], sin)}
    if case["train"]:
        res |= {"query": turn(s["grad_query"], -sin), "key": turn(s["grad_key"], -sin)}
    return res


# ---------------------------------------------------------------------------------------
# What a pass cannot do without, and its definition in 64 bits
# ---------------------------------------------------------------------------------------
def work(case):
    e, H, K, D = DTYPES[case["dtype"]].itemsize, case["heads"], case["key_heads"], case["size"]
    passes = 2 if case["train"] else 1
    if case["op"] == "rotary":
        M = case["rows"]
        return {"bytes": passes * 2 * M * (H + K) * D * e + 4 * M * case["axes"],
                "flops": passes * 3.0 * M * (H + K) * case["rotary_dim"]}
    # samples of even size; causal ones see half
    pairs = case["queries"] * case["keys"] / case["samples"] * (0.5 if case["causal"] else 1.0)
    rows = 2 * case["queries"] * H + 2 * case["keys"] * K                  # query, out, key, value
    if case["train"]:                                                      # grad and the three gradients
        rows += 2 * case["queries"] * H + 2 * case["keys"] * K
    return {"bytes": rows * D * e + 4 * (case["samples"] + 1) * (2 if case["cross"] else 1),
            "flops": (14.0 if case["train"] else 4.0) * pairs * H * D}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s, case)
    if work(case)["flops"] > 8e12:
        return None
    H, K, D = case["heads"], case["key_heads"], case["size"]
    ends = s["offsets"].tolist()
    key_ends = s["key_offsets"].tolist() if case["cross"] else ends
    outs = {"out": torch.zeros(case["queries"], H, D, dtype=torch.float64, device="cuda")}
    if case["train"]:
        outs |= {k: torch.zeros(s[k].shape, dtype=torch.float64, device="cuda") for k in s["leaves"]}
    for b in range(case["samples"]):
        i, j = slice(ends[b], ends[b + 1]), slice(key_ends[b], key_ends[b + 1])
        n, m = i.stop - i.start, j.stop - j.start
        if n == 0 or m == 0:
            continue
        at_once = max(1, int(4e8 / (n * m * (H // K))))
        for k0 in range(0, K, at_once):
            kv, qh = slice(k0, k0 + at_once), slice(k0 * (H // K), (k0 + at_once) * (H // K))
            v = {"query": s["query"][i, qh], "key": s["key"][j, kv], "value": s["value"][j, kv]}
            v = {k: t.detach().double().requires_grad_(case["train"]) for k, t in v.items()}
            heads = {k: torch.repeat_interleave(t, H // K if k != "query" else 1, dim=1).transpose(0, 1) for k, t in v.items()}
            scores = torch.matmul(heads["query"], heads["key"].transpose(1, 2)) / math.sqrt(D)
            if case["causal"]:
                hidden = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
                scores = scores.masked_fill(hidden, -math.inf)
                weights = torch.softmax(scores, -1).masked_fill(hidden.all(1)[:, None], 0.0)
            else:
                weights = torch.softmax(scores, -1)
            out = torch.matmul(weights, heads["value"]).transpose(0, 1)
            outs["out"][i, qh] = out.detach()
            if case["train"]:
                got = torch.autograd.grad(out, list(v.values()), s["grad"][i, qh].double())
                outs["query"][i, qh], outs["key"][j, kv], outs["value"][j, kv] = got
    return outs


def _exact_rotary(s, case):
    """Pairs as complex numbers, multiplied by amplitude * exp(i angle)."""
    theta, amplitude = _frequencies(case)
    turn = torch.polar(torch.full((), amplitude, dtype=torch.float64, device="cuda").expand(s["positions"].shape[0], case["axes"], theta.numel()),
                       s["positions"].double().unsqueeze(-1) * theta).reshape(s["positions"].shape[0], 1, -1)
    count, half = turn.shape[-1], case["rotary_dim"] // 2

    def turned(x, turn):
        x = x.detach().double()
        head, rest = x[..., :2 * half], x[..., 2 * half:]
        if case["layout"] == "half":
            pairs = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous())
        else:
            pairs = torch.view_as_complex(head.reshape(*head.shape[:-1], half, 2).contiguous())
        pairs = torch.cat([pairs[..., :count] * turn, pairs[..., count:]], -1)
        parts = torch.view_as_real(pairs)
        parts = parts.transpose(-1, -2).flatten(-2) if case["layout"] == "half" else parts.flatten(-2)
        return torch.cat([parts, rest], -1)

    outs = {"rotated_query": turned(s["query"], turn), "rotated_key": turned(s["key"], turn)}
    if case["train"]:
        outs |= {"query": turned(s["grad_query"], turn.conj()), "key": turned(s["grad_key"], turn.conj())}
    return outs
