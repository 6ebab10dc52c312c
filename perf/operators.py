"""The operators around a sparse convolution, as measured work: the pointwise linear layer with
its epilogue, the gated residual step with a norm on either side of it, and gradient clipping.

``own`` false computes them in elementary torch operations in 32 bits; ``own`` true makes the
calls a user makes of ``sparseconv.ops``. ``exact`` is the definition in 64 bits (its gradients
come from autograd, the plain form's from the written-out formulas).

Sizes follow the benchmark's voxel workloads (indoor: 2.0 M voxels of 64 channels in 8 scenes,
lidar: 883,771 of 16, cube: 168,546 of 32, wide: 1.34 M of 128 in 16 scenes) and the deeper,
narrower-in-voxels and wider-in-channels stages that a network builds on them.
"""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-5


@functools.cache
def _ops():
    """The framework's package (it lives one folder below the repository's root)."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-conv_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from sparseconv.ops import clip, linear, norm
    return linear, norm, clip


# ---------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # one conditioning vector per scene of a batch through its embedding layer: latency
        linear_case("linear_embed_8", 8, 256, 1024, "bfloat16", "silu"),
        # the widening half of a feed-forward pair over every voxel of eight indoor scenes
        linear_case("linear_indoor", 2_000_000, 64, 256, "bfloat16", "gelu"),
        # the narrowing half with the skip connection added, on lidar sweeps
        linear_case("linear_lidar_residual", 883_771, 64, 16, "float16", "none", residual=True),
        # a deep stage: few voxels, many channels; the tensor cores' rate counts
        linear_case("linear_deep", 84_000, 512, 2048, "bfloat16", "gelu"),
        # a training step of the pointwise layer on the wide scenes
        linear_case("linear_wide_train", 1_342_011, 128, 128, "bfloat16", "gelu", residual=True, train=True),
        # class scores of every voxel in full precision: an odd number of outputs
        linear_case("linear_head_fp32_train", 168_546, 32, 13, "float32", "none", train=True),
        # one scene's bottleneck tokens: latency of the gated residual step
        norm_case("norm_small", 512, 1024, 1, "bfloat16", "rms", "rms", gate="sample"),
        # eight indoor scenes, LayerNorm on both sides of the residual, a gate per scene
        norm_case("norm_indoor", 2_000_000, 64, 8, "bfloat16", "layer", "layer", gate="sample"),
        # its training step on the wide scenes, parameters in 32 bits
        norm_case("norm_wide_train", 1_342_011, 128, 16, "bfloat16", "layer", "layer", gate="sample", train=True),
        # a training step at an odd channel count (features with 3 coordinates appended)
        norm_case("norm_odd_train", 168_546, 35, 4, "float16", "none", "rms", gate="channel", train=True),
        # clipping a small network's gradients: many small tensors, latency
        clip_case("clip_small", 16, 3, 1, 1.0, "float32"),
        # clipping a large network's gradients
        clip_case("clip_large", 64, 5, 2, 1.0, "bfloat16"),
    ]


def linear_case(name, rows, cin, cout, dtype, activation, residual=False, train=False):
    return {"name": name, "op": "linear", "rows": rows, "cin": cin, "cout": cout, "dtype": dtype,
            "activation": activation, "residual": residual, "train": train}


def norm_case(name, rows, channels, samples, dtype, norm, next_norm, gate="none", train=False):
    return {"name": name, "op": "norm", "rows": rows, "channels": channels, "samples": samples, "dtype": dtype,
            "norm": norm, "next_norm": next_norm, "gate": gate, "train": train}


def clip_case(name, width, stages, blocks, max_norm, dtype):
    return {"name": name, "op": "clip", "width": width, "stages": stages, "blocks": blocks,
            "max_norm": max_norm, "dtype": dtype}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges: rows from one to two million, channels from three to 2048."""
    op = rng.choice(["linear", "linear", "norm", "norm", "clip"])
    train = rng.random() < 0.5
    if op == "clip":
        case = clip_case("", rng.choice([16, 24, 32, 48, 64]), rng.randint(1, 5), rng.randint(1, 2),
                         rng.choice([0.5, 1.0, 1e9]), rng.choice(list(DTYPES)))
        if case["dtype"] == "float32":
            case["stages"] = min(case["stages"], 4)
    elif op == "linear":
        dtype = rng.choice(["float32", "float16", "float16", "bfloat16", "bfloat16"])
        cin, cout = _log_int(rng, 3, 2048), _log_int(rng, 3, 2048)
        if rng.random() < 0.7:                    # most layers have channels in eights
            cin, cout = max(8, cin // 8 * 8), max(8, cout // 8 * 8)
        work = 80e9 / (3 if train else 1) / (8 if dtype == "float32" else 1)
        most = min(2_000_000, int(0.8e9 / DTYPES[dtype].itemsize / (3 if train else 1) / (cin + cout)),
                   int(work / (cin * cout)))
        case = linear_case("", _log_int(rng, 1, max(2, most)), cin, cout, dtype,
                           rng.choice(["none", "relu", "gelu", "silu"]), residual=rng.random() < 0.5, train=train)
    else:
        channels = _log_int(rng, 3, 2048)
        if rng.random() < 0.7:
            channels = max(8, channels // 8 * 8)
        dtype = rng.choice(list(DTYPES))
        most = min(2_000_000, int(128e6 / channels / (2 if dtype == "float32" else 1)))
        case = norm_case("", _log_int(rng, 1, most), channels, rng.randint(1, 16), dtype,
                         rng.choice(["none", "layer", "rms"]), rng.choice(["layer", "rms"]),
                         rng.choice(["none", "channel", "sample"]), train=train)
    del case["name"]
    return case


def _clip_shapes(case):
    """Gradient shapes of a sparse network: per stage and block a 3x3x3 convolution, a norm and
    a feed-forward pair; a class head last."""
    shapes = []
    for s in range(case["stages"]):
        c = case["width"] << s
        for _ in range(case["blocks"]):
            shapes += [(c, 3, 3, 3, c), (c,), (c,), (c,), (4 * c, c), (4 * c,), (c, 4 * c), (c,)]
    return shapes + [(13, case["width"]), (13,)]


# ---------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, offset=0.0, dtype=dtype):
        t = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
        return (t * scale + offset).to(dtype)

    if case["op"] == "linear":
        M, Ci, Co = case["rows"], case["cin"], case["cout"]
        state = {"feats": randn(M, Ci), "weight": randn(Co, Ci, scale=Ci ** -0.5), "bias": randn(Co, scale=0.1),
                 "residual": randn(M, Co) if case["residual"] else None,
                 "grad": randn(M, Co) if case["train"] else None}
        leaves = ("feats", "weight", "bias", "residual")
    elif case["op"] == "norm":
        M, C, B = case["rows"], case["channels"], case["samples"]
        # scenes of uneven size, as voxelised scenes are
        share = torch.rand(B, generator=g, device="cuda", dtype=torch.float64) + 0.25
        ends = (share.cumsum(0) / share.sum() * M).round().to(torch.int32)
        ends[-1] = M
        state = {"feats": randn(M, C, scale=2.0, offset=0.5), "residual": randn(M, C),
                 "offsets": torch.cat([torch.zeros_like(ends[:1]), ends]),
                 "gate": None, "weight": None, "bias": None, "next_bias": None,
                 "next_weight": randn(C, scale=0.2, offset=1.0, dtype=torch.float32)}
        if case["gate"] != "none":
            state["gate"] = randn(*((B, C) if case["gate"] == "sample" else (C,)), scale=0.5, dtype=torch.float32)
        if case["norm"] != "none":
            state["weight"] = randn(C, scale=0.2, offset=1.0, dtype=torch.float32)
        if case["norm"] == "layer":
            state["bias"] = randn(C, scale=0.1, dtype=torch.float32)
        if case["next_norm"] == "layer":
            state["next_bias"] = randn(C, scale=0.1, dtype=torch.float32)
        if case["train"]:
            state["grad_hidden"], state["grad_normed"] = randn(M, C), randn(M, C)
        leaves = ("feats", "residual", "gate", "weight", "bias", "next_weight", "next_bias")
    else:
        shapes = _clip_shapes(case)
        sizes = [math.prod(s) for s in shapes]
        # a network's gradients differ in size from layer to layer
        grads = [randn(*s, scale=10.0 ** -(1 + i % 3)) for i, s in enumerate(shapes)]
        flat = torch.zeros(sum(sizes), device="cuda", dtype=dtype)
        out = [v.view(s) for v, s in zip(flat.split(sizes), shapes)]
        return {"case": case, "grads": grads, "flat": flat, "out": out}
    if case["train"]:
        for k in leaves:
            if state[k] is not None:
                state[k].requires_grad_(True)
    state["case"] = case
    state["leaves"] = [k for k in leaves if state[k] is not None]
    return state


# ---------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    with torch.no_grad():
        return {"linear": _plain_linear, "norm": _plain_norm, "clip": _plain_clip}[case["op"]](state, case)


def _run_own(s, case):
    linear, norm, clip = _ops()
    if case["op"] == "linear":
        out = linear.sparse_linear(s["feats"], s["weight"], s["bias"], residual=s["residual"],
                                   activation=case["activation"])
        if not case["train"]:
            return {"out": out}
        grads = torch.autograd.grad(out, [s[k] for k in s["leaves"]], s["grad"])
        return {"out": out, **dict(zip(s["leaves"], grads))}
    if case["op"] == "norm":
        hidden, normed = norm.sparse_residual_norm(
            s["feats"], s["residual"], gate=s["gate"], batch_offsets=s["offsets"],
            norm=case["norm"], weight=s["weight"], bias=s["bias"],
            next_norm=case["next_norm"], next_weight=s["next_weight"], next_bias=s["next_bias"], eps=EPS)
        if not case["train"]:
            return {"hidden": hidden, "normed": normed}
        grads = torch.autograd.grad([hidden, normed], [s[k] for k in s["leaves"]],
                                    [s["grad_hidden"], s["grad_normed"]])
        return {"hidden": hidden, "normed": normed, **dict(zip(s["leaves"], grads))}
    total = clip.clip_gradients(s["grads"], case["max_norm"], out=s["out"])
    return {"total_norm": total, "clipped": s["flat"]}


def _act(z, name):
    """(value, derivative) of the activation at z."""
    if name == "relu":
        pos = (z > 0).to(z.dtype)
        return z * pos, pos
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    if name == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig))
    return z, torch.ones_like(z)


def _plain_linear(s, case):
    dtype = s["feats"].dtype
    x, w = s["feats"].float(), s["weight"].float()
    value, slope = _act(x @ w.t() + s["bias"].float(), case["activation"])
    out = value if s["residual"] is None else value + s["residual"].float()
    if not case["train"]:
        return {"out": out.to(dtype)}
    dz = s["grad"].float() * slope
    res = {"out": out.to(dtype), "feats": (dz @ w).to(dtype), "weight": (dz.t() @ x).to(dtype),
           "bias": dz.sum(0).to(dtype)}
    if s["residual"] is not None:
        res["residual"] = s["grad"].clone()
    return res


def _normalise(x, kind):
    """(normalised rows, 1 / deviation) of x, for the kinds with statistics."""
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
    return x * rstd, rstd


def _normalise_back(d, xhat, rstd, kind):
    """Gradient at the rows from the gradient at the normalised rows."""
    d = d - xhat * (d * xhat).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if kind == "layer" else 0.0)
    return d * rstd


def _plain_norm(s, case):
    dtype = s["feats"].dtype
    x, r = s["feats"].float(), s["residual"].float()
    row = torch.arange(x.shape[0], device=x.device)
    sample = (row[:, None] >= s["offsets"][None, 1:]).sum(1)
    u, xhat, rstd = x, None, None
    if case["norm"] != "none":
        xhat, rstd = _normalise(x, case["norm"])
        u = xhat * s["weight"]
        if s["bias"] is not None:
            u = u + s["bias"]
    gate = torch.ones_like(x[:1]) if s["gate"] is None else s["gate"][sample] if case["gate"] == "sample" else s["gate"]
    h = r + gate * u
    hhat, hrstd = _normalise(h, case["next_norm"])
    y = hhat * s["next_weight"]
    if s["next_bias"] is not None:
        y = y + s["next_bias"]
    if not case["train"]:
        return {"hidden": h.to(dtype), "normed": y.to(dtype)}
    dh, dy = s["grad_hidden"].float(), s["grad_normed"].float()
    res = {"hidden": h.to(dtype), "normed": y.to(dtype), "next_weight": (dy * hhat).sum(0)}
    if s["next_bias"] is not None:
        res["next_bias"] = dy.sum(0)
    dh = dh + _normalise_back(dy * s["next_weight"], hhat, hrstd, case["next_norm"])
    res["residual"] = dh.to(dtype)
    if case["gate"] == "channel":
        res["gate"] = (dh * u).sum(0)
    elif case["gate"] == "sample":
        # long sums in an order that changes: in 64 bits
        res["gate"] = torch.zeros_like(s["gate"], dtype=torch.float64).index_add_(0, sample, (dh * u).double()).float()
    du = dh * gate
    if case["norm"] != "none":
        res["weight"] = (du * xhat).sum(0)
        if s["bias"] is not None:
            res["bias"] = du.sum(0)
        du = _normalise_back(du * s["weight"], xhat, rstd, case["norm"])
    res["feats"] = du.to(dtype)
    return res


def _plain_clip(s, case):
    flat = torch.cat([g.reshape(-1) for g in s["grads"]]).float()
    total = (flat * flat).sum(dtype=torch.float64).sqrt()
    coef = torch.clamp(case["max_norm"] / (total + 1e-6), max=1.0).float()
    s["flat"].copy_(flat * coef)
    return {"total_norm": total.float(), "clipped": s["flat"]}


# ---------------------------------------------------------------------------------------
# What a pass cannot do without, and its definition in 64 bits
# ---------------------------------------------------------------------------------------
def work(case):
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] == "linear":
        M, Ci, Co = case["rows"], case["cin"], case["cout"]
        res = M * Co if case["residual"] else 0
        total = M * Ci + Co * Ci + Co + M * Co + res          # feats, weight, bias, out, residual
        flops = 2.0 * M * Ci * Co
        if case["train"]:                                     # + grad; feats', weight', bias', residual'
            total += M * Co + M * Ci + Co * Ci + Co + res
            flops *= 3
        return {"bytes": total * e, "flops": flops}
    if case["op"] == "norm":
        M, C, B = case["rows"], case["channels"], case["samples"]
        params = {"none": 0, "rms": 1, "layer": 2}
        small = 4 * C * (params[case["norm"]] + params[case["next_norm"]] +
                         {"none": 0, "channel": 1, "sample": B}[case["gate"]])
        full = 8 if case["train"] else 4
        return {"bytes": full * M * C * e + small * (2 if case["train"] else 1) + 4 * (B + 1),
                "flops": (50.0 if case["train"] else 20.0) * M * C}
    n = sum(math.prod(s) for s in _clip_shapes(case))
    return {"bytes": 2 * n * e + 4, "flops": 3.0 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        sq = sum(torch.linalg.vector_norm(g.double()) ** 2 for g in s["grads"])
        total = sq.sqrt()
        coef = min(1.0, case["max_norm"] / (total.item() + 1e-6))
        return {"total_norm": total, "clipped": torch.cat([(g.double() * coef).flatten() for g in s["grads"]])}
    if case["op"] == "linear":
        if case["rows"] * case["cin"] * case["cout"] > 5e11:
            return None
        v = {k: s[k].detach().double().requires_grad_(case["train"]) for k in s["leaves"]}
        f = torch.nn.functional
        act = {"none": lambda z: z, "relu": f.relu, "gelu": f.gelu, "silu": f.silu}[case["activation"]]
        out = act(f.linear(v["feats"], v["weight"], v["bias"]))
        if "residual" in v:
            out = out + v["residual"]
        outs, grads = {"out": out}, [s["grad"]]
    else:
        v = {k: s[k].detach().double().requires_grad_(case["train"]) for k in s["leaves"]}
        counts = (s["offsets"][1:] - s["offsets"][:-1]).long()

        def norm(t, kind, w, b):
            if kind == "none":
                return t
            if kind == "layer":
                return torch.nn.functional.layer_norm(t, t.shape[1:], w, b, EPS)
            return t / (t.square().mean(1, keepdim=True) + EPS).sqrt() * w

        u = norm(v["feats"], case["norm"], v.get("weight"), v.get("bias"))
        if case["gate"] == "sample":
            u = u * torch.repeat_interleave(v["gate"], counts, dim=0)
        elif case["gate"] == "channel":
            u = u * v["gate"]
        hidden = v["residual"] + u
        outs = {"hidden": hidden, "normed": norm(hidden, case["next_norm"], v["next_weight"], v.get("next_bias"))}
        grads = [s.get("grad_hidden"), s.get("grad_normed")]
    if not case["train"]:
        return outs
    got = torch.autograd.grad(list(outs.values()), list(v.values()), [g.double() for g in grads])
    return {**{k: t.detach() for k, t in outs.items()}, **dict(zip(v, got))}
