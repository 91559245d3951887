"""Measured cases of the channel-norm, gated-join and adapted-projection operators of ``nnunet_mlx_b200.kernels``.

``run`` with ``own`` false computes each operator from elementary torch
operations in float32; with ``own`` true it makes the framework's calls.
Rows are the voxels or tokens of channels-last activations.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
DEVICE = "cuda"

LARGEST_PRODUCT = 8192 * 4096 * 4096
LARGEST_ROWS = 16384 * 4096


def listed():
    return [
        # one row of a bottleneck activation through a small projection with one site's adapter: the latency of a call
        {"name": "project one row", "op": "project", "rows": 1, "k": 320, "n": 320, "rank": 8, "adapters": 4,
         "requests": 1, "samples": 0, "dtype": "bf16", "ragged": False, "wide": 0, "bias": True},
        # a decode-like batch: 64 requests of one row each, most with another adapter; bound by the weights
        {"name": "project 64 requests", "op": "project", "rows": 64, "k": 4096, "n": 4096, "rank": 16, "adapters": 48,
         "requests": 64, "samples": 0, "dtype": "bf16", "ragged": False, "wide": 0, "bias": False},
        # odd sizes throughout, ranks that differ, rows taken out of a wider buffer, float16
        {"name": "project odd sizes", "op": "project", "rows": 1777, "k": 1001, "n": 333, "rank": 13, "adapters": 5,
         "requests": 9, "samples": 0, "dtype": "f16", "ragged": True, "wide": 7, "bias": True},
        # an ordinary batch: eight ragged requests' rows widened fourfold
        {"name": "project ragged requests", "op": "project", "rows": 2048, "k": 1024, "n": 4096, "rank": 16,
         "adapters": 8, "requests": 8, "samples": 0, "dtype": "bf16", "ragged": True, "wide": 0, "bias": True},
        # two samples of full-resolution 128^3 activations through a 32 -> 32 projection, an adapter each: bound by HBM
        {"name": "project two volumes", "op": "project", "rows": 2 * 128 ** 3, "k": 32, "n": 32, "rank": 4,
         "adapters": 3, "requests": 2, "samples": 2, "dtype": "bf16", "ragged": False, "wide": 0, "bias": True},
        # the largest: many long requests through a square projection with wide adapters; bound by the tensor cores
        {"name": "project long requests", "op": "project", "rows": 8192, "k": 4096, "n": 4096, "rank": 64,
         "adapters": 16, "requests": 24, "samples": 0, "dtype": "bf16", "ragged": True, "wide": 0, "bias": False},
        # one token's norm before a block: latency
        {"name": "norm one token", "op": "norm", "rows": 1, "channels": 320, "kind": "rms", "dtype": "f32",
         "out": "bf16", "wide": 0},
        # the norm of a full-resolution 128^3 activation of 32 channels, rounded for the next projection
        {"name": "norm volume", "op": "norm", "rows": 128 ** 3, "channels": 32, "kind": "layer", "dtype": "f32",
         "out": "bf16", "wide": 0},
        # a decode-like batch of joins with the next norm
        {"name": "join 64 tokens", "op": "join", "rows": 64, "channels": 2048, "dtype": "bf16", "branch": "bf16",
         "post": "rms", "gate": "full", "act": "sigmoid", "next": "rms", "out": "bf16", "samples": 0, "wide": 0},
        # odd sizes, layer norms, a gate value per row, rows out of a wider buffer
        {"name": "join odd sizes", "op": "join", "rows": 3001, "channels": 333, "dtype": "f16", "branch": "f16",
         "post": "layer", "gate": "row", "act": "tanh", "next": "none", "out": "f16", "samples": 0, "wide": 5},
        # an ordinary block on a 64^3 activation of two samples, gated per sample and channel, float32 stream
        {"name": "join volume", "op": "join", "rows": 2 * 64 ** 3, "channels": 64, "dtype": "f32", "branch": "bf16",
         "post": "rms", "gate": "sample", "act": "none", "next": "layer", "out": "bf16", "samples": 2, "wide": 0},
        # the largest join: long batch, float32 stream beside a bf16 branch and a full gate
        {"name": "join long batch", "op": "join", "rows": 16384, "channels": 4096, "dtype": "f32", "branch": "bf16",
         "post": "rms", "gate": "full", "act": "silu", "next": "rms", "out": "bf16", "samples": 0, "wide": 0},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A channel count: half of them any number, half a multiple of 32."""
    c = _spread(rng, lo, hi)
    return c if rng.random() < 0.5 else max(32, c // 32 * 32)


def draw(rng):
    op = rng.choice(["project", "project", "norm", "join"])
    if op == "project":
        k, n = _width(rng, 16, 4096), _width(rng, 16, 4096)
        samples = rng.choice([0, 0, 0, rng.randint(1, 4)])
        most = 2 * 128 ** 3 if k * n <= 64 * 64 else 16384
        rows = _spread(rng, 1, max(1, min(most, LARGEST_PRODUCT // (k * n))))
        if samples:
            rows = samples * max(1, rows // samples)
        mixed = not samples and rows <= 256
        requests = samples or (rows if mixed else rng.randint(1, 24))
        return {"op": op, "rows": rows, "k": k, "n": n, "rank": _spread(rng, 1, 64),
                "adapters": _spread(rng, 1, 8 if rows > 16384 else 64), "requests": requests, "samples": samples,
                "dtype": rng.choice(["bf16", "bf16", "f16"]), "ragged": rng.random() < 0.5,
                "wide": rng.choice([0, 0, rng.randint(1, 64)]), "bias": rng.random() < 0.5}
    c = _width(rng, 8, 8192)
    rows = _spread(rng, 1, min(2 * 128 ** 3, LARGEST_ROWS // c))
    wide = rng.choice([0, 0, rng.randint(1, 64)])
    if op == "norm":
        return {"op": op, "rows": rows, "channels": c, "kind": rng.choice(["rms", "layer"]),
                "dtype": rng.choice(["f32", "bf16", "f16"]), "out": rng.choice(["f32", "bf16", "f16"]), "wide": wide}
    dtype, branch = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
    samples = rng.randint(1, 4)
    gate = rng.choice(["none", "full", "row", "sample"])
    if gate == "sample":
        rows = samples * max(1, rows // samples)
        wide = 0
    return {"op": op, "rows": rows, "channels": c, "dtype": dtype, "branch": branch,
            "post": rng.choice(["none", "rms", "layer"]), "gate": gate,
            "act": rng.choice(["none", "sigmoid", "silu", "tanh"]), "next": rng.choice(["none", "rms", "layer"]),
            "out": rng.choice([branch, "f32"]), "samples": samples if gate == "sample" else 0, "wide": wide}


def _ranks(case):
    """Each adapter's rank: the case's, or where they differ a fourth, a half, three fourths or all of it."""
    r = case["rank"]
    return [max(1, r * (4 - i % 4) // 4) if case["ragged"] else r for i in range(case["adapters"])]


def _rows(gen, rows, c, dtype, wide):
    """An activation with channels of different size and mean, as residual streams have; `wide` columns behind each row."""
    size = torch.exp(0.5 * torch.randn(c + wide, device=DEVICE, generator=gen))
    x = torch.randn((rows, c + wide), device=DEVICE, generator=gen).mul_(size).add_(0.3 * size)
    return x.to(DTYPES[dtype])[:, :c]


def _norm(gen, kind, c):
    if kind == "none":
        return None
    weight = 1 + 0.2 * torch.randn(c, device=DEVICE, generator=gen)
    bias = 0.1 * torch.randn(c, device=DEVICE, generator=gen) if kind == "layer" else None
    return {"kind": kind, "weight": weight, "bias": bias, "eps": 1e-5}


def _own_norm(norm):
    if not own or norm is None:
        return None
    from nnunet_mlx_b200 import kernels

    return kernels.ChannelNorm(norm["kind"], norm["weight"], norm["bias"], norm["eps"])


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["op"] == "norm":
        norm = _norm(gen, case["kind"], case["channels"])
        return {"case": case, "x": _rows(gen, case["rows"], case["channels"], case["dtype"], case["wide"]),
                "norm": norm, "own_norm": _own_norm(norm)}
    if case["op"] == "join":
        rows, c = case["rows"], case["channels"]
        post, following = _norm(gen, case["post"], c), _norm(gen, case["next"], c)
        branch = _rows(gen, rows, c, case["branch"], case["wide"])
        skip = _rows(gen, rows, c, case["dtype"], case["wide"])
        gate = None
        if case["gate"] != "none":
            shape = {"full": (rows, c), "row": (rows, 1), "sample": (case["samples"] or 1, c)}[case["gate"]]
            gate = torch.randn(shape, device=DEVICE, generator=gen).to(DTYPES[case["branch"]])
        if case["samples"]:
            branch, skip = (t.view(case["samples"], -1, c) for t in (branch, skip))
        return {"case": case, "branch": branch, "skip": skip, "gate": gate, "post": post, "next": following,
                "scale": 0.5 + 0.2 * torch.randn(c, device=DEVICE, generator=gen), "alpha": 0.7,
                "own_post": _own_norm(post), "own_next": _own_norm(following)}
    rows, k, n, count = case["rows"], case["k"], case["n"], case["adapters"]
    dtype = DTYPES[case["dtype"]]
    x = torch.randn((rows, k + case["wide"]), device=DEVICE, generator=gen).to(dtype)[:, :k]
    weight = (torch.randn((n, k), device=DEVICE, generator=gen) / math.sqrt(k)).to(dtype)
    bias = 0.1 * torch.randn(n, device=DEVICE, generator=gen) if case["bias"] else None
    ranks = _ranks(case)
    down = (torch.randn((count, case["rank"], k), device=DEVICE, generator=gen) / math.sqrt(k)).to(dtype)
    up = (torch.randn((count, n, case["rank"]), device=DEVICE, generator=gen) / math.sqrt(case["rank"])).to(dtype)
    # below an adapter's own rank: the padded columns hold nothing
    keep = torch.arange(case["rank"], device=DEVICE)[None, :] < torch.tensor(ranks, device=DEVICE)[:, None]
    down, up = down * keep[:, :, None], up * keep[:, None, :]
    scales = torch.rand(count, device=DEVICE, generator=gen) + 0.25
    # each request has an adapter, or none (-1); a request's rows follow one another
    adapter = torch.randint(-1, count, (case["requests"],), device=DEVICE, generator=gen)
    if case["samples"]:
        x = x.unflatten(0, (case["samples"], -1))
        index = adapter
    else:
        cuts = torch.rand(rows, device=DEVICE, generator=gen).argsort() < case["requests"] - 1
        index = adapter[cuts.cumsum(0) - cuts.long()] if case["requests"] < rows else adapter
    state = {"case": case, "x": x, "weight": weight, "bias": bias, "down": down, "up": up, "scales": scales,
             "index": index.to(torch.int32), "projection": None}
    if own:
        from nnunet_mlx_b200 import kernels

        host = scales.tolist()
        state["projection"] = kernels.pack_projection(
            weight, [kernels.Adapter(down[i, :r], up[i, :, :r], host[i]) for i, r in enumerate(ranks)], bias=bias)
    return state


def _plain_norm(x, norm):
    if norm["kind"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + norm["eps"]) * norm["weight"]
    return y if norm["bias"] is None else y + norm["bias"]


def _plain_gate(gate, act):
    g = gate.float()
    if act == "tanh":
        return torch.tanh(g)
    if act == "none":
        return g
    s = 1 / (1 + torch.exp(-g))
    return g * s if act == "silu" else s


def _plain_join(s):
    case = s["case"]
    z = s["branch"].float()
    if s["post"] is not None:
        z = _plain_norm(z, s["post"])
    if s["gate"] is not None:
        g = _plain_gate(s["gate"], case["act"])
        z = z * (g[:, None, :] if case["gate"] == "sample" else g)
    stream = s["skip"].float() + s["alpha"] * s["scale"] * z
    out = {"stream": stream.to(DTYPES[case["dtype"]])}
    if s["next"] is not None:
        out["next"] = _plain_norm(stream, s["next"]).to(DTYPES[case["out"]])
    return out


def _plain_project(s):
    x = s["x"].flatten(0, -2).float()
    rows, k = x.shape
    count, rank, _ = s["down"].shape
    index = s["index"].long()
    if index.numel() != rows:
        index = index[:, None].expand(-1, rows // index.numel()).flatten()
    y = x @ s["weight"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"]
    # every adapter's low-rank rows, of which each row keeps its own adapter's
    low = (x @ s["down"].float().view(count * rank, k).t()).view(rows, count, rank)
    mine = (index[:, None] == torch.arange(count, device=x.device)) * s["scales"]
    low = (low * mine[:, :, None]).view(rows, count * rank)
    y = y + low @ s["up"].float().transpose(1, 2).reshape(count * rank, -1)
    return y.to(s["weight"].dtype).view(*s["x"].shape[:-1], -1)


def run(state):
    case = state["case"]
    if not own:
        if case["op"] == "norm":
            return _plain_norm(state["x"].float(), state["norm"]).to(DTYPES[case["out"]])
        return _plain_join(state) if case["op"] == "join" else _plain_project(state)
    from nnunet_mlx_b200 import kernels

    if case["op"] == "norm":
        return kernels.channel_norm(state["x"], state["own_norm"], out_dtype=DTYPES[case["out"]])
    if case["op"] == "join":
        stream, following = kernels.gated_residual_join(
            state["branch"], state["skip"], post=state["own_post"], gate=state["gate"], gate_act=case["act"],
            scale=state["scale"], residual_scale=state["alpha"], next_norm=state["own_next"],
            next_dtype=DTYPES[case["out"]])
        return {"stream": stream} if following is None else {"stream": stream, "next": following}
    return kernels.adapted_projection(state["x"], state["projection"], state["index"])


def work(case):
    if case["op"] == "norm":
        values = case["rows"] * case["channels"]
        return {"bytes": values * (SIZES[case["dtype"]] + SIZES[case["out"]]), "flops": 6 * values}
    if case["op"] == "join":
        rows, c = case["rows"], case["channels"]
        gate = {"none": 0, "full": rows * c, "row": rows, "sample": case["samples"] * c}[case["gate"]]
        moved = rows * c * (SIZES[case["branch"]] + 2 * SIZES[case["dtype"]]) + gate * SIZES[case["branch"]]
        if case["next"] != "none":
            moved += rows * c * SIZES[case["out"]]
        return {"bytes": moved, "flops": 16 * rows * c}
    rows, k, n, ranks = case["rows"], case["k"], case["n"], _ranks(case)
    mean_rank = sum(ranks) / len(ranks)
    used = min(case["adapters"], case["requests"])
    return {"bytes": int(2 * (rows * (k + n) + n * k + used * mean_rank * (k + n))),
            "flops": int(2 * rows * (n * k + mean_rank * (k + n)))}


def _exact_norm(x, norm):
    spread = x.var(-1, correction=0, keepdim=True) if norm["kind"] == "layer" else x.pow(2).mean(-1, keepdim=True)
    if norm["kind"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = norm["weight"].double() * (x / (spread + norm["eps"]).sqrt())
    return y if norm["bias"] is None else norm["bias"].double() + y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s["x"].double(), s["norm"])
    if case["op"] == "join":
        z = s["branch"].double()
        if s["post"] is not None:
            z = _exact_norm(z, s["post"])
        if s["gate"] is not None:
            g = s["gate"].double()
            g = {"none": lambda v: v, "tanh": torch.tanh, "sigmoid": torch.sigmoid,
                 "silu": lambda v: v * torch.sigmoid(v)}[case["act"]](g)
            z = z * (g.unsqueeze(1) if case["gate"] == "sample" else g)
        stream = s["skip"].double() + z * s["scale"].double() * s["alpha"]
        return {"stream": stream} if s["next"] is None else {"stream": stream, "next": _exact_norm(stream, s["next"])}
    x = s["x"].reshape(-1, case["k"]).double()
    y = torch.mm(x, s["weight"].double().t())
    if s["bias"] is not None:
        y += s["bias"].double()
    index = torch.repeat_interleave(s["index"], x.shape[0] // s["index"].numel())
    for a in range(case["adapters"]):
        at = (index == a).nonzero().flatten()
        if at.numel():
            low = torch.mm(x[at], s["down"][a].double().t())
            y[at] += s["scales"][a].double() * torch.mm(low, s["up"][a].double().t())
    return y.view(*s["x"].shape[:-1], -1)
