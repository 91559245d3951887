"""channel_norm and gated_residual_join on B200 against float64, element by element.

Tolerances are sums of roundings, derived before the first run.  ``U`` is half
a float32 step.  A row's sums run over at most 32 values in a thread, then 5
shuffles and 16 warps (or 16 values and 32 warps, summed by fours), so a sum of
C terms is off by at most 53 U times the sum of their magnitudes; products, the root and the quotient add a few U.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def rounding(ref, dtype):
    """Half a step of the stored type, its subnormal step included."""
    return torch.finfo(dtype).eps / 2 * ref.abs() + SMALLEST[dtype] / 2


def norm64(x, kind, weight, bias, eps, dx=0.0):
    """Float64 norm of rows and how far float32 arithmetic may be from it, `x` itself being off by at most `dx`."""
    dx = torch.as_tensor(dx, dtype=torch.float64, device=x.device).expand_as(x)
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    d = x - mean
    inv = 1 / (d.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    w = 1.0 if weight is None else weight.double()
    b = 0.0 if bias is None else bias.double()
    y = d * inv * w
    dd = dx + U * x.abs()
    if kind == "layer":
        dd = dd + dx.mean(-1, keepdim=True) + 56 * U * x.abs().mean(-1, keepdim=True)
    rel = 64 * U + dd.pow(2).mean(-1, keepdim=True).sqrt() * inv  # of the inverse deviation
    off = (dd * inv * w).abs() + y.abs() * rel
    y = y + b
    return y, off + U * y.abs()


def assert_within(got, ref, off, what):
    g, r = got.double(), ref
    bad = ((g - r).abs() > off + rounding(r, got.dtype)) | (g.isnan() != r.isnan())
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, the first at "
                           f"{bad.nonzero()[0].tolist()}: {g[bad][0].item()!r} for {r[bad][0].item()!r}")


def make(rng, shape, dtype, device, mean=0.3, size=1.0):
    v = rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal(shape[-1:])) * size + mean
    return torch.from_numpy(v).to(device).to(TYPES[dtype])


def params(rng, channels, device, bias=True):
    w = torch.from_numpy(1 + 0.2 * rng.standard_normal(channels)).float().to(device)
    return w, torch.from_numpy(0.1 * rng.standard_normal(channels)).float().to(device) if bias else None


def check_norm(x, kind, weight, bias, eps, out_dtype, **more):
    from nnunet_mlx_b200 import kernels

    ref, off = norm64(x.double(), kind, weight, bias, eps)
    got = kernels.channel_norm(x, kernels.ChannelNorm(kind, weight, bias, eps), out_dtype=out_dtype, **more)
    assert got.shape == x.shape
    assert_within(got, ref, off, f"{kind} {tuple(x.shape)} {x.dtype}")
    return got


@pytest.mark.parametrize("channels", [1, 3, 8, 31, 32, 33, 64, 100, 128, 200, 256, 320, 333, 512, 520, 1000, 1024,
                                      2048, 2049, 4096, 5001, 8192, 9000, 16384])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_over_channel_counts(cuda_device, channels, kind):
    rng = np.random.default_rng(channels)
    for rows, dtype, out in ((1, "f32", "bf16"), (5, "bf16", "bf16"), (131, "f16", "f32"), (37, "f32", "f32")):
        weight, bias = params(rng, channels, cuda_device, bias=rows != 5)
        check_norm(make(rng, (rows, channels), dtype, cuda_device), kind, weight, bias, 1e-5, TYPES[out])


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norm_of_more_rows_than_the_grid_holds(cuda_device, kind):
    rng = np.random.default_rng(1)
    for rows, channels in ((300_001, 32), (9001, 64), (4001, 1024)):
        weight, bias = params(rng, channels, cuda_device)
        check_norm(make(rng, (rows, channels), "bf16", cuda_device), kind, weight, bias, 1e-5, torch.float32)


@pytest.mark.parametrize("channels", [32, 40, 333, 1024])
def test_norm_strides_and_layouts(cuda_device, channels):
    rng = np.random.default_rng(2)
    weight, bias = params(rng, channels, cuda_device)
    for extra, start in ((8, 0), (8, 8), (5, 0), (5, 3), (1, 1)):  # aligned and odd strides and starts
        wide = make(rng, (19, channels + extra), "bf16", cuda_device)
        check_norm(wide[:, start:start + channels], "layer", weight, bias, 1e-5, torch.bfloat16)
    volume = make(rng, (2, 3, 4, 5, channels), "f32", cuda_device)
    check_norm(volume, "rms", weight, None, 1e-5, torch.bfloat16)
    check_norm(volume[:1, 1:2, :, 0], "rms", weight, None, 1e-5, torch.bfloat16)  # axes of one, a spaced axis
    check_norm(make(rng, (1, channels), "f16", cuda_device).expand(7, channels), "rms", weight, bias, 1e-5,
               torch.float16)  # one row for all
    weight2 = torch.cat([weight.new_zeros(1), weight])[1:].contiguous()
    check_norm(volume, "layer", weight2, bias, 1e-5, torch.float32)


def test_norm_in_place_out_and_empty(cuda_device):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(3)
    weight, bias = params(rng, 320, cuda_device)
    n = kernels.ChannelNorm("layer", weight, bias)
    for x in (make(rng, (50, 320), "f32", cuda_device), make(rng, (50, 325), "f16", cuda_device)[:, 2:322]):
        want = kernels.channel_norm(x, n)
        got = kernels.channel_norm(x, n, out=x)
        assert got is x and torch.equal(x, want)
    behind = torch.full((60, 330), 7.0, device=cuda_device)
    kernels.channel_norm(make(rng, (50, 320), "bf16", cuda_device), n, out=behind[5:55, 4:324])
    assert (behind[:5] == 7).all() and (behind[55:] == 7).all() and (behind[:, :4] == 7).all()
    assert (behind[:, 324:] == 7).all()
    assert kernels.channel_norm(torch.empty((0, 4, 320), device=cuda_device), n).shape == (0, 4, 320)


def test_norm_values_at_the_edges(cuda_device):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(4)
    x = make(rng, (6, 96), "f32", cuda_device)
    x[0] = 0.0                      # nothing to divide by but eps
    x[1] = 1000.0                   # a constant row: the variance is zero exactly
    x[2] = x[2] * 1e-3 + 1000.0     # a mean far above the spread
    x[3] *= 1e15
    weight, bias = params(rng, 96, cuda_device)
    for kind in ("rms", "layer"):
        check_norm(x, kind, weight, bias, 1e-5, torch.float32)
    x[4, 7] = float("nan")
    x[5, 3] = float("inf")
    got = kernels.channel_norm(x, kernels.ChannelNorm("rms", weight, bias))
    assert got[4].isnan().all() and got[5, 3].isnan() and got[:4].isfinite().all()
    assert torch.equal(got[5, 4:], bias[4:])  # a finite value over an infinite root


JOINS = [  # stream, branch, post, gate, act, next, next type
    ("f32", "f32", "rms", "full", "sigmoid", "layer", "f32"),
    ("f32", "bf16", "layer", "row", "tanh", "rms", "bf16"),
    ("f32", "f16", None, "full", "silu", "rms", "f16"),
    ("bf16", "bf16", "rms", "none", "none", None, None),
    ("bf16", "bf16", "rms", "full", "sigmoid", "rms", "bf16"),
    ("f16", "f16", "layer", "row", "none", "layer", "f32"),
    ("f32", "f32", None, "none", "none", None, None),
    ("f16", "f16", "rms", "sample", "sigmoid", "rms", "f16"),
]


def gate64(gate, act):
    """The gate's factor in float64 and its error relative to it, from the documented bounds of exp and tanh."""
    g = gate.double()
    value = {"none": g, "sigmoid": torch.sigmoid(g), "silu": g * torch.sigmoid(g), "tanh": torch.tanh(g)}[act]
    # exp(-g) is within 2 + 1.16 |g| units, a unit being at most 2 U; sum, quotient (2 units) and product follow
    rel = {"none": 0 * g, "tanh": 4 * U + 0 * g}.get(act, (2 * (2 + 1.16 * g.abs()) + 8) * U)
    return value, rel


def check_join(branch, skip, post, gate, act, scale, alpha, following, next_dtype, out=None):
    from nnunet_mlx_b200 import kernels

    def norm(n):
        return None if n is None else kernels.ChannelNorm(*n)

    z, dz = branch.double(), torch.zeros(branch.shape, dtype=torch.float64, device=branch.device)
    if post is not None:
        z, dz = norm64(z, *post)
    if gate is not None:
        value, rel = gate64(gate, act)
        if gate.dim() == 2 and branch.dim() > 2:
            value, rel = (v.view(-1, *[1] * (branch.dim() - 2), v.shape[-1]) for v in (value, rel))
        z, dz = z * value, dz * value.abs() + (z * value).abs() * rel
    f = alpha * (1.0 if scale is None else scale.double())
    term = z * f
    dt = dz * abs(f) + 4 * U * term.abs()
    stream = skip.double() + term
    ds = dt + U * stream.abs()
    got, normed = kernels.gated_residual_join(
        branch, skip, post=norm(post), gate=gate, gate_act=act, scale=scale, residual_scale=alpha,
        next_norm=norm(following), next_dtype=next_dtype, out=out)
    assert got.dtype == skip.dtype and got.shape == skip.shape
    if following is None:
        assert normed is None
    else:
        assert normed.dtype == (next_dtype or branch.dtype)
        ref, off = norm64(stream, *following, dx=ds)
        assert_within(normed, ref, off, f"next {tuple(branch.shape)}")
    assert_within(got, stream, ds, f"stream {tuple(branch.shape)}")
    return got, normed


@pytest.mark.parametrize("channels", [1, 7, 32, 64, 100, 320, 512, 1000, 2048, 4096, 5000, 8192, 16384])
@pytest.mark.parametrize("join", JOINS, ids=lambda j: "-".join(str(v) for v in j))
def test_join(cuda_device, channels, join):
    dtype, btype, post, gate, act, following, ntype = join
    rng = np.random.default_rng(channels)
    for rows in (1, 6, 133) if channels < 4096 else (5,):
        shape = (3, rows, 1, channels) if gate == "sample" else (rows, channels)
        branch, skip = make(rng, shape, btype, cuda_device), make(rng, shape, dtype, cuda_device)
        gshape = {"none": None, "full": shape, "row": (rows, 1), "sample": (3, channels)}[gate]
        g = None if gshape is None else make(rng, gshape, btype, cuda_device, mean=0.0, size=3.0)
        scale = params(rng, channels, cuda_device)[0] if rows != 6 else None
        p = None if post is None else (post, *params(rng, channels, cuda_device, post == "layer"), 1e-5)
        n = None if following is None else (following, *params(rng, channels, cuda_device), 1e-6)
        check_join(branch, skip, p, g, act, scale, 0.7, n, None if ntype is None else TYPES[ntype])


# One length for every number of threads a row and elements a thread, aligned and not, with more rows than the GPU
# holds at once.
@pytest.mark.parametrize("channels", [
    40, 72, 136, 264, 400, 640, 776, 1280, 1536, 1544, 2304, 2816, 3096, 4560, 5128, 6152, 8200, 10248, 12296,
    13, 21, 37, 45, 61, 75, 91, 121, 150, 189, 251, 301, 381, 501, 701, 1001, 1201, 1501, 2001, 2501, 3001, 4001, 4501,
    5001, 6001, 8001, 10001, 12001])
def test_every_number_of_threads(cuda_device, channels):
    rows = max(450, min(5000, 1_200_000 // channels))
    gen = torch.Generator(device=cuda_device).manual_seed(channels)

    def values(shape, dtype):
        return torch.randn(shape, device=cuda_device, generator=gen).add_(0.3).to(TYPES[dtype])

    def norm(kind):
        return kind, values(channels, "f32"), values(channels, "f32"), 1e-5

    for dtype, kind, out in (("f32", "rms", "bf16"), ("f16", "layer", "f32")):
        _, weight, bias, eps = norm(kind)
        check_norm(values((rows, channels), dtype), kind, weight, bias, eps, TYPES[out])
    for dtype, btype, gate in (("f32", "bf16", (rows, channels)), ("bf16", "bf16", (rows, 1)), ("f32", "f32", None)):
        check_join(values((rows, channels), btype), values((rows, channels), dtype), norm("layer"),
                   None if gate is None else values(gate, btype), "none" if gate is None else "sigmoid",
                   values(channels, "f32"), 0.7, norm("rms"), None)


@pytest.mark.parametrize("channels", [24, 333, 1024])
def test_join_strides_and_in_place(cuda_device, channels):
    rng = np.random.default_rng(5)
    for extra in (0, 8, 3):
        wide = [make(rng, (21, channels + extra), "f16", cuda_device)[:, extra // 2:extra // 2 + channels]
                for _ in range(3)]
        p, n = ("rms", *params(rng, channels, cuda_device), 1e-5), ("layer", *params(rng, channels, cuda_device), 1e-5)
        check_join(wide[0], wide[1], p, wide[2], "silu", None, 1.3, n, None)
        check_join(wide[0], wide[1], p, wide[2][:, :1], "tanh", None, 1.3, n, None)
        before = wide[1].clone()
        want, want_next = check_join(wide[0], before, p, wide[2][:1], "sigmoid", None, 1.3, n, None)
        got, got_next = check_join(wide[0], before, p, wide[2][:1], "sigmoid", None, 1.3, n, None, out=before)
        assert got is before and torch.equal(got, want) and torch.equal(got_next, want_next)


def test_join_of_many_rows(cuda_device):
    rng = np.random.default_rng(6)
    for rows, channels in ((200_003, 32), (3001, 2048)):
        branch, skip = (make(rng, (rows, channels), t, cuda_device) for t in ("bf16", "f32"))
        p, n = ("rms", *params(rng, channels, cuda_device), 1e-5), ("rms", *params(rng, channels, cuda_device), 1e-5)
        check_join(branch, skip, p, make(rng, (rows, 1), "bf16", cuda_device), "sigmoid", None, 1.0, n, None)


def test_gate_values_at_the_edges(cuda_device):
    from nnunet_mlx_b200 import kernels

    g = torch.tensor([[-200.0, -88.5, -87.0, -30.0, 0.0, 30.0, 200.0, 3e38]], device=cuda_device)
    branch, skip = torch.ones_like(g), torch.zeros_like(g)
    for act in ("sigmoid", "tanh"):
        got, _ = kernels.gated_residual_join(branch, skip, gate=g, gate_act=act)
        value, rel = gate64(g, act)
        assert_within(got, value, value.abs() * rel + 1e-37, act)  # below float32's normal range the quotient is zero
    empty, normed = kernels.gated_residual_join(branch[:0], skip[:0], next_norm=kernels.ChannelNorm())
    assert empty.shape == normed.shape == (0, 8)


def test_what_lies_behind_a_row_is_not_read(cuda_device):
    rng = np.random.default_rng(11)
    for channels in (24, 31, 320, 333, 2048, 5000):
        for dtype in ("f32", "bf16"):
            wide = [make(rng, (9, channels + 8), dtype, cuda_device) for _ in range(3)]
            for t in wide:
                t[:, channels:] = float("nan")
            branch, skip, gate = (t[:, :channels] for t in wide)
            p, n = (("layer", *params(rng, channels, cuda_device), 1e-5) for _ in range(2))
            check_norm(branch, "layer", p[1], p[2], 1e-5, torch.float32)
            check_join(branch, skip, p, gate, "sigmoid", p[1], 0.7, n, torch.float32)


def test_other_stream_and_capture(cuda_device):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(7)
    branch, skip = (make(rng, (64, 320), t, cuda_device) for t in ("bf16", "f32"))
    n = kernels.ChannelNorm("rms", *params(rng, 320, cuda_device))
    want, want_next = kernels.gated_residual_join(branch, skip, post=n, next_norm=n)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got, got_next = kernels.gated_residual_join(branch, skip, post=n, next_norm=n)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got_next, want_next)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held, held_next = kernels.gated_residual_join(branch, skip, post=n, next_norm=n)
        again = kernels.channel_norm(held, n)
    branch.copy_(make(rng, (64, 320), "bf16", cuda_device))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    want, want_next = kernels.gated_residual_join(branch, skip, post=n, next_norm=n)
    assert torch.equal(held, want) and torch.equal(held_next, want_next)
    assert torch.equal(again, kernels.channel_norm(want, n))


def test_refusals(cuda_device):
    from nnunet_mlx_b200 import kernels
    from nnunet_mlx_b200.errors import ContractError

    d = cuda_device
    x, n = torch.zeros((4, 32), device=d), kernels.ChannelNorm()
    w = torch.ones(32, device=d)

    def refused(call, match):
        with pytest.raises(ContractError, match=match):
            call()

    refused(lambda: kernels.channel_norm(x.double(), n), "float32, bfloat16 or float16")
    refused(lambda: kernels.channel_norm(x, n, out_dtype=torch.int32), "out_dtype")
    refused(lambda: kernels.channel_norm(x.t(), n), "evenly spaced")
    refused(lambda: kernels.channel_norm(torch.zeros((4, 4, 4, 32), device=d)[:, :2, 1:3], n), "evenly spaced")
    refused(lambda: kernels.channel_norm(x, kernels.ChannelNorm("rms", w[:31])), "norm weight")
    refused(lambda: kernels.channel_norm(x, kernels.ChannelNorm("rms", w.bfloat16())), "norm weight")
    refused(lambda: kernels.channel_norm(x, kernels.ChannelNorm("rms", w.cpu())), "norm weight")
    refused(lambda: kernels.channel_norm(torch.zeros((1, 16385), device=d), n), "16385 channels")
    refused(lambda: kernels.channel_norm(torch.zeros((4, 0), device=d), n), "channels in its last axis")
    refused(lambda: kernels.channel_norm(x, n, out=torch.empty((4, 31), device=d)), "out must be")
    refused(lambda: kernels.channel_norm(x[:3], n, out=x[1:]), "out overlaps x")
    refused(lambda: kernels.channel_norm(x[:1], kernels.ChannelNorm("rms", w), out=w.view(1, 32)), "out overlaps weight")
    refused(lambda: kernels.channel_norm(x, n, out=x[:1].expand(4, 32)), "overlap")
    refused(lambda: kernels.channel_norm(x.requires_grad_(), n), "no backward pass")
    refused(lambda: kernels.channel_norm(x.detach(), kernels.ChannelNorm("rms", torch.nn.Parameter(w))),
            "no backward pass")
    with torch.no_grad():
        assert not kernels.channel_norm(x, kernels.ChannelNorm("rms", torch.nn.Parameter(w))).requires_grad
    x = x.detach()
    join = kernels.gated_residual_join
    refused(lambda: join(x, x[:3]), "residual shapes differ")
    refused(lambda: join(x, x.bfloat16()), "stream of its own type")
    refused(lambda: join(x.half(), x.bfloat16()), "stream of its own type")
    refused(lambda: join(x, x, gate=x.half()), "the gate must have")
    refused(lambda: join(x, x, gate=x[:, :2]), "fits no element")
    refused(lambda: join(x, x, gate=x[:2]), "fits no element")
    refused(lambda: join(x, x, gate=x, gate_act="relu"), "unknown gate activation")
    refused(lambda: join(x, x, scale=w[1:]), "scale")
    refused(lambda: join(x, x, next_norm=n, next_dtype=torch.float64), "next_dtype")
    refused(lambda: join(x, torch.ones_like(x), out=x), "out overlaps branch")
    refused(lambda: join(x, x, out=torch.empty((4, 32), device=d, dtype=torch.half)), "out must be")
