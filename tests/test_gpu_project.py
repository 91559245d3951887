"""adapted_projection on B200 against float64, element by element.

Tolerances, derived before the first run: a float32 accumulation of K products
in groups of 16 or fewer-term chains makes at most K / 8 + 32 additions, each
off by at most a whole float32 step (tensor cores cut, they do not round) of
the sum of magnitudes; a low-rank value kept as two bfloat16 parts is off by
2^-17 of itself, and the product of two remainders that is left out by 2^-18.
The result is rounded once to the stored type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
SMALLEST = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def problem(rng, k, n, ranks, dtype, device, bias=True):
    def matrix(*shape, size):
        return torch.from_numpy(rng.standard_normal(shape) * size).to(device).to(TYPES[dtype])

    from nnunet_mlx_b200 import kernels

    weight = matrix(n, k, size=k ** -0.5)
    adapters = [kernels.Adapter(matrix(r, k, size=k ** -0.5), matrix(n, r, size=r ** -0.5), 0.25 + 0.5 * i)
                for i, r in enumerate(ranks)]
    b = torch.from_numpy(0.1 * rng.standard_normal(n)).float().to(device) if bias else None
    return weight, adapters, b


def rows64(x, weight, adapters, bias, index):
    """Float64 result and how far the operator may be from it before the last rounding."""
    k = x.shape[-1]
    flat = x.reshape(-1, k).double()
    chain = (k / 8 + 32) * STEP
    y = flat @ weight.double().t()
    off = chain * (flat.abs() @ weight.double().abs().t())
    if bias is not None:
        y, off = y + bias.double(), off + STEP * bias.double().abs()
    per_row = index.reshape(-1).repeat_interleave(flat.shape[0] // max(1, index.numel()))
    for a, adapter in enumerate(adapters):
        at = (per_row == a).nonzero().flatten()
        if at.numel() == 0:
            continue
        down, up, s = adapter.down.double(), adapter.up.double(), adapter.scale
        low, low_off = flat[at] @ down.t(), chain * (flat[at].abs() @ down.abs().t())
        y[at] += s * (low @ up.t())
        off[at] += abs(s) * ((low_off + (2.0 ** -16 + chain) * low.abs()) @ up.abs().t())
    shape = (*x.shape[:-1], weight.shape[0])
    return y.view(shape), (off + STEP * y.abs()).view(shape)


def check(x, parts, index, projection=None, **more):
    from nnunet_mlx_b200 import kernels

    projection = projection or kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    got = kernels.adapted_projection(x, projection, index, **more)
    ref, off = rows64(x, *parts, index)
    assert got.shape == ref.shape and got.dtype == x.dtype
    bad = (got.double() - ref).abs() > off + torch.finfo(x.dtype).eps / 2 * ref.abs() + SMALLEST[x.dtype]
    assert not bad.any() and not got.isnan().any(), (
        f"{int(bad.sum())} of {bad.numel()} values off, the first at {bad.nonzero()[:1].tolist()}: "
        f"{got[bad][:1].tolist()} for {ref[bad][:1].tolist()}")
    return got


def make_rows(rng, shape, dtype, device):
    return torch.from_numpy(rng.standard_normal(shape)).to(device).to(TYPES[dtype])


def make_index(rng, rows, adapters, mode, device):
    if mode == "mixed":
        v = rng.integers(-1, adapters, rows)
    elif mode == "none":
        v = np.full(rows, -1)
    elif mode == "one":
        v = np.full(rows, adapters - 1)
    else:  # runs of ragged lengths
        v = np.repeat(rng.integers(-1, adapters, rows), rng.integers(1, 2 + rows // 3, rows))[:rows]
    return torch.from_numpy(v.astype(np.int32)).to(device)


SHAPES = [  # rows, k, n, ranks, index
    (1, 320, 320, [8, 8, 8, 8], "one"),
    (1, 1, 1, [1], "one"),
    (1, 33, 7, [3, 1], "none"),
    (2, 8, 16, [16], "mixed"),
    (7, 64, 64, [4, 16, 1], "mixed"),
    (31, 100, 33, [17], "mixed"),
    (64, 512, 1024, [16] * 48, "mixed"),
    (127, 256, 320, [32, 8], "runs"),
    (128, 32, 32, [4, 4, 4], "runs"),
    (129, 96, 48, [64], "runs"),
    (130, 1001, 333, [13, 9, 6, 3, 13], "runs"),
    (257, 320, 512, [48, 40], "runs"),
    (300, 72, 256, [20] * 130, "mixed"),      # over a hundred adapters among the rows of a tile
    (1000, 128, 264, [256, 100], "runs"),
    (1777, 1001, 333, [13, 9, 6, 3, 13], "runs"),
    (2048, 1024, 640, [16] * 8, "runs"),
    (640, 2048, 2048, [64] * 5, "runs"),
    (4096, 64, 32, [4, 2], "runs"),
    (20000, 32, 64, [8, 8, 8], "mixed"),
    (3000, 40, 24, [5], "none"),
    (700, 4096, 16, [16, 16], "runs"),
    (260, 16, 2000, [16, 16, 2], "mixed"),
    (256, 320, 700, [16, 9] * 40, "mixed"),    # many adapters in tiles of every width
    (1500, 256, 2000, [40, 9] * 20, "mixed"),
    (1100, 192, 8000, [20] * 50, "mixed"),
    (100, 4096, 320, [16] * 20, "mixed"),      # up to 128 rows: clusters of every size, shares of few and many rows
    (128, 640, 129, [144, 80], "mixed"),
    (3, 192, 4000, [24, 256], "mixed"),
    (128, 136, 40000, [16], "runs"),
    (17, 520, 10001, [8, 8], "mixed"),
    (5000, 128, 128, [32, 16, 7], "runs"),     # projections of few channels: every group count of 32
    (333, 127, 97, [40, 16, 7], "mixed"),
    (1, 96, 64, [200], "one"),
    (77, 40, 96, [24] * 30, "mixed"),
    (900, 90, 31, [2], "mixed"),
    (4000, 31, 128, [64, 3], "runs"),
    (600, 32, 32, [24, 20], "runs"),           # a last block of ranks that is whole, or up to 8
    (600, 64, 40, [22, 5], "mixed"),
    (600, 30, 32, [8, 7], "mixed"),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}x{s[1]}-{s[2]}-r{max(s[3])}x{len(s[3])}-{s[4]}")
def test_projection(cuda_device, shape, dtype):
    rows, k, n, ranks, mode = shape
    rng = np.random.default_rng(rows + k)
    parts = problem(rng, k, n, ranks, dtype, cuda_device, bias=rows % 2 == 1)
    check(make_rows(rng, (rows, k), dtype, cuda_device), parts,
          make_index(rng, rows, len(ranks), mode, cuda_device))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,ranks", [(48, [16, 3]), (264, [40, 9, 64]), (1400, [24] * 5)])
def test_tiles_of_one_adapter_beside_tiles_of_several(cuda_device, dtype, n, ranks):
    rng = np.random.default_rng(n)
    rows, k = 40_001, 136
    runs = [np.full(rng.choice([1, 64, 128, 256, 300, 1024]), rng.integers(-1, len(ranks))) for _ in range(400)]
    index = torch.from_numpy(np.concatenate(runs)[:rows].astype(np.int32)).to(cuda_device)
    assert index.numel() == rows
    check(make_rows(rng, (rows, k), dtype, cuda_device), problem(rng, k, n, ranks, dtype, cuda_device), index)
    one = torch.full((rows,), len(ranks) - 1, dtype=torch.int32, device=cuda_device)
    check(make_rows(rng, (rows, k), dtype, cuda_device), problem(rng, k, n, ranks, dtype, cuda_device), one)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_index_per_sample(cuda_device, dtype):
    rng = np.random.default_rng(1)
    for shape, k, n in (((3, 5, 6, 7), 32, 32), ((2, 40, 50), 64, 200), ((2, 3, 4), 40, 8), ((5, 100), 32, 320)):
        parts = problem(rng, k, n, [4, 8], dtype, cuda_device)
        x = make_rows(rng, (*shape, k), dtype, cuda_device)
        for axes in range(1, len(shape) + 1):
            index = make_index(rng, int(np.prod(shape[:axes])), 2, "mixed", cuda_device).view(shape[:axes])
            check(x, parts, index)


@pytest.mark.parametrize("k,n", [(64, 64), (72, 40), (33, 30), (320, 328)])
def test_projection_strides(cuda_device, k, n):
    rng = np.random.default_rng(2)
    parts = problem(rng, k, n, [16, 5], "bf16", cuda_device)
    for extra, start in ((8, 0), (8, 8), (5, 0), (5, 3), (2, 1)):
        x = make_rows(rng, (200, k + extra), "bf16", cuda_device)[:, start:start + k]
        index = make_index(rng, 200, 2, "runs", cuda_device)
        want = check(x, parts, index)
        behind = torch.full((210, n + extra), 7.0, dtype=torch.bfloat16, device=cuda_device)
        got = check(x, parts, index, out=behind[4:204, start:start + n])
        assert torch.equal(got, want)
        assert (behind[:4] == 7).all() and (behind[204:] == 7).all()
        assert (behind[:, :start] == 7).all() and (behind[:, start + n:] == 7).all()
    one = make_rows(rng, (1, k), "bf16", cuda_device)
    check(one.expand(150, k), parts, make_index(rng, 150, 2, "mixed", cuda_device))
    check(one[:, :k], parts, make_index(rng, 1, 2, "one", cuda_device))
    check(make_rows(rng, (9, 20, k), "bf16", cuda_device)[:, 3], parts, make_index(rng, 9, 2, "mixed", cuda_device))


def test_long_rows_offsets_past_32_bits(cuda_device):
    # rows * n and rows * stride pass 2^31 elements; the last rows are compared
    rng = np.random.default_rng(3)
    rows, k, n = 2 ** 21 + 77, 32, 1040
    parts = problem(rng, k, n, [4, 4], "bf16", cuda_device)
    from nnunet_mlx_b200 import kernels

    projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    wide = torch.empty((rows, 1032), dtype=torch.bfloat16, device=cuda_device)
    x = wide[:, 1000:]
    x.normal_()
    index = torch.full((rows,), 1, dtype=torch.int32, device=cuda_device)
    index[:1000] = 0
    got = kernels.adapted_projection(x, projection, index)
    for part in (slice(0, 2000), slice(rows - 3000, rows)):
        ref, off = rows64(x[part], *parts, index[part])
        assert ((got[part].double() - ref).abs() <= off + 2.0 ** -8 * ref.abs()).all()


def test_values_do_not_reach_other_rows(cuda_device):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(4)
    for dtype in ("bf16", "f16"):
        parts = problem(rng, 64, 96, [8, 8, 8], dtype, cuda_device)
        projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
        x = make_rows(rng, (200, 64), dtype, cuda_device)
        index = make_index(rng, 200, 3, "mixed", cuda_device)
        want = kernels.adapted_projection(x, projection, index)
        x[17, 5], x[90, 0], x[150, 63] = float("nan"), float("inf"), -float("inf")
        got = kernels.adapted_projection(x, projection, index)
        rest = torch.ones(200, dtype=torch.bool, device=cuda_device)
        rest[[17, 90, 150]] = False
        assert torch.equal(got[rest], want[rest])
        assert got[17].isnan().all() and not got[[90, 150]].isfinite().all()
    # low-rank values far above float16's range meet a small up side
    parts[1][0].down.mul_(3e4)
    parts[1][0].up.mul_(1e-4)
    check(make_rows(rng, (150, 64), "f16", cuda_device), parts, make_index(rng, 150, 3, "one", cuda_device) * 0)


@pytest.mark.parametrize("rows,k,n", [(1, 330, 40), (5, 1001, 48), (100, 330, 200), (300, 1001, 333), (700, 100, 90)])
def test_what_lies_behind_a_row_is_not_read(cuda_device, rows, k, n):
    rng = np.random.default_rng(10)
    for dtype in ("bf16", "f16"):
        parts = problem(rng, k, n, [8, 20], dtype, cuda_device)
        buffer = make_rows(rng, (rows + 2, (k + 15) // 8 * 8), dtype, cuda_device)  # rows that are read in place
        buffer[:, k:] = float("nan")
        buffer[rows:] = float("inf")
        check(buffer[:rows, :k], parts, make_index(rng, rows, 2, "mixed", cuda_device))


def test_first_call_inside_a_capture():
    """A process whose first call of every operator is captured: nothing needs a call outside before it."""
    import subprocess
    import sys

    program = """
import torch
from nnunet_mlx_b200 import kernels
d = torch.device("cuda:0")
def rows(r, k): return torch.ones((r, k), dtype=torch.bfloat16, device=d)
cases = []
for r, k, n in ((1, 256, 64), (64, 1024, 256), (300, 256, 512), (300, 255, 64), (4000, 32, 32)):
    p = kernels.pack_projection(rows(n, k), [kernels.Adapter(rows(16, k), rows(n, 16))])
    cases.append((rows(r, k), p, torch.zeros(r, dtype=torch.int32, device=d)))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = [kernels.adapted_projection(*c) for c in cases]
    normed = kernels.channel_norm(cases[0][0], kernels.ChannelNorm())
    joined, _ = kernels.gated_residual_join(normed, cases[0][0], next_norm=kernels.ChannelNorm())
for _ in range(2):
    graph.replay()
torch.cuda.synchronize()
for (x, p, i), o in zip(cases, out):
    k = x.shape[1]
    assert (o == torch.tensor(17.0 * k).bfloat16()).all(), (o.min(), o.max(), k)
assert (joined == 2).all()
"""
    done = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_order_of_rows_does_not_matter(cuda_device):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(5)
    parts = problem(rng, 256, 512, [16] * 6, "bf16", cuda_device)
    projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    x = make_rows(rng, (900, 256), "bf16", cuda_device)
    index = make_index(rng, 900, 6, "runs", cuda_device)
    want = kernels.adapted_projection(x, projection, index)
    order = torch.from_numpy(rng.permutation(900)).to(cuda_device)
    assert torch.equal(kernels.adapted_projection(x[order], projection, index[order]), want[order])
    assert torch.equal(kernels.adapted_projection(x, projection, index), want)


def test_bad_index_is_reported(cuda_device):
    from nnunet_mlx_b200 import _native, kernels

    rng = np.random.default_rng(6)
    parts = problem(rng, 64, 64, [8, 8], "bf16", cuda_device)
    projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    for rows in (9, 400):
        x = make_rows(rng, (rows, 64), "bf16", cuda_device)
        index = make_index(rng, rows, 2, "mixed", cuda_device)
        bad = index.clone()
        bad[3], bad[7], bad[8] = 2, -2, 2 ** 31 - 1
        got = kernels.adapted_projection(x, projection, bad)
        status, where = _native.device_status(reset=True)
        assert status == -4 and where > 0
        index[[3, 7, 8]] = -1
        assert torch.equal(got, kernels.adapted_projection(x, projection, index))
        assert _native.device_status(reset=True) == (0, 0) or _native.device_status(reset=True)[0] == 0


def test_streams_capture_and_interleaved_calls(cuda_device):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(7)
    parts = problem(rng, 128, 256, [16, 16], "bf16", cuda_device)
    projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    for rows in (5, 700):
        xs = [make_rows(rng, (rows, 128), "bf16", cuda_device) for _ in range(4)]
        index = make_index(rng, rows, 2, "runs", cuda_device)
        want = [kernels.adapted_projection(x, projection, index) for x in xs]
        torch.cuda.synchronize()
        sides = [torch.cuda.Stream() for _ in xs]
        got = [[] for _ in xs]
        for _ in range(5):  # calls on four streams at once
            for i, (x, side) in enumerate(zip(xs, sides)):
                with torch.cuda.stream(side):
                    got[i].append(kernels.adapted_projection(x, projection, index))
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)
        graphs, held = [], []
        for x in xs[:2]:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held.append(kernels.adapted_projection(x, projection, index))
            graphs.append(graph)
        xs[0].copy_(xs[2])
        index.copy_(index.flip(0))
        for _ in range(3):
            for graph in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for h, x in zip(held, xs):
            assert torch.equal(h, kernels.adapted_projection(x, projection, index))


def test_block_of_operators(cuda_device):
    """A residual block as it is used: norm, adapted projections, gated join with the next norm, projection."""
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(8)
    channels, hidden, rows = 320, 640, 500
    first = problem(rng, channels, hidden, [16, 8], "bf16", cuda_device)
    second = problem(rng, hidden, channels, [16, 8], "bf16", cuda_device, bias=False)
    p1, p2 = (kernels.pack_projection(w, a, bias=b) for w, a, b in (first, second))
    index = make_index(rng, rows, 2, "runs", cuda_device)
    weight = torch.from_numpy(1 + 0.2 * rng.standard_normal(channels)).float().to(cuda_device)
    pre, post = kernels.ChannelNorm("rms", weight), kernels.ChannelNorm("layer", weight)
    stream = torch.from_numpy(rng.standard_normal((rows, channels))).float().to(cuda_device)
    gate = make_rows(rng, (rows, channels), "bf16", cuda_device)
    start = stream.clone()
    x = kernels.channel_norm(stream, pre, out_dtype=torch.bfloat16)
    h = kernels.adapted_projection(x, p1, index)
    branch = kernels.adapted_projection(h, p2, index)
    joined, normed = kernels.gated_residual_join(branch, stream, post=post, gate=gate, gate_act="sigmoid",
                                                 scale=weight, residual_scale=0.5, next_norm=pre, out=stream)
    assert joined is stream

    # the same block in float64, from the bfloat16 values that are stored between the operators
    s = start.double()
    x64 = s / (s.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
    assert ((x.double() - x64).abs() <= 2.0 ** -8 * x64.abs() + 1e-5).all()
    for got, source, parts in ((h, x, first), (branch, h, second)):
        ref, off = rows64(source, *parts, index)
        assert ((got.double() - ref).abs() <= off + 2.0 ** -8 * ref.abs()).all()
    z = branch.double()
    z = (z - z.mean(-1, keepdim=True)) / (z.var(-1, correction=0, keepdim=True) + 1e-6).sqrt() * weight.double()
    s = s + 0.5 * weight.double() * torch.sigmoid(gate.double()) * z
    assert ((joined.double() - s).abs() <= 1e-5).all()
    n64 = s / (s.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
    assert ((normed.double() - n64).abs() <= 2.0 ** -8 * n64.abs() + 1e-4).all()


def test_empty_and_refusals(cuda_device):
    from nnunet_mlx_b200 import kernels
    from nnunet_mlx_b200.errors import ContractError

    d = cuda_device
    rng = np.random.default_rng(9)
    weight, adapters, bias = problem(rng, 64, 48, [8, 4], "bf16", d)
    p = kernels.pack_projection(weight, adapters, bias=bias)
    x, index = make_rows(rng, (6, 64), "bf16", d), torch.zeros(6, dtype=torch.int32, device=d)
    assert kernels.adapted_projection(x[:0], p, index[:0]).shape == (0, 48)
    assert kernels.adapted_projection(x.view(2, 3, 64)[:, :0], p, index[:2]).shape == (2, 0, 48)
    before = p.weight.clone()
    weight.zero_()
    assert torch.equal(p.weight, before)  # the pack is a copy

    def refused(call, match):
        with pytest.raises(ContractError, match=match):
            call()

    run, pack, adapter = kernels.adapted_projection, kernels.pack_projection, kernels.Adapter
    refused(lambda: run(x.half(), p, index), "x must hold")
    refused(lambda: run(x.float(), p, index), "x must hold")
    refused(lambda: run(x[:, :63], p, index), "x must hold")
    refused(lambda: run(x.t().contiguous().t(), p, index), "evenly spaced")
    refused(lambda: run(x, p, index[:5]), "index must")
    refused(lambda: run(x, p, index.long()), "index must")
    refused(lambda: run(x, p, index.cpu()), "index must")
    refused(lambda: run(x, p, index.view(6, 1)), "index must")
    refused(lambda: run(x[0], p, index[0]), "index must")
    refused(lambda: run(x, weight, index), "packed by pack_projection")
    refused(lambda: run(x, p, index, out=torch.empty((6, 47), dtype=torch.bfloat16, device=d)), "out must be")
    square = pack(torch.zeros((64, 64), dtype=torch.bfloat16, device=d), [adapter(adapters[0].down, torch.zeros(
        (64, 8), dtype=torch.bfloat16, device=d))])
    refused(lambda: run(x, square, index, out=x), "out overlaps x")
    refused(lambda: run(x.requires_grad_(), p, index), "no backward pass")
    refused(lambda: pack(weight, []), "at least one adapter")
    refused(lambda: pack(weight.float(), adapters), "bfloat16 or float16")
    refused(lambda: pack(weight, [adapter(adapters[0].down.half(), adapters[0].up)]), "weight's type")
    refused(lambda: pack(weight, [adapter(adapters[0].down, adapters[1].up)]), "do not fit")
    refused(lambda: pack(weight, [adapter(adapters[0].down[:, 1:], adapters[0].up)]), "do not fit")
    refused(lambda: pack(weight, adapters, bias=bias[1:]), "bias")
    refused(lambda: pack(weight, [adapter(adapters[0].down, adapters[0].up, float("nan"))]), "finite")
    refused(lambda: pack(weight, [adapter(adapters[0].down * float("inf"), adapters[0].up)]), "finite")
    big = torch.zeros((257, 64), dtype=torch.bfloat16, device=d), torch.zeros((48, 257), dtype=torch.bfloat16, device=d)
    refused(lambda: pack(weight, [adapter(*big)]), "rank 257")
