"""Row operators on B200 at the edges of their values, on every kernel that a projection may take.

``PATHS`` names, for each kernel or combination of them, a projection that
takes it.  Ranks of one and two are among the adapters, since an infinite
low-rank value leaves infinities only where the signs of all its products
agree; the other ranks make those be padded.
"""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from tests.test_gpu_project import TYPES, check, make_index, make_rows, problem

pytestmark = pytest.mark.gpu

PATHS = {  # rows, k, n, ranks
    "narrow, 8 ranks": (200, 32, 32, [1, 5, 8]),
    "narrow, one group": (200, 30, 32, [1, 2, 13]),
    "narrow, several groups": (300, 72, 100, [2, 1, 20]),
    "few rows, low-rank rows in the kernel": (4, 320, 320, [1, 2, 8]),
    "few rows, partial sums": (100, 1024, 640, [2, 1, 40]),
    "low-rank rows by rows, tiles of 64": (256, 1024, 512, [1, 2, 16] * 20),
    "low-rank tiles by clusters, tiles of 64": (300, 1024, 333, [2, 13, 1]),
    "low-rank tiles, tiles of 128": (1500, 136, 1500, [1, 20, 2]),
    "low-rank tiles, pairs": (2100, 136, 1100, [1, 2, 20]),
}
BAD_INDEX = 64  # the site that an adapter index out of range is reported at


def adapted_problem(rng, path, dtype, device, bias=True):
    rows, k, n, ranks = PATHS[path]
    parts = problem(rng, k, n, ranks, dtype, device, bias)
    for a in parts[1]:
        a.up[::2] = a.up[::2].bfloat16().to(a.up.dtype)  # (float16) values that leave no remainder beside those that do
    return rows, k, n, ranks, parts


def by_definition(x, parts, index):
    """Float64 rows, each product taken apart, so that nothing but the formula meets an infinity."""
    weight, adapters, bias = parts
    out = []
    for row, a in zip(x.double(), index.tolist()):
        y = (weight.double() * row).sum(-1)
        if bias is not None:
            y = y + bias.double()
        if a >= 0:
            low = (adapters[a].down.double() * row).sum(-1)
            y = y + adapters[a].scale * (adapters[a].up.double() * low).sum(-1)
        out.append(y)
    return torch.stack(out)


@pytest.mark.parametrize("mode", ["mixed", "one"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("path", PATHS)
def test_infinities_follow_the_definition(cuda_device, path, dtype, mode):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(21)
    rows, k, n, ranks, parts = adapted_problem(rng, path, dtype, cuda_device)
    projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    x = make_rows(rng, (rows, k), dtype, cuda_device)
    index = make_index(rng, rows, len(ranks), "mixed", cuda_device)
    if mode == "one":
        index.fill_(ranks.index(1))
    index[:4] = torch.tensor([ranks.index(1), ranks.index(2) if 2 in ranks else 0, -1, len(ranks) - 1])
    if mode == "one":
        index[:4] = ranks.index(1)
    want = kernels.adapted_projection(x, projection, index)
    assert want.isfinite().all()
    hit = torch.tensor([0, 1, 2, 3] + ([rows // 2, rows - 1] if rows > 8 else []), device=cuda_device)
    for i, row in enumerate(hit.tolist()):
        x[row, (7 * i) % k] = float("inf") if i % 2 == 0 else -float("inf")
    got = kernels.adapted_projection(x, projection, index)
    ref = by_definition(x[hit], parts, index[hit])
    mine = got[hit].double()
    assert ref.isinf().any()
    assert torch.equal(mine.isnan(), ref.isnan())
    assert torch.equal(mine.isposinf(), ref.isposinf()) and torch.equal(mine.isneginf(), ref.isneginf())
    rest = torch.ones(rows, dtype=torch.bool, device=cuda_device)
    rest[hit] = False
    assert torch.equal(got[rest], want[rest])
    x[hit[0]] = float("nan")
    got = kernels.adapted_projection(x, projection, index)
    assert got[hit[0]].isnan().all() and torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("path", PATHS)
def test_bad_index_on_every_path(cuda_device, path, dtype):
    from nnunet_mlx_b200 import _native, kernels

    rng = np.random.default_rng(22)
    rows, k, n, ranks, parts = adapted_problem(rng, path, dtype, cuda_device)
    projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    x = make_rows(rng, (rows, k), dtype, cuda_device)
    for mode in ("mixed", "one"):
        index = make_index(rng, rows, len(ranks), mode, cuda_device)
        for bad_rows in ([0, rows - 1], list(range(rows // 2, rows))):  # (the second leaves whole tiles without any)
            bad = index.clone()
            bad[bad_rows] = torch.tensor([len(ranks), -2, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32,
                                         device=cuda_device).repeat(len(bad_rows))[:len(bad_rows)]
            got = kernels.adapted_projection(x, projection, bad)
            assert _native.device_status(reset=True) == (-4, BAD_INDEX)
            good = index.clone()
            good[bad_rows] = -1
            assert torch.equal(got, kernels.adapted_projection(x, projection, good))
            assert _native.device_status(reset=True)[0] == 0


@pytest.mark.parametrize("path", PATHS)
def test_low_rank_values_beyond_float16(cuda_device, path):
    rng = np.random.default_rng(23)
    rows, k, n, ranks, parts = adapted_problem(rng, path, "f16", cuda_device)
    for a in parts[1]:
        a.down.mul_(3e4)
        a.up.mul_(1e-4)
    for mode in ("mixed", "one"):
        check(make_rows(rng, (rows, k), "f16", cuda_device), parts,
              make_index(rng, rows, len(ranks), mode, cuda_device))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("path", PATHS)
def test_calls_repeat_bit_by_bit(cuda_device, path, dtype):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(24)
    rows, k, n, ranks, parts = adapted_problem(rng, path, dtype, cuda_device)
    projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    xs = [make_rows(rng, (rows, k), dtype, cuda_device) for _ in range(2)]
    index = make_index(rng, rows, len(ranks), "mixed", cuda_device)
    want = [kernels.adapted_projection(x, projection, index) for x in xs]
    for _ in range(10):
        for x, w in zip(xs, want):
            assert torch.equal(kernels.adapted_projection(x, projection, index), w)


@pytest.mark.parametrize("factor", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("path", PATHS)
def test_an_infinite_factor_reaches_its_own_rows_alone(cuda_device, path, factor):
    """``pack_projection`` refuses it; laid out by other means it spoils no other request."""
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(25)
    rows, k, n, ranks, parts = adapted_problem(rng, path, "bf16", cuda_device)
    projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
    scales = projection.scales.clone()
    scales.view(len(ranks), -1)[0, 0] = factor
    spoilt = dataclasses.replace(projection, scales=scales)
    x = make_rows(rng, (rows, k), "bf16", cuda_device)
    index = make_index(rng, rows, len(ranks), "mixed", cuda_device)
    index[0] = 0
    want, got = (kernels.adapted_projection(x, p, index) for p in (projection, spoilt))
    others = index != 0
    assert torch.equal(got[others], want[others])
    assert not got[~others].isfinite().any()


def test_factors_outside_float32_are_refused(cuda_device):
    from nnunet_mlx_b200 import kernels
    from nnunet_mlx_b200.errors import ContractError

    rng = np.random.default_rng(26)
    weight, adapters, bias = problem(rng, 64, 48, [8, 4], "bf16", cuda_device)
    for scale in (1e39, -1e39, 3.5e38, float("inf")):
        with pytest.raises(ContractError, match="finite"):
            kernels.pack_projection(weight, [adapters[0], kernels.Adapter(adapters[1].down, adapters[1].up, scale)])


def test_residual_scales_outside_float32_are_refused(cuda_device):
    from nnunet_mlx_b200 import kernels
    from nnunet_mlx_b200.errors import ContractError

    x = torch.ones((4, 32), device=cuda_device)
    for scale in (1e39, -1e39):
        with pytest.raises(ContractError, match="residual_scale"):
            kernels.gated_residual_join(x, x, residual_scale=scale)
    got, _ = kernels.gated_residual_join(x, x, residual_scale=float("inf"))
    assert got.isposinf().all()


def test_packing_refuses_what_requires_a_gradient(cuda_device):
    from nnunet_mlx_b200 import kernels
    from nnunet_mlx_b200.errors import ContractError

    rng = np.random.default_rng(27)
    weight, adapters, bias = problem(rng, 64, 48, [8, 4], "bf16", cuda_device)
    tracked = [torch.nn.Parameter(t) for t in (weight, adapters[0].down, adapters[0].up, bias)]
    calls = [
        lambda: kernels.pack_projection(tracked[0], adapters, bias=bias),
        lambda: kernels.pack_projection(weight, [kernels.Adapter(tracked[1], adapters[0].up), adapters[1]], bias=bias),
        lambda: kernels.pack_projection(weight, [adapters[1], kernels.Adapter(adapters[0].down, tracked[2])], bias=bias),
        lambda: kernels.pack_projection(weight, adapters, bias=tracked[3]),
    ]
    for call in calls:
        with pytest.raises(ContractError, match="no backward pass"):
            call()
        with torch.no_grad():
            p = call()
        assert not any(t.requires_grad for t in (p.weight, p.down, p.up, p.scales))


def test_forward_mode_tangents_are_refused(cuda_device):
    from torch.autograd import forward_ad

    from nnunet_mlx_b200 import kernels
    from nnunet_mlx_b200.errors import ContractError

    rng = np.random.default_rng(28)
    weight, adapters, bias = problem(rng, 32, 32, [8], "bf16", cuda_device)
    p = kernels.pack_projection(weight, adapters, bias=bias)
    x, index = make_rows(rng, (6, 32), "bf16", cuda_device), torch.zeros(6, dtype=torch.int32, device=cuda_device)
    plain, w = x.float(), torch.ones(32, device=cuda_device)
    norm = kernels.ChannelNorm("rms", w)
    with forward_ad.dual_level():
        kernels.channel_norm(plain, norm)  # no tangent, no refusal
        kernels.adapted_projection(x, p, index)
        dual, dual_x, dual_w = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (plain, x, w))
        for call in (
            lambda: kernels.channel_norm(dual, norm),
            lambda: kernels.channel_norm(plain, kernels.ChannelNorm("rms", dual_w)),
            lambda: kernels.gated_residual_join(dual, plain),
            lambda: kernels.gated_residual_join(plain, dual),
            lambda: kernels.gated_residual_join(plain, plain, gate=dual),
            lambda: kernels.gated_residual_join(plain, plain, scale=dual_w),
            lambda: kernels.adapted_projection(dual_x, p, index),
            lambda: kernels.pack_projection(forward_ad.make_dual(weight, weight), adapters),
        ):
            with pytest.raises(ContractError, match="tangent"):
                call()


def test_results_written_in_place_are_seen_by_autograd(cuda_device):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(29)
    weight, adapters, bias = problem(rng, 32, 32, [8], "bf16", cuda_device)
    p = kernels.pack_projection(weight, adapters, bias=bias)
    x, index = make_rows(rng, (6, 32), "bf16", cuda_device), torch.zeros(6, dtype=torch.int32, device=cuda_device)
    norm = kernels.ChannelNorm()
    for call in (lambda out: kernels.channel_norm(x, norm, out=out),
                 lambda out: kernels.gated_residual_join(x, x, out=out),
                 lambda out: kernels.adapted_projection(x, p, index, out=out)):
        out = torch.zeros((6, 32), dtype=torch.bfloat16, device=cuda_device)
        factor = torch.ones_like(out, requires_grad=True)
        y = factor * out  # keeps `out` for its backward pass
        call(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():
        inner = torch.zeros((6, 32), dtype=torch.bfloat16, device=cuda_device)
        kernels.channel_norm(x, norm, out=inner)
    kernels.channel_norm(x, norm, out=inner)  # an inference tensor has no versions
    assert torch.equal(inner, kernels.channel_norm(x, norm))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gates_of_every_size(cuda_device, dtype):
    """A float32 gate's sigmoid within 16 float32 roundings whatever its size: the base-2 exponential is within 2^-22.5
    (3 U), what its argument leaves out is made up for (2 U), the reciprocal within 2^-23 (2 U), and the sum's and the
    products' roundings follow.  A bfloat16 gate's by the fast exponential, within 2 + 1.16 |g| units of the last place.
    Either is zero where it is below float32's normal range."""
    from nnunet_mlx_b200 import kernels

    U = 2.0 ** -24
    g = torch.cat([torch.linspace(-110.0, 110.0, 200_001, dtype=torch.float64),
                   torch.tensor([-200.0, -3e38, 3e38, 0.0, -0.0, 1e-30, -1e-30])]).to(cuda_device)
    gate = g[:g.numel() // 8 * 8].to(TYPES.get(dtype, torch.float32)).view(-1, 8)
    branch, skip = torch.ones_like(gate), torch.zeros(gate.shape, device=cuda_device)
    v = gate.double()
    for act in ("sigmoid", "silu"):
        got, _ = kernels.gated_residual_join(branch, skip, gate=gate, gate_act=act)
        ref = torch.sigmoid(v) * (v if act == "silu" else 1.0)
        times = v.abs().clamp(1.0, 128.0) if act == "silu" else 1.0
        if dtype == "f32":
            off = 16 * U * ref.abs() + 2.0 ** -126 * times
        else:
            off = (2 * (2 + 1.16 * v.abs().clamp(max=200.0)) + 8) * U * ref.abs() + 2.0 ** -126 * times
        assert ((got.double() - ref).abs() <= off).all()
    edge = torch.tensor([[float("nan"), float("inf"), -float("inf")]], device=cuda_device, dtype=gate.dtype)
    for act, want in (("sigmoid", (1.0, 0.0)), ("silu", (float("inf"), None))):
        got, _ = kernels.gated_residual_join(torch.ones_like(edge), torch.zeros_like(edge), gate=edge, gate_act=act)
        assert got[0, 0].isnan() and got[0, 1] == want[0]
        assert got[0, 2].isnan() if want[1] is None else got[0, 2] == want[1]


def test_norm_and_join_past_32_bits(cuda_device):
    """More than 2^31 elements of every operand; rows from the end are compared with the same rows by themselves."""
    from nnunet_mlx_b200 import kernels

    for channels in (16384, 40):
        rows = (2 ** 31) // channels + 77
        x = torch.empty((rows, channels), dtype=torch.bfloat16, device=cuda_device).normal_()
        skip = torch.empty_like(x).normal_()
        norm = kernels.ChannelNorm("layer", torch.linspace(0.5, 1.5, channels, device=cuda_device))
        got = kernels.channel_norm(x, norm)
        stream, normed = kernels.gated_residual_join(x, skip, post=norm, gate=x, gate_act="tanh", next_norm=norm)
        for part in (slice(0, 50), slice(rows - 100, rows)):
            assert torch.equal(got[part], kernels.channel_norm(x[part].clone(), norm))
            a, b = kernels.gated_residual_join(x[part].clone(), skip[part].clone(), post=norm, gate=x[part].clone(),
                                               gate_act="tanh", next_norm=norm)
            assert torch.equal(stream[part], a) and torch.equal(normed[part], b)
        del x, skip, got, stream, normed


def test_narrow_projection_past_32_bits(cuda_device):
    from nnunet_mlx_b200 import kernels

    rng = np.random.default_rng(30)
    for ranks, per_row in (([4, 7], True), ([16, 9], False)):
        rows = 2 ** 26 + 6 * 77
        parts = problem(rng, 32, 40, ranks, "bf16", cuda_device)
        projection = kernels.pack_projection(parts[0], parts[1], bias=parts[2])
        x = torch.empty((rows, 32), dtype=torch.bfloat16, device=cuda_device).normal_()
        if per_row:
            index = torch.arange(rows, device=cuda_device).remainder_(3).sub_(1).int()
            got = kernels.adapted_projection(x, projection, index)
        else:
            index = torch.tensor([1, 0], dtype=torch.int32, device=cuda_device)
            got = kernels.adapted_projection(x.view(2, -1, 32), projection, index).view(rows, 40)
            index = index.repeat_interleave(rows // 2)
        for part in (slice(0, 500), slice(rows // 2 - 300, rows // 2 + 300), slice(rows - 500, rows)):
            want = kernels.adapted_projection(x[part].clone(), projection, index[part].clone())
            assert torch.equal(got[part], want)
        check(x[-500:], parts, index[-500:].clone(), projection)
        del x, got


@pytest.mark.parametrize("index", [None, [0, 0, 0, 0], 0])
def test_an_index_that_is_no_tensor_is_refused(cuda_device, index):
    from nnunet_mlx_b200 import kernels
    from nnunet_mlx_b200.errors import ContractError

    rng = np.random.default_rng(31)
    weight, adapters, _ = problem(rng, 32, 32, [8], "bf16", cuda_device)
    projection = kernels.pack_projection(weight, adapters)
    with pytest.raises(ContractError, match="index must be"):
        kernels.adapted_projection(make_rows(rng, (4, 32), "bf16", cuda_device), projection, index)
