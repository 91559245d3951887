"""Row operators on the CPU: what the wrappers and the C entry points refuse before any launch."""

from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from nnunet_mlx_b200 import _native, kernels
from nnunet_mlx_b200.errors import ContractError

ROOT = Path(__file__).resolve().parent.parent


def test_channel_norm_arguments():
    for bad in (dict(kind="batch"), dict(eps=0.0), dict(eps=-1e-5), dict(eps=math.nan), dict(eps=math.inf)):
        with pytest.raises(ContractError):
            kernels.ChannelNorm(**bad)
    with pytest.raises(ContractError, match="CUDA tensor"):
        kernels.channel_norm(torch.zeros(4, 8), kernels.ChannelNorm())
    with pytest.raises(ContractError, match="CUDA tensor"):
        kernels.gated_residual_join(torch.zeros(4, 8), torch.zeros(4, 8))


def test_row_strides():
    t = torch.zeros(6, 10, 16)
    assert kernels._row_stride(t, "t") == 16
    assert kernels._row_stride(t[:, :, 3:9], "t") == 16
    assert kernels._row_stride(t[1], "t") == 16
    assert kernels._row_stride(t[:, 4], "t") == 160
    assert kernels._row_stride(t[:, 4:5], "t") == 160
    assert kernels._row_stride(t[2, 3], "t") == 16
    assert kernels._row_stride(t[:1, :1, :7], "t") == 7
    assert kernels._row_stride(t[0, 0].expand(5, 16), "t") == 0
    assert kernels._row_stride(t[:, :, :1], "t") == 16
    for bad in (t[:, :4], t.transpose(0, 1), t[..., ::2], t.expand(2, 6, 10, 16)):
        with pytest.raises(ContractError, match="evenly spaced"):
            kernels._row_stride(bad, "t")


def test_overlap():
    t = torch.zeros(8, 16)
    assert kernels._overlap(t, t[3:])
    assert kernels._overlap(t[:, :8], t[:, 8:])  # address ranges that meet are refused though no element is shared
    assert not kernels._overlap(t[:4], t[4:])
    assert not kernels._overlap(t, torch.zeros(8, 16))
    assert not kernels._overlap(t[:0], t)


def _norm_args(**over):
    values = dict(x=16, out=16, rows=1, x_stride=8, out_stride=8, channels=8, x_type=0, out_type=0,
                  norm=_native.ChannelNorm(1, 1e-5, 0, 0))
    values.update(over)
    return _native.NormArgs(**values)


def _join_args(**over):
    values = dict(branch=16, skip=16, gate=0, stream=16, normed=0, rows=2, branch_stride=8, skip_stride=8,
                  stream_stride=8, channels=8)
    values.update(over)
    return _native.JoinArgs(**values)


@pytest.mark.parametrize("over", [
    dict(x=0), dict(out=0), dict(rows=0), dict(channels=0), dict(channels=16385), dict(x_type=3), dict(out_type=-1),
    dict(norm=_native.ChannelNorm(0, 1e-5, 0, 0)), dict(norm=_native.ChannelNorm(3, 1e-5, 0, 0)),
    dict(norm=_native.ChannelNorm(1, 0.0, 0, 0)), dict(rows=2, out_stride=7), dict(x_stride=-8)])
def test_c_entry_refuses_norm(over):
    args = _norm_args(**over)
    assert _native.load().nnb_channel_norm_rows(ctypes.byref(args), None) == -1
    assert b"channel_norm" in _native.load().nnb_last_error()


@pytest.mark.parametrize("over", [
    dict(branch=0), dict(skip=0), dict(stream=0), dict(rows=0), dict(channels=0), dict(channels=20000),
    dict(post=_native.ChannelNorm(5, 1e-5, 0, 0)), dict(next=_native.ChannelNorm(1, 1e-5, 0, 0)),
    dict(gate_mode=4), dict(gate_mode=1), dict(gate_mode=3, gate=16, rows_per_sample=0), dict(gate_act=9),
    dict(stream_stride=4), dict(branch_stride=-1), dict(next=_native.ChannelNorm(2, -1.0, 0, 0), normed=16),
    dict(next=_native.ChannelNorm(1, 1e-5, 0, 0), normed=16, normed_stride=8, normed_type=7)])
def test_c_entry_refuses_join(over):
    args = _join_args(**over)
    assert _native.load().nnb_gated_join(ctypes.byref(args), None) == -1
    assert b"gated_join" in _native.load().nnb_last_error()


def test_c_entry_refuses_types_of_a_join():
    args = _join_args(branch_type=_native.F32, skip_type=_native.BF16)
    assert _native.load().nnb_gated_join(ctypes.byref(args), None) == -2
    assert _native.load().nnb_gated_join(None, None) == -1
    assert _native.load().nnb_channel_norm_rows(None, None) == -1


def _project_args(**over):
    values = dict(x=16, weight=16, down=16, up=16, scales=16, bias=0, index=16, out=16, low=16, rows=2, x_stride=8,
                  out_stride=8, rows_per_index=1, weight_stride=8, k=8, n=8, adapters=1, rank=16, used_rank=9, type=_native.BF16)
    values.update(over)
    return _native.ProjectArgs(**values)


@pytest.mark.parametrize("over", [
    *(dict([(name, 0)]) for name in ("x", "weight", "down", "up", "scales", "index", "out", "rows", "k", "n",
                                     "adapters", "rank", "rows_per_index")),
    dict(rows=2 ** 31), dict(used_rank=0), dict(used_rank=17), dict(rank=8), dict(rank=272), dict(rank=24), dict(type=_native.F32), dict(x_stride=-1),
    dict(out_stride=7), dict(weight_stride=0), dict(weight_stride=12), dict(weight=18), dict(down=8), dict(up=4),
    dict(low=20), dict(low=0, k=256, weight_stride=256, x_stride=256, rows=200)])
def test_c_entry_refuses_projection(over):
    args = _project_args(**over)
    assert _native.load().nnb_project(ctypes.byref(args), None) == -1
    assert b"project" in _native.load().nnb_last_error()


def test_projection_workspace():
    load = _native.load()
    assert load.nnb_project_workspace_bytes(ctypes.byref(_project_args(rows=100, rank=32, k=4096))) >= 100 * 32 * 4
    assert load.nnb_project_workspace_bytes(ctypes.byref(_project_args(rows=300, rank=48, k=256,
                                                                       x_stride=256))) == 300 * 2 * 128
    # rows off 16 bytes are copied; a row or few, or few channels, need nothing else
    assert load.nnb_project_workspace_bytes(ctypes.byref(_project_args(rows=2, x_stride=9))) == 2 * 8 * 2
    assert load.nnb_project_workspace_bytes(ctypes.byref(_project_args(rows=1, k=256, x_stride=256))) == 0
    assert load.nnb_project_workspace_bytes(ctypes.byref(_project_args(rows=1000))) == 0
    for bad in (dict(rows=0), dict(k=0), dict(rank=0)):
        assert load.nnb_project_workspace_bytes(ctypes.byref(_project_args(**bad))) == -1
    assert load.nnb_project_workspace_bytes(None) == -1
    assert load.nnb_project(None, None) == -1


def test_packed_arguments_are_the_structures():
    values = list(range(1, 10))
    norm = _native.ChannelNorm(2, 0.5, 21, 22)
    assert _native.pack_norm(*values, 2, 0.5, 21, 22) == bytes(_native.NormArgs(*values, norm))
    values = [*range(1, 19), 0.25, 0, 23]
    join = _native.JoinArgs(*values, norm, _native.ChannelNorm(1, 2.0, 31, 0))
    assert _native.pack_join(*values, 2, 0.5, 21, 22, 1, 2.0, 31, 0) == bytes(join)
    values = list(range(1, 21))
    assert _native.pack_project(*values) == bytes(_native.ProjectArgs(*values))


def test_structures_match_the_header(tmp_path):
    names = {"nnb_channel_norm": _native.ChannelNorm, "nnb_norm_args": _native.NormArgs,
             "nnb_join_args": _native.JoinArgs, "nnb_project_args": _native.ProjectArgs}
    lines = []
    for c_name, struct in names.items():
        lines.append(f'printf("{c_name} %zu\\n", sizeof({c_name}));')
        lines += [f'printf("{c_name}.{f[0]} %zu\\n", offsetof({c_name}, {f[0]}));' for f in struct._fields_]
    source = tmp_path / "layout.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "nnb.h"\nint main(void) {\n'
                      + "\n".join(lines) + "\nreturn 0;\n}\n")
    program = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(source), "-o", str(program)], check=True)
    found = dict(line.split() for line in subprocess.run([str(program)], check=True, capture_output=True,
                                                         text=True).stdout.splitlines())
    for c_name, struct in names.items():
        assert int(found[c_name]) == ctypes.sizeof(struct)
        for field in struct._fields_:
            assert int(found[f"{c_name}.{field[0]}"]) == getattr(struct, field[0]).offset


@pytest.mark.parametrize("eps", [1e39, 1e-60])  # an infinity and a zero there
def test_channel_norm_eps_in_float32(eps):
    with pytest.raises(ContractError, match="eps"):
        kernels.ChannelNorm(eps=eps)
