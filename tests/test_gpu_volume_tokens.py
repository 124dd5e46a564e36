"""The example that runs the token operators together, against the same network in float64.

The network in float32: each operator and product errs by some 1e-6 of its result, and two blocks of
four such steps each pass an error on about once each; 1e-4 is ten times the sum."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import numpy as np
import pytest
import torch

from nnunet_mlx.model import tokens
from oracle import tokens as ot

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = Path(__file__).resolve().parents[1] / "examples" / "volume_tokens.py"
    spec = importlib.util.spec_from_file_location("volume_tokens", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _f64(x):
    return x.detach().double().cpu().numpy()


def _network(net, cubes):
    """The example's network over every foreground token, float64."""
    pair = lambda p: tuple(map(_f64, p))  # noqa: E731
    plan = net.plan
    frequencies = np.array([s % (1 << 64) for s in plan.steps.tolist()]) / 2.0**64 * 2 * math.pi
    positions, axes = cubes.positions.cpu().numpy()[None], plan.axes.cpu().numpy()
    turn = lambda x: ot.rotate(x, positions, frequencies, axes, 1.0, "half", False)  # noqa: E731
    residual, y = ot.residual_norm(_f64(cubes.voxels) @ _f64(net.embed), None, pre=pair(net.first_norm), eps=1e-6)
    see = np.broadcast_to(cubes.foreground.cpu().numpy()[:, None, None, :],
                          (1, y.shape[1], net.heads, y.shape[1]))
    for layer in net.layers:
        qkv = (y @ _f64(layer["qkv"])).reshape(1, -1, 3 * net.heads, net.head_dim)
        q, k, v = np.split(qkv, 3, axis=2)
        mixed, _ = ot.attention(turn(q), turn(k), v, see, net.head_dim**-0.5)
        residual, y = ot.residual_norm(mixed.reshape(y.shape) @ _f64(layer["out"]), residual,
                                       post=pair(layer["post"]), scale=_f64(layer["scale"]),
                                       pre=pair(layer["mlp_pre"]), eps=1e-6)
        hidden = torch.nn.functional.gelu(torch.from_numpy(y @ _f64(layer["up"]))).numpy()
        residual, y = ot.residual_norm(hidden @ _f64(layer["down"]), residual, post=pair(layer["mlp_post"]),
                                       scale=_f64(layer["scale"]), pre=pair(layer["next_pre"]), eps=1e-6)
    return y


def test_blocks_against_float64(device, example):
    cubes = example.cut(example.phantom(40), 8)  # 125 tokens in 8 blocks of 16: all are kept
    net = example.VolumeTokens(8, heads=2, head_dim=32, block=16, keep=8, dtype=torch.float32)
    got, kept, _, _ = net(cubes)
    want = _network(net, cubes)
    assert 0 < int(cubes.foreground.sum()) < 125
    assert np.linalg.norm(_f64(got) - want) <= 1e-4 * np.linalg.norm(want)
    assert ((kept >= 0).sum(-1) >= 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_point_against_the_held_volume(device, example, dtype):
    """With every block kept, a point's answer is plain attention over the foreground."""
    cubes = example.cut(example.phantom(64), 8)
    net = example.VolumeTokens(8, heads=3, head_dim=48, block=64, keep=8, dtype=dtype)
    _, kept, k, v = net(cubes)
    assert (kept[..., 0] >= 0).all()
    query = torch.randn(1, 1, 3, 48, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    at = torch.tensor([[1, 2, 3]], dtype=torch.int32, device="cuda")
    answer = net.point(query, at, k, v, tokens.summarize_blocks(k, 64, key_mask=cubes.foreground), cubes.foreground)
    turned, _ = tokens.rotate(query, None, at, net.plan)
    see = np.broadcast_to(cubes.foreground.cpu().numpy()[:, None, None, :], (1, 1, 3, 512))
    want, size = ot.attention(_f64(turned), _f64(k), _f64(v), see, 48**-0.5)
    unit = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}[dtype]
    assert (np.abs(_f64(answer) - want) <= (4 * unit + 5e-4) * size[..., None]).all()


def test_command(device, example, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["volume_tokens.py", "--size", "64", "--keep", "4"])
    example.main()
    assert "512 tokens" in capsys.readouterr().out
