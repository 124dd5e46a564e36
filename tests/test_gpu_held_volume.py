"""The example that answers points against a held volume, against the same block in float64.

The block in float32 against float64 over the same quantised codes: each operator errs by some 1e-6 of its result and
passes an error on about once, 1e-4 is ten times the sum.  A code may still fall to the other side of a half-way
value, where the float32 keys and values that it is formed of differ from float64's: it is off by one step of 127
then, in one element of some thousand, less than 1e-4 of what attention gathers.  bfloat16 rounds eight tensors on
the way to 2^-9 of their elements each, which no step passes on more than twice: 16 * 2^-9, some 3 in 100; 16-bit
roundings also move codes by a step, 1 in 127 of a row's largest, of a random half of the elements, another 1 in 100."""

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
    path = Path(__file__).resolve().parents[1] / "examples" / "held_volume.py"
    spec = importlib.util.spec_from_file_location("held_volume", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _f64(x):
    return x.detach().double().cpu().numpy()


class _Block:
    """The example's block in float64, over tokens that are held as it quantises them."""

    def __init__(self, block):
        matrix = lambda p: _f64(tokens.unpack_weight(p, torch.float32)).T  # noqa: E731
        self.block = block
        self.qkv, self.out, self.gate, self.up, self.down = map(matrix, (block.qkv, block.out, block.gate, block.up, block.down))
        self.frequencies = np.array([s % (1 << 64) for s in block.plan.steps.tolist()]) / 2.0**64 * 2 * math.pi
        self.axes = block.plan.axes.cpu().numpy()
        self.k = self.v = None

    def norm(self, x, residual, affine):
        return ot.residual_norm(x, residual, kind="rms", pre=(_f64(affine[0]), None))

    def project(self, y, positions):
        b = self.block
        qkv = (y @ self.qkv).reshape(*y.shape[:2], -1, b.head_dim)
        q, k, v = np.split(qkv, [b.heads, b.heads + b.kv_heads], 2)
        turn = lambda x: ot.rotate(x, positions[None], self.frequencies, self.axes, 1.0, "half", False)  # noqa: E731
        return turn(q), turn(k), v

    def hold(self, k, v):
        new = []
        for x in (k, v):
            codes, scales = ot.hold(x.astype(np.float32))
            new.append(codes.astype(np.float64) * scales[..., None])
        self.k, self.v = new if self.k is None else (np.concatenate([a, b], 1) for a, b in zip((self.k, self.v), new))

    def volume(self, x, positions):
        _, k, v = self.project(self.norm(x, None, self.block.pre)[1], positions)
        self.hold(k, v)

    def __call__(self, x, positions):
        residual, y = self.norm(x, None, self.block.pre)
        q, k, v = self.project(y, positions)
        before = self.k.shape[1]
        self.hold(k, v)
        see = np.arange(self.k.shape[1])[None, :] <= before + np.arange(x.shape[1])[:, None]
        see = np.broadcast_to(see[None, :, None, :], (*x.shape[:2], self.block.kv_heads, see.shape[1]))
        mixed, _ = ot.attention(q, self.k, self.v, see, self.block.head_dim**-0.5)
        residual, y = self.norm(mixed.reshape(*x.shape[:2], -1) @ self.out, residual, self.block.mlp_pre)
        hidden = ot.gated(y @ self.up, y @ self.gate, "silu")
        return self.norm(hidden @ self.down, residual, self.block.next_pre)


@pytest.mark.parametrize("dtype,most", [(torch.float32, 1e-4), (torch.bfloat16, 0.05)])
def test_points_against_float64(device, example, dtype, most):
    """Two steps of points behind a volume of 125 tokens."""
    block = example.PointBlock(heads=4, kv_heads=2, head_dim=48, hidden=200, group=32, dtype=dtype)
    want = _Block(block)
    gen = torch.Generator().manual_seed(5)
    positions = torch.randint(0, 30, (125, 3), generator=gen, dtype=torch.int32)
    volume = torch.randn(1, 125, 192, generator=gen).to(dtype)
    held = block.hold(volume.cuda(), positions.cuda(), room=10)
    want.volume(_f64(volume), positions.numpy())
    lengths = torch.full((1,), 125, dtype=torch.int32, device="cuda")
    for n in (1, 7):
        points = torch.randn(1, n, 192, generator=gen).to(dtype)
        at = torch.randint(0, 30, (n, 3), generator=gen, dtype=torch.int32)
        got = block(points.cuda(), at.cuda(), held, lengths)
        for a, b in zip(got, want(_f64(points), at.numpy())):
            assert np.linalg.norm(_f64(a) - b) <= most * np.linalg.norm(b)
    assert lengths.tolist() == [133]


def test_a_captured_step(device, example):
    """The step of a point as a graph: replayed, it holds and answers what the eager one does."""
    block = example.PointBlock()
    gen = torch.Generator().manual_seed(6)
    positions = torch.randint(0, 30, (300, 3), generator=gen, dtype=torch.int32).cuda()
    volume = torch.randn(1, 300, 320, generator=gen).to(torch.bfloat16).cuda()
    held, eager = (block.hold(volume, positions, room=64) for _ in range(2))
    lengths, others = (torch.full((1,), 300, dtype=torch.int32, device="cuda") for _ in range(2))
    point, at = volume[:, :1].clone(), positions[:1].clone()
    graph = torch.cuda.CUDAGraph()
    block(point, at, eager, others)  # the first call loads what the capture needs
    with torch.cuda.graph(graph):
        answer = block(point, at, held, lengths)[1]
    others.fill_(300)
    for i in range(4):
        point.copy_(torch.randn(point.shape, generator=gen))
        at.copy_(torch.randint(0, 30, at.shape, generator=gen, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(answer, block(point, at, eager, others)[1])
        assert lengths.tolist() == others.tolist() == [301 + i]
    for a, b in zip(held, eager):
        assert torch.equal(a, b)


def test_command(device, example, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["held_volume.py", "--size", "64"])
    example.main()
    assert "512 tokens held" in capsys.readouterr().out
