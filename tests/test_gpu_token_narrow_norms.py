"""Norms over rows of few channels: fewer than a wide access holds, and just above, where nearly every
access is moved back to end with its row; and over many rows, which fewer lanes share.

Tolerances: a row is a few float32 sums (1e-5 of its largest result) and one rounding.  A LayerNorm of few
channels can divide by a small deviation: with eps 0.25 its square root is 0.5 at least, so an error of
1e-6 of a row's largest sum grows no more than twice."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nnunet_mlx.model import tokens
from oracle import tokens as ot

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("channels", [1, 2, 3, 4, 5, 7, 8, 9, 15, 17])
def test_few_channels(device, channels, kind, dtype):
    gen = torch.Generator().manual_seed(channels)
    rows = 300
    x, residual, gate = (torch.randn(rows, channels, generator=gen).to(dtype).cuda() for _ in range(3))
    scale, *vectors = (torch.randn(channels, generator=gen).cuda() for _ in range(5))
    post, pre = vectors[:2], vectors[2:]
    total, y = tokens.residual_norm(x, residual, kind=kind, post=post, pre=pre, gate=gate, gate_activation="silu",
                                    scale=scale, residual_scale=0.7, eps=0.25)
    want, want_y = ot.residual_norm(_f64(x), _f64(residual), kind=kind, post=[_f64(p) for p in post],
                                    pre=[_f64(p) for p in pre], gate=_f64(gate), activation="silu", scale=_f64(scale),
                                    residual_scale=0.7, eps=0.25)
    for got, expected in ((total, want), (y, want_y)):
        size = np.abs(expected).max(-1, keepdims=True) + np.abs(want).max(-1, keepdims=True) + 1
        assert (np.abs(_f64(got) - expected) <= U[dtype] * np.abs(expected) + 1e-5 * size).all()


@pytest.mark.parametrize("dtype", list(U))
def test_one_channel_has_no_deviation(device, dtype):
    """The LayerNorm of one channel is its bias, exactly."""
    x = torch.randn(50, 1, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    weight, bias = torch.full((1,), 3.0, device="cuda"), torch.full((1,), -0.5, device="cuda")
    total, y = tokens.residual_norm(x, x, post=(weight, bias), pre=(weight, bias), eps=1e-5)
    assert torch.equal(total, (x.float() - 0.5).to(dtype)) and (y == -0.5).all()


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("channels", [129, 256, 257, 320, 384, 385])
def test_many_rows(device, channels, dtype):
    """Rows about the 8192 from which 16 lanes take a row: each as it is among few, up to the order of sums."""
    gen = torch.Generator().manual_seed(channels)
    x, residual = (torch.randn(8200, channels, generator=gen).to(dtype).cuda() for _ in range(2))
    affine = (torch.randn(channels, generator=gen).cuda(), torch.randn(channels, generator=gen).cuda())
    total, y = tokens.residual_norm(x, residual, post=affine, pre=affine, eps=1e-3)
    for rows in (slice(0, 70), slice(8130, 8200)):
        want, want_y = ot.residual_norm(_f64(x[rows]), _f64(residual[rows]), post=[_f64(a) for a in affine],
                                        pre=[_f64(a) for a in affine], eps=1e-3)
        for got, expected in ((total[rows], want), (y[rows], want_y)):
            size = np.abs(expected).max(-1, keepdims=True)
            assert (np.abs(_f64(got) - expected) <= U[dtype] * np.abs(expected) + 1e-5 * size).all()
