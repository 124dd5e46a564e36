"""Rows at the borders of what is held, keys and values each against the oracle."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nnunet_mlx.model import tokens
from oracle import tokens as ot

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_values_at_the_borders(device, dtype):
    """Zero, tiny, at the end of the type, not finite, half-way: values as keys, and both as the oracle.  Where m is the
    type's end, scale = min(m, 3.4028233e38) / 127 and 127 times that are off by a rounding each and the minimum by
    2^-23: 2^-22 of m; a 16-bit type's rounding takes that back to m."""
    top = torch.finfo(dtype).max
    x = torch.zeros(1, 12, 2, 16)
    x[0, 1, :, 3] = 2.0**-61 if dtype != torch.float16 else 0.0
    x[0, 2, :, :] = torch.arange(16) / 8 - 1
    x[0, 3, :, :2] = torch.tensor([top, -top])
    x[0, 4, :, 5] = math.inf
    x[0, 5, :, 6] = -math.inf
    x[0, 6, :, 7] = math.nan
    x[0, 7, :, :] = torch.tensor([127.0] + [i + 0.5 for i in range(15)])
    x[0, 8, :, :] = -x[0, 7, :, :]
    x[0, 9, :, 0] = 2.0**-20
    x[0, 10, :, 15] = -1.0
    x[0, :, 1] *= 0.5
    x = x.to(dtype).cuda()
    y = x.flip(2).contiguous()  # values of their own
    held = tokens.hold_tokens(tokens.held_tokens(1, 12, 2, 16), x, y)
    for side, given in ((0, x), (2, y)):
        codes, scales = ot.hold(given.float().cpu().numpy())
        codes, scales = (np.pad(a.swapaxes(1, 2), [(0, 0), (0, 0), (0, 52)] + [(0, 0)] * (a.ndim - 3)) for a in (codes, scales))
        want = ot.place_values(codes) if side else codes
        assert np.array_equal(held[side].cpu().numpy(), want)
        assert np.array_equal(held[side + 1].cpu().numpy(), scales, equal_nan=True)
    k, v = tokens.read_held(held, dtype, count=12)
    assert torch.equal(k.nan_to_num(7.0), v.flip(2).nan_to_num(7.0))
    end = float(k[0, 3, 0, 0])
    if dtype == torch.float32:
        assert abs(end - top) <= 2.0**-22 * top
    else:
        assert end == top
    assert float(k[0, 3, 0, 1]) == -end
