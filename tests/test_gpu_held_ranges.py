"""Held attention as its formulas in float32 have it: one rounding of a result, and values of any size.

u = 2^-24, U a type's unit roundoff.  A result before its rounding is off by float32's own errors; how large those
may be stands at each test.  Rounding is monotonous, so a result lies between the rounded ends of that range."""

from __future__ import annotations

import pytest
import torch

from nnunet_mlx.model import tokens

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TYPES = list(U)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rounded_between(got, want, off):
    """Whether got is a float64 of want - off to want + off rounded to its type."""
    low, high = ((want + sign * off).to(got.dtype) for sign in (-1, 1))
    return bool(((got >= low) & (got <= high)).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_one_rounding(device, dtype):
    """Two million results of eight slots.  Logits below 1 err by less than (16 + 4) u, weights by twice that and 4 u,
    the operands and sums of 8 slots by 10 u: 58 u of the mean |v| in all, before the result is rounded."""
    k, v = (torch.randn(1, 8, 4, 16, generator=_gen(i)).cuda() for i in (1, 2))
    held = tokens.hold_tokens(tokens.held_tokens(1, 8, 4, 16), k, v)
    q = (0.05 * torch.randn(1, 32768, 4, 16, generator=_gen(3))).to(dtype).cuda()
    got = tokens.held_attention(q, held, 8)[0]
    k, v = (x.double()[0].permute(1, 2, 0).contiguous() for x in tokens.read_held(held, torch.float32, count=8))
    logits = torch.matmul(q.double()[0].permute(1, 0, 2).contiguous(), k) / 4  # (heads, queries, 8)
    assert float(logits.abs().max()) < 1
    p = torch.softmax(logits, -1)
    want = torch.matmul(p, v.transpose(1, 2).contiguous()).permute(1, 0, 2)
    size = torch.matmul(p, v.abs().amax(1)[..., None])[..., 0].t()[..., None]
    assert _rounded_between(got, want, 58 * 2.0**-24 * size)
