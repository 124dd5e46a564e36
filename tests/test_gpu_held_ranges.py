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


CAUSAL = [
    # dim, queries, heads, key heads, slots, first position, the slot of the large value
    (16, 2, 1, 1, 2, 0, 1),
    (32, 40, 4, 2, 100, 30, 50),
    (64, 100, 2, 2, 200, 100, 163),
    (128, 17, 8, 2, 70, 50, 64),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("power", [20, 40, 100])
@pytest.mark.parametrize("case", CAUSAL)
def test_values_behind_a_query(device, case, power, dtype):
    """What slots behind a query hold does not change a bit of its result, however large they are."""
    dim, queries, heads, kv_heads, n, start, large = case
    k, v = (torch.randn(1, n, kv_heads, dim, generator=_gen(i)).cuda() for i in (4, 5))
    q = torch.randn(1, queries, heads, dim, generator=_gen(6)).to(dtype).cuda()
    before = large - start  # queries that do not see it
    assert 0 < before < queries
    held = tokens.hold_tokens(tokens.held_tokens(1, n, kv_heads, dim), k, v)
    want = tokens.held_attention(q, held, n, causal=True, start=start)[:, :before]
    v[:, large] *= 2.0**power
    tokens.hold_tokens(held, k, v)
    got = tokens.held_attention(q, held, n, causal=True, start=start)[:, :before]
    assert torch.equal(got, want)
    held.v_scales[:, :, large] = 1e-30
    assert torch.equal(tokens.held_attention(q, held, n, causal=True, start=start)[:, :before], want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("power", [-60, 0, 20, 40, 57, 80, 100])
@pytest.mark.parametrize("case", [(1, 1, 1, 200, 32), (2, 40, 2, 200, 64), (1, 3, 1, 5000, 128), (1, 2, 2, 9, 96)])
def test_the_smallest_value_weighs_most(device, case, power, dtype):
    """Slot 0 outweighs the others by 2^57, whose values are 2^power times as large in even channels and 0 in odd ones.
    Odd channels are slot 0's value but for its weight, 1 to within 2^-40, and 16 roundings: products, sums, shares of
    parts.  In even channels a logit below 21 is off by (dim + 4) u of that, weights by twice as much and 6 u, n of them by n u more
    in their sums, of which each counts twice.

    Where slot 0 holds 0 in an even channel, the others' 2^-57 times values of 2^-60 are all there is, and operands of
    them fall below float32's least normal value as in the next test: 2^-126 twice a slot, times codes below 2^7 and the
    factor 2^34 of scales on the way, over a sum of weights of 1 and more, is n 2^-84."""
    batch, queries, heads, n, dim = case
    gen, u = _gen(7), 2.0**-24
    k = -1 + 0.02 * torch.randn(batch, n, heads, dim, generator=gen)
    k[:, 0] = 1
    v = torch.randn(batch, n, heads, dim, generator=gen)
    v[:, 1:] *= 2.0**power
    v[:, 1:, :, 1::2] = 0
    q = (20 + 0.1 * torch.randn(batch, queries, heads, dim, generator=gen)).to(dtype).cuda()
    held = tokens.hold_tokens(tokens.held_tokens(batch, n, heads, dim), k.cuda(), v.cuda())
    got = tokens.held_attention(q, held, n, scale=1 / dim)
    k, v = (x.double().transpose(1, 2).contiguous() for x in tokens.read_held(held, torch.float32, count=n))
    logits = torch.matmul(q.double().transpose(1, 2), k.transpose(2, 3).contiguous()) / dim
    assert float(logits.abs().max()) < 21
    p = torch.softmax(logits, -1)
    assert float((1 - p[..., 0]).max()) < 2.0**-40
    want, size = (torch.matmul(p, x).transpose(1, 2) for x in (v, v.abs()))
    odd, even = slice(1, None, 2), slice(0, None, 2)
    assert _rounded_between(got[..., odd], want[..., odd], 16 * u * want[..., odd].abs())
    off = 2 * (2 * (dim + 4) * 21 + 6 + n) * u
    off = off * size + n * 2.0**-84
    inside = (want.abs() + off)[..., even] <= torch.finfo(dtype).max
    got, want, off = (x[..., even][inside] for x in (got, want, off))
    assert _rounded_between(got, want, off)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("power", [-58, -40, 60, 120])
def test_values_of_one_size(device, dtype, power):
    """Values near both ends of what is held differ from others by their power of two alone.  Of the smallest, 2^-58 and
    more, operands of products may fall below float32's least normal value: 2^-126 twice for each of 300 slots,
    times codes below 2^7 and 2^34, the factor of scales on the way, which is below 2^-17 of them.  So a result, which
    is rounded twice, may be off by that and two roundings."""
    n = 300
    k, v = (torch.randn(1, n, 2, 48, generator=_gen(i)).cuda() for i in (8, 9))
    v = v.clamp(-3, 3) + torch.sign(v)
    q = torch.randn(1, 33, 2, 48, generator=_gen(10)).to(dtype).cuda()
    held = tokens.hold_tokens(tokens.held_tokens(1, n, 2, 48), k, v)
    want = tokens.held_attention(q, held, n)
    tokens.hold_tokens(held, k, v * 2.0**power)
    got = tokens.held_attention(q, held, n)
    if power > -58:
        assert torch.equal(got.float(), (want.float() * 2.0**power).to(dtype).float())
    else:
        off = 4 * U[dtype] * want.double().abs() + 2.0**-17
        assert bool(((got.double() * 2.0**-power - want.double()).abs() <= off).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 70, 5000])
@pytest.mark.parametrize("queries", [1, 40])
def test_infinite_queries(device, queries, n, dtype):
    """An infinite element makes its row NaN, as the softmax of infinite logits is, also where all of them are -inf."""
    k, v = (torch.randn(1, n, 2, 32, generator=_gen(i)).cuda() for i in (11, 12))
    held = tokens.hold_tokens(tokens.held_tokens(1, n, 2, 32), k.abs() + 0.5, v)
    q = torch.randn(1, queries, 4, 32, generator=_gen(13)).to(dtype).cuda()
    want = tokens.held_attention(q, held, n)
    for sign in (-1, 1):
        odd = q.clone()
        odd[0, -1, 3, 9] = sign * float("inf")
        got = tokens.held_attention(odd, held, n)
        assert torch.isnan(got[0, -1, 3]).all()
        got[0, -1, 3] = want[0, -1, 3]
        assert torch.equal(got, want)
        assert not tokens.held_attention(odd, held, 0).any()
