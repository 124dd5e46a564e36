"""What attention over selected blocks keeps of its values: every channel by itself, at any magnitude.

Tolerances.  U is a type's unit roundoff (half the spacing at 1).  Each channel is held against the mean
over its own weights of |v|, which is what an error of the weights can move it by.  Weights may be off by
U where they are rounded to the type, and by 5e-4 through a float32 logit of up to 130 terms that sum to
less than 20 in magnitude (130 * 2^-24 * 20 = 1.6e-4, a weight by twice that); partials and the result are
rounded by at most U each: 3 U + 5e-4."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from nnunet_mlx.model import tokens
from oracle import tokens as ot

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TYPES = list(U)


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def _attention(q, k, v, see, scale):
    """Float64 attention over the seen keys and the same of |v|, by channel."""
    q, k, v = map(_f64, (q, k, v))
    group = q.shape[2] // k.shape[2]
    k, v, see = (np.repeat(a, group, 2) for a in (k, v, see))
    logits = np.einsum("bthd,bshd->bths", q, k) * scale
    logits = np.where(see, logits, -np.inf)
    top = logits.max(-1, keepdims=True)
    p = np.exp(logits - np.where(np.isfinite(top), top, 0))
    p /= np.maximum(p.sum(-1, keepdims=True), 1e-300)
    return np.einsum("bths,bshd->bthd", p, v), np.einsum("bths,bshd->bthd", p, np.abs(v))


def _inputs(seed, dtype, queries, keys, heads=4, kv_heads=2, dim=64):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(1, n, h, dim, generator=gen) for n, h in ((queries, heads), (keys, kv_heads), (keys, kv_heads)))
    return q.to(dtype).cuda(), k.to(dtype).cuda(), v.to(dtype).cuda()


def _ids(queries, kv_heads, blocks, keep, seed):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.rand(1, queries, kv_heads, blocks, generator=gen).topk(keep).indices.sort(-1).values
    return ids.to(torch.int32).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [3, 1500])
@pytest.mark.parametrize("dim,block", [(64, 32), (40, 16), (128, 128)])
def test_channels_of_very_different_size(device, dtype, queries, dim, block):
    """A few channels 64 to 4096 times larger than the others, which keep their own precision."""
    keys, keep = 8 * block - 5, 4
    q, k, v = _inputs(queries + dim, dtype, queries, keys, dim=dim)
    sizes = torch.full((dim,), 2.0**-4)
    sizes[3], sizes[dim // 2], sizes[dim - 1], sizes[1] = 4.0, 32.0, 256.0, 2.0**-10
    v = (v.float() * sizes.cuda()).to(dtype)
    ids = _ids(queries, 2, 8, keep, queries)
    got = _f64(tokens.block_attention(q, k, v, ids, block))
    see = ot.seen(ids.cpu().numpy(), keys, block, np.ones((1, keys), bool))
    want, size = _attention(q, k, v, see, dim**-0.5)
    # float16 has no finer spacing than 2^-24 below 2^-14
    bound = (3 * U[dtype] + 5e-4) * size + (2.0**-24 if dtype == torch.float16 else 0)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,heads,dim,block", [(5, 4, 64, 32), (250, 2, 40, 16), (255, 4, 128, 128), (90, 260, 8, 32)])
def test_values_that_are_not_finite_stay_in_their_channel(device, dtype, causal, queries, heads, dim, block):
    """An infinity or NaN reaches the channel it is in, of the rows that see its key; a key behind the query
    shares a block with keys before it and may hold anything."""
    keys, blocks = 256, 256 // block
    q, k, v = _inputs(queries + dim, dtype, queries, keys, heads, 2, dim)
    start = keys - queries - 1
    keep = max(1, blocks // 2)
    ids = _ids(queries, 2, blocks, keep, 5)
    ids[..., -1] = blocks - 1  # the block that holds the last keys, in every row
    odd = torch.zeros(1, keys, 2, dim)
    odd[0, keys - 3, :, 1], odd[0, keys - 2, 0, 2], odd[0, keys - 1, 1, 2] = float("inf"), float("-inf"), float("nan")
    odd[0, keys - 4, 0, 5], odd[0, keys - 2, 0, 5], odd[0, 40, 1, 7] = float("inf"), float("-inf"), float("-inf")
    v = torch.where(odd == 0, v.cpu(), odd.to(dtype)).cuda()
    got = tokens.block_attention(q, k, v, ids, block, causal=causal, start=start)
    see = ot.seen(ids.cpu().numpy(), keys, block, np.ones((1, keys), bool), causal=causal, start=np.array([start]))
    want, size = _attention(q, k, torch.where(odd.cuda() == 0, v, 0), see, dim**-0.5)
    # what a row sees of the odd ones adds up to an infinity or NaN, or to 0
    group = heads // 2
    with np.errstate(invalid="ignore"):
        poison = np.zeros((1, queries, 2, dim))
        for _, key, head, channel in np.argwhere(odd.numpy() != 0):
            poison[:, :, head, channel] += np.where(see[:, :, head, key], odd[0, key, head, channel].item(), 0)
    poison = poison.repeat(group, 2)
    got = _f64(got)
    assert np.array_equal(got[poison != 0], poison[poison != 0], equal_nan=True)
    assert (poison != 0).any() and (poison == 0).any()
    clean = poison == 0
    assert (np.abs(got - want)[clean] <= (3 * U[dtype] + 5e-4) * size[clean]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [3, 700])
@pytest.mark.parametrize("block,keep", [(16, 30), (64, 7), (128, 3)])
def test_values_at_the_end_of_their_type(device, dtype, queries, block, keep):
    """Sums of such values pass the type's range, and float32's, on the way to a mean within it."""
    blocks = keep + 1
    keys = blocks * block - 3
    q, k, v = _inputs(queries + block, dtype, queries, keys)
    top = 65504.0 if dtype == torch.float16 else 3.38e38
    v = ((0.5 + 0.5 * torch.rand(v.shape, generator=torch.Generator().manual_seed(2))) * top).to(dtype).cuda()
    v[..., 1::2] *= -1
    ids = _ids(queries, 2, blocks, keep, 6)
    for size_of_k in (0, 1):
        got = tokens.block_attention(q, k * size_of_k, v, ids, block)
        see = ot.seen(ids.cpu().numpy(), keys, block, np.ones((1, keys), bool))
        want, size = _attention(q, k * size_of_k, v, see, 64**-0.5)
        assert torch.isfinite(got).all()
        assert (np.abs(_f64(got) - want) <= (3 * U[dtype] + 5e-4) * size).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("queries", [6, 900])
@pytest.mark.parametrize("dim,block", [(64, 64), (80, 16), (128, 32)])
def test_no_rounding_but_the_results_own(device, dtype, queries, dim, block):
    """The distance to float64 is that of the float64 result rounded once: rounding errors are independent
    and add in squares, and bfloat16's partials, an eighth of its unit, add less than a hundredth; float32
    sums and exponents add some 1e-6 of the size of the terms."""
    blocks, keep = 12, 5
    keys = blocks * block - 7
    q, k, v = _inputs(queries + dim + block, dtype, queries, keys, dim=dim)
    ids = _ids(queries, 2, blocks, keep, 7)
    got = _f64(tokens.block_attention(q, k, v, ids, block))
    see = ot.seen(ids.cpu().numpy(), keys, block, np.ones((1, keys), bool))
    want, size = _attention(q, k, v, see, dim**-0.5)
    once = _f64(torch.from_numpy(want).to(dtype)) - want
    assert np.linalg.norm(got - want) <= 1.05 * np.linalg.norm(once) + 1e-5 * np.linalg.norm(size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [2, 400])
def test_a_query_without_keys_gets_zeros_whatever_it_holds(device, dtype, queries):
    """Rows of infinities and NaN over blocks of masked keys: zeros, as any row that sees nothing."""
    q, k, v = _inputs(queries, dtype, queries, 200)
    q[0, 0, 0], q[0, 1, 1, 3], q[0, 1, 2] = float("inf"), float("nan"), float("-inf")
    mask = torch.zeros(1, 200, dtype=torch.bool, device="cuda")
    mask[0, 32:64] = True
    ids = torch.tensor([0, 3, 6], dtype=torch.int32).expand(1, queries, 2, 3).contiguous().cuda()
    for args in (dict(key_mask=mask), dict(lengths=torch.zeros(1, dtype=torch.int32, device="cuda")),
                 dict(key_mask=mask, causal=True, start=3)):
        assert not tokens.block_attention(q, k, v, ids, 32, **args).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_many_items_of_few_queries(device, dtype):
    """Single tokens of many items: more pairs than blocks of one item, fewer than all blocks, in more than
    one launch."""
    batch, keys, heads, kv_heads, dim, block, keep = 40, 300 * 16, 64, 4, 128, 16, 130
    gen = torch.Generator(device="cuda").manual_seed(11)
    q, k, v = (torch.randn(batch, n, h, dim, generator=gen, device="cuda").to(dtype)
               for n, h in ((1, heads), (keys, kv_heads), (keys, kv_heads)))
    lengths = torch.arange(batch, dtype=torch.int32, device="cuda") * (keys // batch) + 5
    ids = torch.rand(batch, 1, kv_heads, 300, generator=gen, device="cuda").topk(keep).indices.sort(-1).values.to(torch.int32)
    got = tokens.block_attention(q, k, v, ids, block, lengths=lengths)
    for item in (0, 1, 19, 20, 21, 39):
        one = slice(item, item + 1)
        valid = np.arange(keys)[None] < int(lengths[item])
        see = ot.seen(ids[one].cpu().numpy(), keys, block, valid)
        want, size = _attention(q[one], k[one], v[one], see, dim**-0.5)
        assert (np.abs(_f64(got[one]) - want) <= (3 * U[dtype] + 5e-4) * size).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [3, 800])
def test_blocks_that_count_alike_at_any_logit(device, dtype, queries):
    """Equal keys under logits of tens of thousands: every key counts the same however many its block has, so
    the result is the mean of the values seen.  A sum of a block's, then the blocks', and a division err by at
    most one unit of 2^-24 a term (bfloat16's l and partials by 2^-16 and 2^-12), the result by U."""
    block, blocks, keep = 32, 9, 6
    keys = blocks * block - 11
    _, _, v = _inputs(queries, dtype, queries, keys)
    k = torch.ones(1, keys, 2, 64, dtype=dtype, device="cuda")
    q = (1.0 + torch.arange(queries, device="cuda").remainder(100) / 128).to(dtype)[None, :, None, None].expand(1, queries, 4, 64).contiguous()
    mask = torch.rand(1, keys, generator=torch.Generator().manual_seed(8)) < 0.6
    ids = _ids(queries, 2, blocks, keep, 9)
    see = ot.seen(ids.cpu().numpy(), keys, block, mask.numpy())
    for scale in (1e-3, 777.7, -7919.0):
        got = _f64(tokens.block_attention(q, k, v, ids, block, scale=scale, key_mask=mask.cuda()))
        want, size = _attention(torch.zeros_like(q), k, v, see, 1.0)
        bound = U[dtype] + (block + keep + 4) * 2.0**-24 + (2.0**-12 + 2.0**-16 if dtype == torch.bfloat16 else 0)
        assert (np.abs(got - want) <= bound * size).all()


@pytest.mark.parametrize("dim", [96, 128])
@pytest.mark.parametrize("queries", [2, 700])
def test_logits_whose_channels_cancel(device, dim, queries):
    """float32 logits are summed 32 channels at a time: what small channels add up to is not lost to large ones
    that cancel in the end.  The small ones, 1 or 3 each, add up to even numbers, which 2^24 can hold beside
    it, so the logits are exact."""
    keys, block = 200, 64
    gen = torch.Generator().manual_seed(dim)
    q, k = torch.zeros(1, queries, 4, dim), torch.zeros(1, keys, 2, dim)
    q[..., 0], q[..., dim - 1], k[..., 0], k[..., dim - 1] = 2.0**12, -(2.0**12), 2.0**12, 2.0**12
    q[..., 32:64] = 1.0 + 2 * torch.randint(0, 2, (1, queries, 4, 1), generator=gen)
    k[..., 32:63] = torch.randint(0, 2, (1, keys, 2, 31), generator=gen).float()
    k[..., 63] = k[..., 32:63].sum(-1) % 2
    v = torch.randn(1, keys, 2, dim, generator=gen)
    ids = _ids(queries, 2, 4, 3, 10)
    got = _f64(tokens.block_attention(q.cuda(), k.cuda(), v.cuda(), ids, block, scale=0.25))
    see = ot.seen(ids.cpu().numpy(), keys, block, np.ones((1, keys), bool))
    want, size = _attention(q, k, v, see, 0.25)
    # exponents of at most 24 log2(e), each a product rounded once, weights and their sums
    assert (np.abs(got - want) <= (64 + 70) * 2.0**-24 * size).all()
