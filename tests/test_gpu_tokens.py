"""The token operators (rotary positions, the norms around a block, attention over selected
blocks) against the float64 oracle.

Tolerances.  U is a type's unit roundoff (half the spacing at 1).  A rotation is two products and
a sum in float32 with cos and sin good to 3e-7, then one rounding: |x| (1e-6 + U).  A norm row is a
few float32 sums (1e-5 of the largest result) and one rounding.  Attention in 16 bits may round the
weights and one partial result to the type's bits before its last rounding, so a row's error stays
below 4 U times the weighted mean of its largest |v|; a float32 logit of up to 130 terms that sum
to less than 20 in magnitude is off by less than 130 * 2^-24 * 20 = 1.6e-4 and a weight by twice
that, 3.2e-4 (worst case; 5e-4 is asked), and rounding errors that do not agree in sign bring the
whole within 3 U + 2e-5 in relative L2.  Kept blocks are whole numbers and compare exactly."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nnunet_mlx.errors import ContractError
from nnunet_mlx.model import tokens
from oracle import tokens as ot

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TYPES = list(U)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def _np32(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy()


# ---- rotary positions -----------------------------------------------------------------

ROTATIONS = [
    # batch, tokens, heads, kv_heads, dim, rotary, axes, scaling
    (1, 1, 5, 5, 64, 60, 3, None),
    (2, 37, 6, 2, 64, 64, 1, None),
    (3, 5, 1, 0, 128, 96, 1, "ramp"),
    (1, 130, 3, 1, 80, 22, 2, "linear"),
    (2, 19, 2, 3, 33, 10, 1, "base"),
    (1, 7, 1, 1, 2, 2, 1, None),
    (1, 3, 2, 0, 1024, 1000, 3, None),
    (1, 3000, 4, 4, 32, 30, 3, None),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("case", ROTATIONS)
def test_rotate(device, case, layout, dtype):
    batch, n, heads, kv, dim, rotary, axes, scaling = case
    gen = _gen(ROTATIONS.index(case))
    q = torch.randn(batch, n, heads, dim, generator=gen).to(dtype).cuda()
    k = torch.randn(batch, n, kv, dim, generator=gen).to(dtype).cuda() if kv else None
    positions = torch.randint(-5, 1 << 20, (batch, n, axes), generator=gen, dtype=torch.int32).cuda()
    plan = tokens.rotary_plan(rotary, axes=axes, scaling=scaling, factor=1.0 if scaling is None else 8.0)
    inverse = n % 2 == 1
    got = tokens.rotate(q, k, positions, plan, layout=layout, inverse=inverse)
    steps = np.array([s % (1 << 64) for s in plan.steps.tolist()], dtype=np.float64) / 2.0**64 * 2 * math.pi
    for x, y in zip((q, k), got):
        if x is None:
            assert y is None
            continue
        want = ot.rotate(_f64(x), positions.cpu().numpy(), steps, plan.axes.cpu().numpy(), plan.amplitude,
                         layout, inverse)
        size = np.abs(want).max(-1, keepdims=True)
        assert (np.abs(_f64(y) - want) <= size * (2e-6 + U[dtype])).all()
        assert torch.equal(y[..., rotary:], x[..., rotary:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotate_strided_in_place_and_shared_positions(device, layout, dtype):
    """Views of one projection at an odd offset, rotated into a new tensor and in place."""
    gen = _gen(5)
    wide = torch.randn(2, 41, 9, 71, generator=gen).to(dtype).cuda()
    q, k = wide[:, :, :4, 3:67], wide[:, :, 4:6, 3:67]
    positions = torch.arange(41, dtype=torch.int32, device="cuda")[:, None]
    plan = tokens.rotary_plan(48)
    want = tokens.rotate(q.contiguous(), k.contiguous(), positions.expand(2, 41, 1), plan, layout=layout)
    got = tokens.rotate(q, k, positions, plan, layout=layout)
    before = wide.clone()
    placed = tokens.rotate(q, k, positions, plan, layout=layout, out=(q, k))
    assert placed[0] is q
    for a, b, c in zip(want, got, placed):
        assert torch.equal(a, b) and torch.equal(a, c)
    untouched = torch.ones_like(wide, dtype=torch.bool)
    untouched[:, :, :6, 3:67] = False
    assert torch.equal(wide[untouched], before[untouched])


def test_rotate_gradient_is_the_inverse_rotation(device):
    """The directional difference of sum(w * rotate(x)) is the product with the inverse rotation of
    w (the map is linear, so a difference over any step is exact up to rounding)."""
    gen = _gen(6)
    x, w, e = (torch.randn(1, 9, 2, 40, generator=gen).cuda() for _ in range(3))
    positions = torch.randint(0, 5000, (9, 1), generator=gen, dtype=torch.int32).cuda()
    plan = tokens.rotary_plan(32, scaling="ramp", factor=2.0)
    turn = lambda z, inv=False: tokens.rotate(z, None, positions, plan, inverse=inv)[0].double()  # noqa: E731
    difference = ((turn(x + e) - turn(x - e)) * w.double()).sum() / 2
    gradient = (turn(w, True) * e.double()).sum()
    assert float(abs(difference - gradient)) <= 1e-4


def test_rotate_offsets_beyond_32_bits(device):
    """A tensor of more than 2^32 bytes and 2^31 elements: its last token is turned like a small one."""
    n = (1 << 31) // (16 * 128) + 3
    x = torch.zeros(1, n, 16, 128, dtype=torch.bfloat16, device="cuda")
    x[0, -2:] = torch.randn(2, 16, 128, generator=_gen(7)).to(torch.bfloat16).cuda()
    positions = torch.arange(n, dtype=torch.int32, device="cuda")[:, None]
    plan = tokens.rotary_plan(128)
    small = tokens.rotate(x[:, -2:].contiguous(), None, positions[-2:].contiguous(), plan)[0]
    tokens.rotate(x, None, positions, plan, out=(x, None))
    assert torch.equal(x[:, -2:], small) and not x[0, :-2].any()


# ---- norms ----------------------------------------------------------------------------

NORMS = [
    # rows, channels, kind, post, pre, gate, activation, scale, residual_scale, wide residual
    (1, 320, "layer", True, True, False, "none", False, 1.0, False),
    (1, 1, "rms", True, True, True, "silu", True, 0.5, True),
    (3, 1, "layer", True, True, False, "none", False, 1.0, False),
    (5, 33, "rms", True, True, True, "sigmoid", False, 0.8, False),
    (257, 331, "layer", False, True, False, "none", True, 1.0, True),
    (64, 320, "rms", True, False, True, "none", True, 1.0, False),
    (1001, 64, "layer", True, True, True, "silu", True, -0.7, True),
    (2, 1030, "rms", False, True, False, "none", False, 1.0, True),
    (7, 4096, "layer", True, True, True, "sigmoid", True, 1.0, False),
    (3, 16384, "layer", True, True, False, "none", True, 1.0, True),
    (2, 9001, "rms", True, True, True, "none", False, 1.0, False),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", NORMS)
def test_residual_norm(device, case, dtype):
    rows, channels, kind, post, pre, gated, activation, scaled, residual_scale, wide = case
    gen = _gen(rows * 31 + channels)

    def make(*shape):
        return torch.randn(*shape, generator=gen)

    x = (make(rows, channels) * 2 + 0.5).to(dtype).cuda()
    residual = (make(rows, channels) * 3 - 1).to(torch.float32 if wide else dtype).cuda()
    gate = make(rows, channels).to(dtype).cuda() if gated else None
    scale = make(channels).cuda() if scaled else None
    affine = lambda on: (make(channels).cuda(), make(channels).cuda()) if on else None  # noqa: E731
    a_post, a_pre = affine(post), affine(pre)
    total, y = tokens.residual_norm(x, residual, kind=kind, post=a_post, pre=a_pre, gate=gate,
                                    gate_activation=activation, scale=scale, residual_scale=residual_scale,
                                    eps=1e-5)
    n64 = lambda pair: None if pair is None else tuple(map(_f64, pair))  # noqa: E731
    want, want_y = ot.residual_norm(
        _f64(x), _f64(residual), kind=kind, post=n64(a_post), pre=n64(a_pre),
        gate=None if gate is None else _f64(gate), activation=activation,
        scale=None if scale is None else _f64(scale), residual_scale=residual_scale, eps=1e-5)
    assert total.dtype == residual.dtype

    def close(got, expected, kind_of):
        bound = U[kind_of] * np.abs(expected) + 1e-5 * np.abs(expected).max(-1, keepdims=True) + 1e-6
        # one channel: var is 0 and the norm of a value that rounding moved is at most its bias
        assert (np.abs(_f64(got) - expected) <= bound).all()

    close(total, want, total.dtype)
    assert (y is None) == (want_y is None)
    if y is not None:
        if channels == 1 and kind == "layer":
            return  # 0 / sqrt(0 + eps) of values that differ in their last bits
        close(y, want_y, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_residual_norm_strides_and_missing_parts(device, dtype):
    gen = _gen(9)
    wide = torch.randn(4, 6, 3, 101, generator=gen).to(dtype).cuda()
    x, residual = wide[:, :, 0, 1:98], wide[:, :, 2, 3:100]
    total, y = tokens.residual_norm(x, residual, kind="rms", pre=(None, None))
    want, want_y = tokens.residual_norm(x.contiguous(), residual.contiguous(), kind="rms", pre=(None, None))
    assert torch.equal(total, want) and torch.equal(y, want_y)
    alone, y = tokens.residual_norm(x.contiguous(), None, kind="layer", pre=(None, None))
    assert torch.equal(alone, x)
    expected = ot.norm(_f64(x), (None, None), "layer", 1e-6)
    assert (np.abs(_f64(y) - expected) <= U[dtype] * np.abs(expected) + 2e-5 * np.abs(expected).max()).all()
    empty, none = tokens.residual_norm(x[:0], residual[:0], pre=None)
    assert empty.shape == (0, 6, 97) and none is None


def test_residual_norm_of_a_large_mean(device):
    """The variance about a mean a thousand times larger: no cancellation of squares."""
    x = torch.randn(5, 320, generator=_gen(10)) + 1000.0
    _, y = tokens.residual_norm(x.cuda(), None, pre=(None, None), eps=0.0)
    want = ot.norm(_f64(x), (None, None), "layer", 0.0)
    # a value of 1000 holds 6e-5 of absolute rounding against a deviation of 1
    assert np.abs(_f64(y) - want).max() <= 5e-4


# ---- attention over selected blocks ---------------------------------------------------


def _attention_inputs(case, dtype):
    batch, queries, keys, heads, kv, dim, block, *_ = case
    gen = _gen(sum(int(c) << i for i, c in enumerate(case)))
    kinds = torch.randn(6, kv, dim, generator=gen)
    k = kinds[torch.randint(0, 6, (batch, keys // 24 + 1), generator=gen)][:, torch.arange(keys) // 24]
    k = k + 0.7 * torch.randn(batch, keys, kv, dim, generator=gen)
    q = 0.5 * kinds[torch.randint(0, 6, (batch, queries), generator=gen)].repeat_interleave(heads // kv, 2)
    q = q + 0.7 * torch.randn(batch, queries, heads, dim, generator=gen)
    v = torch.randn(batch, keys, kv, dim, generator=gen)
    return q.to(dtype).cuda(), k.to(dtype).cuda(), v.to(dtype).cuda()


# batch, queries, keys, heads, kv_heads, dim, block, keep, first, local, causal, ragged, masked
ATTENTIONS = [
    (1, 1, 1, 1, 1, 8, 16, 1, 0, 0, False, False, False),
    (1, 1, 700, 5, 5, 64, 64, 4, 0, 1, False, False, False),
    (2, 3, 1000, 16, 2, 128, 64, 5, 0, 0, False, True, True),
    (1, 4, 333, 6, 1, 40, 16, 7, 1, 1, False, False, True),
    (2, 300, 300, 5, 5, 64, 64, 3, 0, 1, False, False, True),
    (1, 513, 513, 4, 4, 128, 128, 2, 0, 1, False, False, False),
    (4, 121, 121, 6, 3, 80, 32, 3, 1, 2, True, True, False),
    (1, 200, 450, 3, 1, 32, 16, 9, 0, 1, False, False, False),
    (1, 257, 257, 8, 2, 16, 16, 40, 1, 1, True, False, False),
    (3, 65, 129, 2, 2, 104, 128, 1, 0, 0, False, True, True),
    (1, 90, 640, 12, 1, 48, 32, 6, 0, 0, False, False, False),
    (1, 33, 95, 7, 1, 64, 64, 2, 0, 0, True, False, True),
    (1, 1100, 1100, 1, 1, 64, 16, 12, 0, 1, False, False, False),
]


def _valid_start(case):
    batch, queries, keys, *_, causal, ragged, masked = case
    lengths = [keys] + [max(0, keys - i * (keys // max(1, batch - 1)) - 3) for i in range(1, batch)] \
        if ragged else [keys] * batch
    valid = np.arange(keys)[None, :] < np.array(lengths)[:, None]
    mask = None
    if masked:
        mask = np.random.default_rng(4).random((batch, keys // 20 + 1)).repeat(20, 1)[:, :keys] < 0.5
        valid &= mask
    start = np.array([max(0, keys - queries - 5 * i) for i in range(batch)], np.int32)
    return lengths, mask, valid, start


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", ATTENTIONS)
def test_sparse_attention(device, case, dtype):
    batch, queries, keys, heads, kv, dim, block, keep, first, local, causal, ragged, masked = case
    q, k, v = _attention_inputs(case, dtype)
    lengths, mask, valid, start = _valid_start(case)
    behind = torch.from_numpy(~valid).cuda()
    # what is not valid may hold anything
    k[behind] = float("nan")
    v[behind] = float("inf")
    args = dict(lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                key_mask=None if mask is None else torch.from_numpy(np.ascontiguousarray(mask)).cuda())
    start_gpu = torch.from_numpy(start).cuda()
    summary = tokens.summarize_blocks(k, block, **args)
    codes, scales = ot.summarize(_np32(k), block, valid)
    assert np.array_equal(summary.codes.cpu().numpy(), codes)
    assert np.array_equal(summary.scales.cpu().numpy(), scales)
    ids = tokens.select_blocks(q, summary, block, keep, causal=causal, start=start_gpu, first=first, local=local)
    want_ids = ot.select(_np32(q), codes, scales, block, keep, causal=causal, start=start, first=first,
                         local=local)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    scale = dim**-0.5
    got = tokens.block_attention(q, k, v, ids, block, causal=causal, start=start_gpu, **args)
    see = ot.seen(want_ids, keys, block, valid, causal=causal, start=start)
    want, size = ot.attention(_f64(q), _f64(k), _f64(v), see, scale)
    got = _f64(got)
    assert (got[~see.any(-1).repeat(heads // kv, 2)] == 0).all()
    assert (np.abs(got - want) <= (4 * U[dtype] + 5e-4) * size[..., None]).all()
    assert np.linalg.norm(got - want) <= (3 * U[dtype] + 2e-5) * np.linalg.norm(want)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strides(device, dtype):
    """Queries, keys and values as views of one projection whose rows start at odd places, a
    transposed output, and the same through contiguous copies."""
    gen = _gen(12)
    wide = torch.randn(2, 150, 8, 67, generator=gen).to(dtype).cuda()
    q, k, v = wide[:, :, :4, 1:65], wide[:, :, 4:6, 2:66], wide[:, :, 6:8, 3:67]
    summary = tokens.summarize_blocks(k, 32)
    want = tokens.summarize_blocks(k.contiguous(), 32)
    assert torch.equal(summary.codes, want.codes) and torch.equal(summary.scales, want.scales)
    ids = tokens.select_blocks(q, summary, 32, 3)
    assert torch.equal(ids, tokens.select_blocks(q.contiguous(), want, 32, 3))
    plain = tokens.block_attention(q.contiguous(), k.contiguous(), v.contiguous(), ids, 32)
    turned = torch.full((2, 4, 150, 64), float("nan"), dtype=dtype, device="cuda").transpose(1, 2)
    tokens.block_attention(q, k, v, ids, 32, out=turned)
    assert torch.equal(turned, plain)
    # one key head for all: a broadcast view
    shared = k[:, :, :1].expand(2, 150, 2, 64)
    again = tokens.block_attention(q, shared, shared, ids, 32)
    assert torch.equal(again, tokens.block_attention(q, shared.contiguous(), shared.contiguous(), ids, 32))


def _some_rows_alone(q, k, v, ids, block, rows, dtype):
    """A few of many queries, computed among all and alone."""
    many = tokens.block_attention(q, k, v, ids, block)
    for t in rows:
        alone = tokens.block_attention(q[:, t:t + 1], k, v, ids[:, t:t + 1].contiguous(), block)
        off = (many[:, t:t + 1].double() - alone.double()).abs().max()
        assert float(off) <= (4 * U[dtype] + 5e-4) * float(v.abs().max()), t
    return many


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_cut_into_spans(device, dtype):
    """Partials of more than the workspace holds at once: 40000 queries of three heads to a key head
    that keep 50 blocks."""
    case = (1, 40000, 4000, 6, 2, 64, 16, 50, 0, 0, False, False, False)
    q, k, v = _attention_inputs(case, dtype)
    ids = torch.rand(1, 40000, 2, 250, generator=_gen(50)).topk(50).indices.sort(-1).values.to(torch.int32).cuda()
    many = _some_rows_alone(q, k, v, ids, 16, (0, 1, 9999, 13333, 13334, 26667, 39999), dtype)
    assert torch.equal(many, tokens.block_attention(q, k, v, ids, 16))


def test_as_many_blocks_as_there_may_be(device):
    case = (1, 700, 32768 * 16, 2, 1, 32, 16, 40, 0, 0, False, False, False)
    q, k, v = _attention_inputs(case, torch.float16)
    ids = torch.randint(0, 32768 // 40, (1, 700, 1, 40), generator=_gen(51), dtype=torch.int32)
    ids = (ids + torch.arange(40, dtype=torch.int32) * (32768 // 40)).cuda()
    ids[0, :, 0, 39] = 32767
    _some_rows_alone(q, k, v, ids, 16, (0, 350, 699), torch.float16)


def test_many_heads_to_a_key_head(device):
    case = (1, 9, 300, 200, 2, 40, 32, 3, 0, 0, False, False, False)
    q, k, v = _attention_inputs(case, torch.float16)
    summary = tokens.summarize_blocks(k, 32)
    ids = tokens.select_blocks(q, summary, 32, 3, local=0)
    codes, scales = (a.cpu().numpy() for a in summary)
    assert np.array_equal(ids.cpu().numpy(), ot.select(_np32(q), codes, scales, 32, 3, local=0))
    want, size = ot.attention(_f64(q), _f64(k), _f64(v), ot.seen(ids.cpu().numpy(), 300, 32, np.ones((1, 300), bool)),
                              40**-0.5)
    got = tokens.block_attention(q, k, v, ids, 32)
    assert (np.abs(_f64(got) - want) <= (4 * 2.0**-11 + 5e-4) * size[..., None]).all()


def test_rows_are_the_same_however_many_queries_come_along(device):
    """Selection is independent of what else is computed; so is a float32 result's order of
    magnitude: one query alone and among many agree within the derived float32 error."""
    case = (1, 600, 600, 4, 2, 64, 32, 6, 0, 0, False, False, False)
    q, k, v = _attention_inputs(case, torch.float32)
    out, ids = tokens.sparse_attention(q, k, v, 32, 6, local=0)
    for t in (0, 311, 599):
        one, one_ids = tokens.sparse_attention(q[:, t:t + 1], k, v, 32, 6, local=0)
        assert torch.equal(one_ids, ids[:, t:t + 1])
        assert float((one - out[:, t:t + 1]).abs().max()) <= 1e-3 * float(v.abs().max())


def test_repeated_calls_are_identical(device):
    case = (2, 300, 300, 5, 5, 64, 64, 3, 0, 1, False, False, True)
    q, k, v = _attention_inputs(case, torch.bfloat16)
    first, ids = tokens.sparse_attention(q, k, v, 64, 3)
    for _ in range(3):
        again, ids2 = tokens.sparse_attention(q, k, v, 64, 3)
        assert torch.equal(first, again) and torch.equal(ids, ids2)


def test_summaries_refreshed_after_appending_keys(device):
    """Keys appended to a cache of capacity 200: refreshing the touched blocks gives the summary of
    the whole."""
    gen = _gen(14)
    k = torch.randn(1, 200, 2, 64, generator=gen).to(torch.bfloat16).cuda()
    lengths = torch.tensor([90], dtype=torch.int32, device="cuda")
    held = tokens.summarize_blocks(k, 16, lengths=lengths)
    lengths.fill_(101)
    tokens.summarize_blocks(k, 16, lengths=lengths, first=90 // 16, count=100 // 16 - 90 // 16 + 1, out=held)
    whole = tokens.summarize_blocks(k, 16, lengths=lengths)
    assert torch.equal(held.codes, whole.codes) and torch.equal(held.scales, whole.scales)


def test_summaries_of_extreme_keys(device):
    """Zeros, subnormals, infinities and NaN among valid keys, and the largest float16 values."""
    k = torch.zeros(1, 64, 1, 16)
    k[0, 16:32] = 1e-30
    k[0, 32:48] = torch.randn(16, 1, 16, generator=_gen(15))
    k[0, 35, 0, 3], k[0, 40, 0, 5] = float("inf"), float("nan")
    k[0, 48:] = 65504.0
    got = tokens.summarize_blocks(k.cuda(), 16)
    codes, scales = ot.summarize(k.numpy(), 16, np.ones((1, 64), bool))
    assert np.array_equal(got.codes.cpu().numpy(), codes) and np.array_equal(got.scales.cpu().numpy(), scales)
    assert scales[0, 0].tolist()[:2] == [0.0, 0.0]


def test_selection_ties_and_zero_queries(device):
    """Equal scores go to the lowest blocks, also through a query of zeros and of NaN."""
    k = torch.randn(1, 16, 2, 32, generator=_gen(16)).repeat(1, 20, 1, 1).cuda()
    summary = tokens.summarize_blocks(k, 16)
    q = torch.randn(1, 4, 4, 32, generator=_gen(17)).cuda()
    q[0, 1] = 0
    q[0, 2] = float("nan")
    ids = tokens.select_blocks(q, summary, 16, 5, local=0)
    assert ids.tolist() == [[[[0, 1, 2, 3, 4]] * 2] * 4]


@pytest.mark.parametrize("keys,block,keep", [(32768 * 16, 16, 256), (70000, 16, 33), (9000, 128, 200)])
def test_selection_over_many_blocks(device, keys, block, keep):
    blocks = -(-keys // block)
    gen = _gen(18)
    codes = torch.randint(-127, 128, (1, 1, blocks, 32), generator=gen, dtype=torch.int8)
    scales = torch.rand(1, 1, blocks, generator=gen)
    scales[0, 0, 5] = -1
    q = torch.randn(1, 9, 2, 32, generator=gen)
    start = torch.tensor([keys - 9], dtype=torch.int32)
    got = tokens.select_blocks(q.cuda(), tokens.BlockSummary(codes.cuda(), scales.cuda()), block, keep,
                               start=start.cuda(), first=2, local=2, causal=True)
    want = ot.select(q.numpy(), codes.numpy(), scales.numpy(), block, keep, start=start.numpy(), first=2,
                     local=2, causal=True)
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("levels", [2, 7, 127])
@pytest.mark.parametrize("blocks,keep,first,local", [
    (3, 2, 0, 1), (64, 64, 1, 1), (65, 17, 0, 0), (200, 128, 0, 3), (256, 1, 0, 0), (257, 129, 2, 1),
    (512, 32, 0, 1), (700, 256, 5, 70), (1500, 100, 90, 90), (2048, 128, 0, 1), (2100, 40, 1, 2), (130, 20, 30, 0)])
def test_selection_with_equal_scores(device, blocks, keep, first, local, levels):
    """Scores of few values, so that cuts fall between equals, among empty blocks, more forced blocks than
    are kept, and queries before the first key and behind the last."""
    gen = _gen(blocks + keep + levels)
    codes = torch.randint(0, levels, (1, 2, blocks, 40), generator=gen, dtype=torch.int8)
    codes[..., 3:] = 0
    scales = torch.randint(0, 3, (1, 2, blocks), generator=gen).float() * 0.5
    scales[torch.rand(1, 2, blocks, generator=gen) < 0.1] = -1
    q = torch.randint(-1, 2, (1, 21, 6, 40), generator=gen).float()
    q[0, 5] = 0
    for causal, begin in ((False, -3), (True, -3), (True, blocks * 16 - 9), (False, blocks * 16 + 50)):
        start = torch.tensor([begin], dtype=torch.int32)
        got = tokens.select_blocks(q.cuda(), tokens.BlockSummary(codes.cuda(), scales.cuda()), 16, keep,
                                   start=start.cuda(), first=first, local=local, causal=causal)
        want = ot.select(q.numpy(), codes.numpy(), scales.numpy(), 16, keep, start=start.numpy(), first=first,
                         local=local, causal=causal)
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("dim,heads", [(40, 6), (128, 20)])
@pytest.mark.parametrize("blocks,keep,first,local", [
    (255, 9, 1, 1), (256, 128, 0, 1), (257, 129, 2, 1), (512, 32, 0, 1), (700, 256, 5, 70), (1500, 100, 90, 90),
    (2048, 128, 0, 1), (2100, 40, 1, 2), (4096, 20, 0, 0), (4099, 130, 1, 40), (8192, 64, 30, 1), (8200, 7, 1, 1)])
def test_selection_alone_and_among_many(device, blocks, keep, first, local, dim, heads):
    """Scores formed by parts for few queries and by whole rows for many: both as the formulas', among equals."""
    gen = _gen(blocks + keep + dim)
    codes = torch.randint(-9, 10, (1, 2, blocks, dim), generator=gen, dtype=torch.int8)
    codes[..., 5:-1] = 0
    scales = torch.randint(0, 9, (1, 2, blocks), generator=gen).float() * 0.5
    scales[torch.rand(1, 2, blocks, generator=gen) < 0.1] = -1
    q = torch.randint(-2, 3, (1, 1100, heads, dim), generator=gen).float()
    summary = tokens.BlockSummary(codes.cuda(), scales.cuda())
    for causal in (False, True):
        begin = blocks * 16 - 900
        start = torch.tensor([begin], dtype=torch.int32)
        args = dict(first=first, local=local, causal=causal)
        many = tokens.select_blocks(q.cuda(), summary, 16, keep, start=start.cuda(), **args)
        for t in (0, 3, 517, 1083):
            few = tokens.select_blocks(q[:, t:t + 17].cuda(), summary, 16, keep, start=begin + t, **args)
            assert torch.equal(few, many[:, t:t + 17])
        want = ot.select(q[:, 517:522].numpy(), codes.numpy(), scales.numpy(), 16, keep,
                         start=np.array([begin + 517]), **args)
        assert np.array_equal(many[:, 517:522].cpu().numpy(), want)


@pytest.mark.parametrize("blocks", [60, 200, 300, 2500, 9000])
@pytest.mark.parametrize("queries", [3, 2100])
def test_selection_of_scores_that_overflow(device, blocks, queries):
    gen = _gen(blocks)
    codes = torch.randint(-127, 128, (1, 1, blocks, 32), generator=gen, dtype=torch.int8)
    scales = torch.rand(1, 1, blocks, generator=gen) * 100
    scales[torch.rand(1, 1, blocks, generator=gen) < 0.5] = -1
    q = torch.randn(1, queries, 2, 32, generator=gen).sign() * torch.tensor([1e37, 1.0])[None, None, :, None]
    q[0, 1] = 1e38
    start = torch.tensor([blocks * 16 - 40], dtype=torch.int32)
    got = tokens.select_blocks(q.cuda(), tokens.BlockSummary(codes.cuda(), scales.cuda()), 16, 20,
                               start=start.cuda(), first=3, local=2)
    want = ot.select(q[:, :3].numpy(), codes.numpy(), scales.numpy(), 16, 20, start=start.numpy(), first=3, local=2)
    assert np.array_equal(got[:, :3].cpu().numpy(), want)


def test_attention_skips_entries_that_are_no_blocks(device):
    case = (1, 70, 100, 2, 2, 64, 32, 4, 0, 0, False, False, False)
    q, k, v = _attention_inputs(case, torch.float16)
    ids = torch.tensor([3, -1, 0, -1], dtype=torch.int32).expand(1, 70, 2, 4).contiguous().cuda()
    odd = torch.tensor([4, 3, 0, -(1 << 31)], dtype=torch.int32).expand(1, 70, 2, 4).contiguous().cuda()
    far = torch.tensor([(1 << 31) - 1, 0, 3, 77], dtype=torch.int32).expand(1, 70, 2, 4).contiguous().cuda()
    want, size = ot.attention(_f64(q), _f64(k), _f64(v), ot.seen(ids.cpu().numpy(), 100, 32, np.ones((1, 100), bool)),
                              0.125)
    for listed in (ids, odd, far):
        got = tokens.block_attention(q, k, v, listed, 32)
        assert (np.abs(_f64(got) - want) <= (4 * 2.0**-11 + 5e-4) * size[..., None]).all()
    none = torch.full((1, 70, 2, 4), -1, dtype=torch.int32, device="cuda")
    assert not tokens.block_attention(q, k, v, none, 32).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [3, 400])
def test_attention_of_values_that_are_not_finite(device, dtype, queries):
    """NaN among the values that a query weighs makes its row NaN; rows that do not keep the block are
    untouched.  A negative scale turns the order of the weights, a scale of 0 makes them equal."""
    case = (1, queries, 200, 2, 1, 64, 32, 2, 0, 0, False, False, False)
    q, k, v = _attention_inputs(case, dtype)
    ids = torch.tensor([[1, 4], [2, 5]], dtype=torch.int32).repeat(queries // 2 + 1, 1)[:queries]
    ids = ids.reshape(1, queries, 1, 2).contiguous().cuda()
    plain = {scale: tokens.block_attention(q, k, v, ids, 32, scale=scale) for scale in (0.125, -0.125, 0.0)}
    see = ot.seen(ids.cpu().numpy(), 200, 32, np.ones((1, 200), bool))
    for scale, got in plain.items():
        want, size = ot.attention(_f64(q), _f64(k), _f64(v), see, scale)
        assert (np.abs(_f64(got) - want) <= (4 * U[dtype] + 5e-4) * size[..., None]).all()
    v[0, 40, 0, 3] = float("nan")
    got = tokens.block_attention(q, k, v, ids, 32)
    assert torch.isnan(got[0, 0::2, :, 3]).all()
    assert torch.equal(got[0, 1::2], plain[0.125][0, 1::2])


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_with_extreme_values(device, dtype):
    """Logits of thousands (one key takes all) and values at the type's range."""
    top = 60000.0 if dtype == torch.float16 else 1e30
    gen = _gen(19)
    q = (torch.randn(1, 40, 2, 64, generator=gen) * 30).to(dtype).cuda()
    k = (torch.randn(1, 64, 2, 64, generator=gen) * 30).to(dtype).cuda()
    v = (torch.randn(1, 64, 2, 64, generator=gen).clamp(-1, 1) * top).to(dtype).cuda()
    ids = torch.tensor([0, 1], dtype=torch.int32).expand(1, 40, 2, 2).contiguous().cuda()
    for queries in (slice(0, 40), slice(7, 8)):
        got = tokens.block_attention(q[:, queries], k, v, ids[:, queries].contiguous(), 32)
        assert torch.isfinite(got).all()
        # float32 logits of some 10^4 are off by 10^4 * 2^-24 * 130 at worst: weights by 0.08
        best = (q[:, queries].double().transpose(1, 2) @ k.double().transpose(1, 2).transpose(2, 3).contiguous()) / 8
        lead = best.topk(2, -1).values
        sure = (lead[..., 0] - lead[..., 1] > 20).cpu()
        at = best.argmax(-1)
        want = torch.gather(v.double().transpose(1, 2), 2, at[..., None].expand(-1, -1, -1, 64)).cpu()
        off = (got.double().transpose(1, 2).cpu() - want).abs().amax(-1)[sure]
        assert sure.any() and float(off.max()) <= 3 * U[dtype] * top + 1e-6 * top


def test_key_offsets_beyond_32_bits(device):
    """A cache of more than 2^31 elements: its last blocks answer like a small cache of them."""
    keys = (1 << 31) // (8 * 128) + 640
    keys -= keys % 64
    k = torch.zeros(1, keys, 8, 128, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    tail = torch.randn(2, 1, 128, 8, 128, generator=_gen(20)).to(torch.float16).cuda()
    k[:, -128:], v[:, -128:] = tail[0], tail[1]
    q = torch.randn(1, 2, 8, 128, generator=_gen(21)).to(torch.float16).cuda()
    block = 128
    n = -(-keys // block)
    ids = torch.tensor([n - 2, n - 1], dtype=torch.int32).expand(1, 2, 8, 2).contiguous().cuda()
    got = tokens.block_attention(q, k, v, ids, block)
    at = (n - 2) * block
    small = torch.tensor([0, 1], dtype=torch.int32).expand(1, 2, 8, 2).contiguous().cuda()
    want = tokens.block_attention(q, k[:, at:].contiguous(), v[:, at:].contiguous(), small, block)
    assert torch.equal(got, want)
    summary = tokens.summarize_blocks(k, block, lengths=torch.tensor([keys], dtype=torch.int32, device="cuda"))
    part = tokens.summarize_blocks(k[:, at:].contiguous(), block)
    assert torch.equal(summary.codes[:, :, n - 2:], part.codes)


def test_on_another_stream(device):
    """The work runs on the current stream: inputs made there are seen without synchronisation."""
    side = torch.cuda.Stream()
    case = (1, 200, 200, 4, 2, 64, 32, 4, 0, 1, False, False, False)
    q, k, v = _attention_inputs(case, torch.float16)
    want, _ = tokens.sparse_attention(q, k, v, 32, 4)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        q2, k2, v2 = (torch.zeros_like(a).add_(a) for a in (q, k, v))
        got, _ = tokens.sparse_attention(q2, k2, v2, 32, 4)
    side.synchronize()
    assert torch.equal(got, want)


def test_graph_replays(device):
    """Captured once with its rotation and norm and replayed on new inputs, with eager work between."""
    case = (1, 300, 300, 4, 2, 64, 32, 4, 0, 1, False, False, False)
    q, k, v = _attention_inputs(case, torch.float16)
    plan = tokens.rotary_plan(64)
    positions = torch.arange(300, dtype=torch.int32, device="cuda")[:, None].contiguous()

    def step():
        a, b = tokens.rotate(q, k, positions, plan)
        out, ids = tokens.sparse_attention(a, b, v, 32, 4)
        total, y = tokens.residual_norm(out.flatten(2), v.repeat(1, 1, 2, 1).flatten(2), pre=(None, None))
        return out, ids, total, y

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(4):
        q.copy_(torch.randn(q.shape, generator=_gen(30 + seed)))
        v.copy_(torch.randn(v.shape, generator=_gen(40 + seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


# ---- refusals -------------------------------------------------------------------------


def test_refusals(device):
    q = torch.zeros(1, 4, 4, 64, device="cuda")
    k = torch.zeros(1, 40, 2, 64, device="cuda")
    ids = torch.zeros(1, 4, 2, 1, dtype=torch.int32, device="cuda")
    plan = tokens.rotary_plan(64)
    positions = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    summary = tokens.summarize_blocks(k, 16)
    x = torch.zeros(3, 8, device="cuda")
    refused = [
        lambda: tokens.rotate(q[..., ::2], None, positions, plan),
        lambda: tokens.rotate(q, k, positions, plan),
        lambda: tokens.rotate(q, None, positions.long(), plan),
        lambda: tokens.rotate(q, None, positions[:3], plan),
        lambda: tokens.rotate(q, None, positions, plan, layout="pairs"),
        lambda: tokens.rotate(q[..., :32], None, positions, plan),
        lambda: tokens.rotate(q.double(), None, positions, plan),
        lambda: tokens.rotate(q, None, positions, plan, out=(q[:, :2], None)),
        lambda: tokens.rotate(q.cpu(), None, positions, plan),
        lambda: tokens.rotate(q, None, torch.zeros(4, 9, dtype=torch.int32, device="cuda"), plan),
        lambda: tokens.residual_norm(x, x[:2], pre=None),
        lambda: tokens.residual_norm(x, x.half(), pre=None),
        lambda: tokens.residual_norm(x, x, kind="batch"),
        lambda: tokens.residual_norm(x, x, gate_activation="silu"),
        lambda: tokens.residual_norm(x, x, scale=torch.zeros(7, device="cuda")),
        lambda: tokens.residual_norm(x, x, pre=(torch.zeros(8, device="cuda").half(), None)),
        lambda: tokens.residual_norm(x, x, eps=-1.0),
        lambda: tokens.residual_norm(torch.zeros(4, 3, 8, device="cuda").transpose(0, 1), None),
        lambda: tokens.residual_norm(torch.zeros(1, 20000, device="cuda"), None, pre=(None, None)),
        lambda: tokens.summarize_blocks(k, 48),
        lambda: tokens.summarize_blocks(k, 16, first=1),
        lambda: tokens.summarize_blocks(k, 16, first=2, count=2, out=summary),
        lambda: tokens.summarize_blocks(k, 16, first=-1, count=1, out=summary),
        lambda: tokens.summarize_blocks(k[..., :60], 16),
        lambda: tokens.summarize_blocks(k, 16, lengths=torch.zeros(2, dtype=torch.int32, device="cuda")),
        lambda: tokens.summarize_blocks(k, 16, key_mask=torch.zeros(1, 39, dtype=torch.bool, device="cuda")),
        lambda: tokens.select_blocks(q, summary, 16, 0),
        lambda: tokens.select_blocks(q, summary, 16, 257),
        lambda: tokens.select_blocks(q[:, :, :3], summary, 16, 1),
        lambda: tokens.select_blocks(q[..., :32], summary, 16, 1),
        lambda: tokens.select_blocks(q, summary, 16, 1, start=-1),
        lambda: tokens.select_blocks(q, summary, 16, 1, first=-1),
        lambda: tokens.block_attention(q, k, k[:, :39], ids, 16),
        lambda: tokens.block_attention(q, k, k.half(), ids, 16),
        lambda: tokens.block_attention(q, k, k, ids.long(), 16),
        lambda: tokens.block_attention(q, k, k, ids[:, :3], 16),
        lambda: tokens.block_attention(q, k, k, ids, 16, scale=float("nan")),
        lambda: tokens.block_attention(q[..., :60], k[..., :60], k[..., :60], ids, 16),
    ]
    for index, call in enumerate(refused):
        with pytest.raises(ContractError):
            call()
            pytest.fail(f"call {index} was not refused")


def test_empty_calls(device):
    q, k = torch.zeros(1, 0, 4, 64, device="cuda"), torch.zeros(1, 40, 2, 64, device="cuda")
    out, ids = tokens.sparse_attention(q, k, k, 16, 3)
    assert out.shape == q.shape and ids.shape == (1, 0, 2, 3)
    q = torch.ones(1, 5, 4, 64, device="cuda")
    out, ids = tokens.sparse_attention(q, k[:, :0], k[:, :0], 16, 3)
    assert not out.any() and (ids == -1).all()
    plan = tokens.rotary_plan(64)
    assert tokens.rotate(q[:, :0], None, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), plan)[0].shape == (1, 0, 4, 64)
