"""Tokens held in 8 bits against the float64 oracle.

Codes and scales are elementwise float32 steps and compare exactly, and so does what is read back
(one product in float32, one rounding).

Attention, U a type's unit roundoff, u = 2^-24.  A float32 logit of D products is off by at most
(D + 4) u times the sum of their magnitudes; a weight's relative error is that of its own logit plus
that of the others in the softmax's sum, at most twice the largest, plus 4 u for the power of two.  A
bfloat16 result's weights may be held in one float16 operand (half a step of 2^-11: 2^-12), the others'
in two, the second of what the first leaves (2^-12 of 2^-12: u); the sums over n slots are off by at most
n u.  All of this moves an output by its relative size times the
weighted mean of the slots' largest |v|, twice where the weights' sum is off too; then the result is
rounded once.  In relative L2 errors do not agree in sign, and n roundings of one size make sqrt(n) of
them: D in a logit, of the logits' size L, twice in a weight; n in the sums; the weights' operands and 8
more roundings."""

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


def _f64(t):
    return t.detach().double().cpu().numpy()


def _np32(t):
    return t.detach().float().cpu().numpy()


def _int32(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows(seed, *shape):
    """Rows with channels of very different size."""
    gen = _gen(seed)
    return torch.randn(*shape, generator=gen) * torch.exp(torch.randn(shape[-1], generator=gen))


def _filled(batch, slots, kv_heads, dim, seed):
    """Held tokens of arbitrary codes and scales."""
    gen = _gen(seed)
    held = tokens.held_tokens(batch, slots, kv_heads, dim)
    for codes in (held.k_codes, held.v_codes):
        codes.copy_(torch.randint(-128, 128, codes.shape, generator=gen, dtype=torch.int8))
    for scales in (held.k_scales, held.v_scales):
        scales.copy_(torch.rand(scales.shape, generator=gen))
    return held


# ---- holding and reading ----------------------------------------------------------------

HOLDS = [
    # batch, tokens, slots, kv_heads, dim, starts, lengths
    (1, 1, 64, 1, 16, None, None),
    (1, 64, 64, 5, 64, None, None),
    (2, 1, 192, 5, 64, (0, 191), None),
    (3, 70, 192, 2, 80, (0, 1, 122), (70, 0, 33)),
    (2, 131, 256, 1, 128, (63, 64), (1, 131)),
    (4, 65, 128, 3, 32, (-70, -3, 100, 1000), None),  # tokens without a slot
    (2, 200, 320, 2, 112, (5, 66), (500, -3)),  # counts that are none
    (1, 1000, 1024, 1, 48, (17,), None),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", HOLDS)
def test_hold(device, case, dtype):
    batch, n, slots, heads, dim, starts, lengths = case
    seed = HOLDS.index(case)
    wide = _rows(seed, batch, n, 2 * heads + 1, dim + 3).to(dtype).cuda()
    k, v = wide[:, :, :heads, 3:], wide[:, :, heads + 1:, 1:dim + 1]  # views at odd places
    held = _filled(batch, slots, heads, dim, seed)
    want = [_np32(s) if s.dtype == torch.float32 else s.cpu().numpy() for s in held]
    got = tokens.hold_tokens(held, k, v, start=0 if starts is None else _int32(*starts),
                             lengths=None if lengths is None else _int32(*lengths))
    assert got is held
    for side, x in ((0, k), (2, v)):
        codes, scales = ot.hold(_np32(x))
        for b in range(batch):
            for t in range(n if lengths is None else max(0, min(n, lengths[b]))):
                slot = (0 if starts is None else starts[b]) + t
                if not 0 <= slot < slots:
                    continue
                want[side + 1][b, :, slot] = scales[b, t]
                if side:
                    p = slot % 64
                    want[2][b, :, slot // 64, :, 16 * (p // 4 % 4) + 4 * (p // 16) + p % 4] = codes[b, t]
                else:
                    want[0][b, :, slot] = codes[b, t]
    for a, b in zip(held, want):
        assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("dtype", TYPES)
def test_hold_borders(device, dtype):
    """Rows that are zero, tiny, at the end of the type, not finite; half-way values."""
    top = torch.finfo(dtype).max
    x = torch.zeros(1, 12, 1, 16)
    x[0, 1, 0, 3] = 2.0**-61 if dtype != torch.float16 else 0.0
    x[0, 2, 0, :] = torch.arange(16) / 8 - 1
    x[0, 3, 0, :2] = torch.tensor([top, -top])
    x[0, 4, 0, 5] = math.inf
    x[0, 5, 0, 6] = -math.inf
    x[0, 6, 0, 7] = math.nan
    x[0, 7, 0, :] = torch.tensor([127.0] + [i + 0.5 for i in range(15)])
    x[0, 8, 0, :] = -x[0, 7, 0, :]
    x[0, 9, 0, 0] = 2.0**-20
    x[0, 10, 0, 15] = -1.0
    x = x.to(dtype).cuda()
    held = tokens.hold_tokens(tokens.held_tokens(1, 12, 1, 16), x, x)
    codes, scales = ot.hold(_np32(x))
    assert np.array_equal(held.k_codes.cpu().numpy()[0, 0, :12], codes[0, :, 0])
    assert np.array_equal(_np32(held.k_scales)[0, 0, :12], scales[0, :, 0], equal_nan=True)
    k, v = tokens.read_held(held, dtype, count=12)
    assert torch.isnan(k[0, 4:7]).all() and torch.isfinite(k[0, 7:]).all() and torch.isfinite(k[0, :4]).all()
    assert k[0, 7, 0].tolist() == [127.0] + [float(2 * ((i + 1) // 2)) for i in range(15)]
    assert torch.equal(k.nan_to_num(), v.nan_to_num()) and abs(float(k[0, 3, 0, 0])) == top or dtype == torch.float32


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 64, 1, 16), (2, 192, 3, 80), (1, 320, 5, 64), (3, 128, 2, 128)])
def test_read(device, shape, dtype):
    batch, slots, heads, dim = shape
    held = _filled(batch, slots, heads, dim, dim)
    codes = np.arange(64)
    place = 16 * (codes // 4 % 4) + 4 * (codes // 16) + codes % 4
    values = held.v_codes.cpu()[..., place].transpose(3, 4).reshape(batch, heads, slots, dim)
    want = [(c.float() * s[..., None]).transpose(1, 2).to(dtype)
            for c, s in ((held.k_codes.cpu(), held.k_scales.cpu()), (values, held.v_scales.cpu()))]
    for first, count in ((0, None), (0, 1), (slots - 1, 1), (5, 50), (63, 1), (0, 0), (slots, None)):
        got = tokens.read_held(held, dtype, first=first, count=count)
        for a, b in zip(got, want):
            assert torch.equal(a.cpu(), b[:, first:] if count is None else b[:, first:first + count])
    wide = torch.full((batch, slots, 2 * heads, dim + 5), 7.0, dtype=dtype, device="cuda")
    out = (wide[:, 3:45, :heads, 2:dim + 2], wide[:, 3:45, heads:, 5:])
    assert tokens.read_held(held, dtype, first=9, count=42, out=out)[0] is out[0]
    for a, b in zip(out, want):
        assert torch.equal(a.cpu(), b[:, 9:51])
    untouched = torch.ones_like(wide, dtype=torch.bool)
    untouched[:, 3:45, :heads, 2:dim + 2] = False
    untouched[:, 3:45, heads:, 5:] = False
    assert (wide[untouched] == 7).all()


# ---- attention --------------------------------------------------------------------------


def _attend_check(q, held, n, dtype, *, lengths, scale=None, causal=False, start=None, mask=None, got=None):
    """Against float64 on what the held tokens stand for."""
    batch, queries, heads, dim = q.shape
    k, v = (_f64(x) for x in tokens.read_held(held, torch.float32, count=n))
    see = np.zeros((batch, queries, held.k_codes.shape[1], n), bool)
    for b in range(batch):
        see[b, :, :, :max(0, min(n, lengths[b]))] = True
        if mask is not None:
            see[b] &= mask[b].cpu().numpy()[None, None, :n]
        if causal:
            at = (0 if start is None else start[b]) + np.arange(queries)
            see[b] &= (np.arange(n)[None, :] <= at[:, None])[:, None, :]
    factor = dim**-0.5 if scale is None else scale
    want, size = ot.attention(_f64(q), np.where(see.any((1, 2))[..., None, None], k, 0),
                              np.where(see.any((1, 2))[..., None, None], v, 0), see, factor)
    group = heads // see.shape[2]
    k = np.where(np.isfinite(k), k, 0)
    span = np.abs(_f64(q)).reshape(batch, queries, -1, group, dim).swapaxes(1, 2).reshape(batch, -1, queries * group, dim) \
        @ np.abs(k).transpose(0, 2, 3, 1) if n else np.zeros((batch, see.shape[2], queries * group, 1))
    largest = span.max(-1).reshape(batch, -1, queries, group).swapaxes(1, 2).reshape(batch, queries, heads)
    u = 2.0**-24
    operands = 2.0**-12 if dtype == torch.bfloat16 else u
    weight = 2 * ((dim + 4) * u * largest * abs(factor) + 4 * u) + operands
    bound = U[dtype] * np.abs(want) + (size * (2 * weight + 2 * n * u))[..., None] + 1e-30
    # what lies past the type's end, whichever way its bound takes it, is infinite; at the end either is right
    end, got = float(torch.finfo(dtype).max), _f64(got)
    past, inside = np.abs(want) - bound > end * (1 + 2 * U[dtype]), np.abs(want) + bound <= end
    assert (got[past] == np.sign(want[past]) * np.inf).all()
    got, want, bound = got[inside], want[inside], bound[inside]
    off = np.abs(got - want)
    assert (off <= bound).all(), (off / bound).max()
    if np.linalg.norm(want):
        rel = np.linalg.norm(got - want) / np.linalg.norm(want)
        rows = _f64(q).reshape(batch, queries, -1, group, dim).swapaxes(1, 2).reshape(batch, -1, queries * group, dim)
        logit = np.abs(rows @ k.transpose(0, 2, 3, 1)).max() * abs(factor)
        most = U[dtype] + operands + (2 * dim**0.5 * logit + n**0.5 + 8) * u
        assert rel <= most, (rel, most)


def _held(batch, n, kv_heads, dim, seed):
    gen = _gen(seed)
    slots = -(-n // 64) * 64 + 64
    k, v = (torch.randn(batch, n, kv_heads, dim, generator=gen).cuda() for _ in range(2))
    return tokens.hold_tokens(tokens.held_tokens(batch, slots, kv_heads, dim), k, v)


ATTENDS = [
    # batch, queries, n, heads, kv_heads, dim, causal, lengths, starts, masked, scale
    (1, 1, 1, 1, 1, 16, False, None, None, False, None),
    (1, 1, 300, 5, 5, 64, False, None, None, False, None),
    (2, 3, 65, 6, 2, 80, False, (65, 0), None, False, None),
    (2, 7, 130, 4, 4, 32, True, (130, 100), (123, 60), False, None),
    (1, 17, 700, 3, 1, 96, False, None, None, True, None),
    (3, 1, 1000, 16, 2, 128, False, (1000, 1, 513), None, True, 0.3),
    (1, 130, 130, 2, 2, 64, True, None, None, True, None),
    (1, 33, 259, 2, 1, 48, False, None, None, False, -0.11),
    (2, 5, 2000, 12, 1, 112, False, (2000, 1999), None, False, None),
    (1, 100, 64, 1, 1, 64, True, None, (-20,), False, None),
    (2, 1, 4111, 8, 1, 64, True, None, (4000, 4110), False, None),
    (1, 70, 90, 130, 1, 16, False, None, None, False, 0.0),
    (1, 257, 1111, 4, 2, 128, True, None, (854,), False, None),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", ATTENDS)
def test_attention(device, case, dtype):
    batch, queries, n, heads, kv, dim, causal, lengths, starts, masked, scale = case
    seed = ATTENDS.index(case)
    held = _held(batch, n, kv, dim, seed)
    gen = _gen(100 + seed)
    q = torch.randn(batch, queries, heads, dim, generator=gen).to(dtype).cuda()
    mask = None
    if masked:
        mask = (torch.rand(batch, n, generator=gen) < 0.6).cuda()
        mask[0, n // 3:n // 2] = False
    got = tokens.held_attention(q, held, n if lengths is None else _int32(*lengths), causal=causal, scale=scale,
                                start=None if starts is None else _int32(*starts), key_mask=mask)
    _attend_check(q, held, n, dtype, lengths=lengths or (n,) * batch, causal=causal, start=starts, mask=mask, scale=scale,
                  got=got)
    # the same call again, of other strides, into place
    wide = torch.full((batch, heads, queries + 1, dim + 7), 3.0, dtype=dtype, device="cuda")
    views = torch.empty(batch, queries, heads, dim + 9, dtype=dtype, device="cuda")
    views[..., 5:dim + 5] = q
    out = wide.transpose(1, 2)[:, 1:, :, 3:dim + 3]
    again = tokens.held_attention(views[..., 5:dim + 5], held, n if lengths is None else _int32(*lengths), causal=causal,
                                  scale=scale, start=None if starts is None else _int32(*starts), key_mask=mask, out=out)
    assert again is out and torch.equal(out, got)
    assert (wide[:, :, 0] == 3).all() and (wide[..., :3] == 3).all() and (wide[..., dim + 3:] == 3).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 40])
def test_what_is_not_seen(device, dtype, queries):
    """Slots behind the lengths and masked ones hold NaN scales: they do not show."""
    n, lengths = 400, (390, 0, 64, 65)
    held = _held(4, n, 2, 64, 3)
    q = torch.randn(4, queries, 4, 64, generator=_gen(4)).to(dtype).cuda()
    mask = (torch.rand(4, n, generator=_gen(5)) < 0.5).cuda()
    mask[2] = False
    want = tokens.held_attention(q, held, _int32(*lengths), key_mask=mask)
    for b, length in enumerate(lengths):
        hidden = torch.ones(held.k_scales.shape[2], dtype=torch.bool, device="cuda")
        hidden[:length] = ~mask[b, :length]
        for codes, scales in ((held.k_codes, held.k_scales), (held.v_codes, held.v_scales)):
            scales[b].masked_fill_(hidden, math.nan)
        held.k_codes[b].masked_fill_(hidden[:, None], 127)
    q[1:3] = math.nan  # of items that see nothing: zeros whatever the query
    got = tokens.held_attention(q, held, _int32(*lengths), key_mask=mask)
    assert not got[1:3].any()
    assert torch.equal(got[0], want[0]) and torch.equal(got[3], want[3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 40])
def test_not_a_number(device, dtype, queries):
    """A seen key that is NaN makes its rows NaN, a seen value its head; a query its own row."""
    held = _held(2, 200, 2, 32, 6)
    q = torch.randn(2, queries, 4, 32, generator=_gen(7)).to(dtype).cuda()
    want = tokens.held_attention(q, held, 200, causal=True, start=160)
    held.k_scales[0, 1, 170] = math.nan
    got = tokens.held_attention(q, held, 200, causal=True, start=160)
    sees = torch.arange(queries, device="cuda") + 160 >= 170
    assert torch.isnan(got[0, sees][:, 2:]).all()
    assert torch.equal(got[0, ~sees], want[0, ~sees]) and torch.equal(got[1], want[1])
    assert torch.equal(got[0, :, :2], want[0, :, :2])
    held.k_scales[0, 1, 170] = 0.5
    held.v_scales[1, 0, 3] = math.nan
    got = tokens.held_attention(q, held, 200, causal=True, start=160)
    assert torch.isnan(got[1, :, :2]).all() and torch.equal(got[1, :, 2:], want[1, :, 2:])
    held.v_scales[1, 0, 3] = 1.0
    want = tokens.held_attention(q, held, 200)
    for odd in (math.nan, math.inf, -math.inf):
        r = q.clone()
        r[1, queries - 1, 3, 5] = odd
        got = tokens.held_attention(r, held, 200)
        assert torch.isnan(got[1, -1, 3]).all()
        got[1, -1, 3] = want[1, -1, 3]
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("queries", [1, 40])
def test_ends_of_the_type(device, dtype, queries):
    """Values near the type's end, and queries whose products with codes pass it, do not overflow on the way."""
    top = torch.finfo(dtype).max
    gen = _gen(8)
    k = torch.randn(1, 300, 1, 64, generator=gen) * 1e-6
    v = (torch.rand(1, 300, 1, 64, generator=gen) * 0.01 + 0.985) * top
    q = torch.randn(1, queries, 2, 64, generator=gen)
    held = tokens.hold_tokens(tokens.held_tokens(1, 300, 1, 64), k.to(dtype).cuda(), v.to(dtype).cuda())
    got = tokens.held_attention(q.to(dtype).cuda(), held, 300)
    # all between 0.98 and 1 of the end, with weights that hardly differ
    assert ((got.float() / top > 0.97) & (got.float() / top <= 1)).all()
    big = (q * 1e36).to(dtype).cuda()
    k = (k * 1e-30).to(dtype).cuda()  # below 2^-60: held as zero
    held = tokens.hold_tokens(held, k, (v / top).to(dtype).cuda())
    want = tokens.read_held(held, torch.float32, count=300)[1].mean(1, keepdim=True)
    got = tokens.held_attention(big, held, 300)
    assert float((got.float() - want).abs().max()) <= U[dtype] + 1e-4
    k = torch.full((1, 300, 1, 64), 2.0**-58, device="cuda").to(dtype)
    held = tokens.hold_tokens(held, k, (v / top).to(dtype).cuda())
    got = tokens.held_attention(big.abs(), held, 300)  # equal logits of some 1e20
    assert float((got.float() - want).abs().max()) <= U[dtype] + 1e-4


def test_long_softmax(device):
    """One key that outweighs 100000 others, and 100000 equal ones."""
    n = 100001
    k = torch.zeros(1, n, 1, 16, device="cuda")
    v = torch.randn(1, n, 1, 16, generator=_gen(9)).cuda()
    k[0, 77, 0] = 1.0
    held = tokens.hold_tokens(tokens.held_tokens(1, n, 1, 16), k, v)
    for size in (0.0, 1.0, 3.0):
        q = torch.full((1, 1, 1, 16), size, device="cuda")
        got = tokens.held_attention(q, held, n)
        _attend_check(q, held, n, torch.float32, lengths=(n,), got=got)


def test_offsets_beyond_32_bits(device):
    """Items whose codes start past 2^32 bytes, written, read and attended to."""
    slots = (1 << 24) + 64
    held = tokens.held_tokens(3, slots, 1, 128)
    small = tokens.held_tokens(1, 128, 1, 128)
    k, v = (torch.randn(3, 100, 1, 128, generator=_gen(i)).cuda() for i in (10, 11))
    start, lengths = _int32(0, 0, slots - 128), _int32(0, 0, 100)
    tokens.hold_tokens(held, k, v, start=start, lengths=lengths)
    tokens.hold_tokens(small, k[2:], v[2:])
    for a, b in zip(tokens.read_held(held, torch.float32, first=slots - 128, count=100),
                    tokens.read_held(small, torch.float32, count=100)):
        assert torch.equal(a[2:], b) and not a[:2].any()
    assert not held.k_codes[:2].any()
    tokens.hold_tokens(held, k, v, lengths=lengths)
    q = torch.randn(3, 2, 2, 128, generator=_gen(12)).cuda()
    got = tokens.held_attention(q, held, lengths)
    want = tokens.held_attention(q[2:], small, 100)
    assert not got[:2].any() and float((got[2:] - want).abs().max()) <= 1e-5


# ---- calls ------------------------------------------------------------------------------


def test_step_by_step(device):
    """A sequence held one token after another, each attended to: as if it had been held at once."""
    k, v = (torch.randn(2, 90, 3, 32, generator=_gen(i)).cuda() for i in (13, 14))
    q = torch.randn(2, 90, 6, 32, generator=_gen(15)).cuda()
    whole = tokens.hold_tokens(tokens.held_tokens(2, 90, 3, 32), k, v)
    want = tokens.held_attention(q, whole, 90, causal=True)
    held = tokens.held_tokens(2, 90, 3, 32)
    for t in range(90):
        tokens.hold_tokens(held, k[:, t:t + 1], v[:, t:t + 1], start=t)
        got = tokens.held_attention(q[:, t:t + 1], held, t + 1)
        assert float((got - want[:, t:t + 1]).abs().max()) <= 1e-5
    for a, b in zip(held, whole):
        assert torch.equal(a, b)


def test_with_the_block_operators(device):
    """What is held is read back for a selection over blocks: with every block kept it is the same attention."""
    held = _held(1, 500, 2, 64, 16)
    q = torch.randn(1, 6, 4, 64, generator=_gen(17)).cuda()
    k, v = tokens.read_held(held, torch.float32, count=500)
    want, kept = tokens.sparse_attention(q, k, v, 64, 8)
    assert (kept >= 0).all()
    got = tokens.held_attention(q, held, 500)
    assert float((got - want).abs().max()) <= 1e-5


def test_nothing_to_do(device):
    held = tokens.held_tokens(2, 0, 3, 32)
    assert held.k_codes.shape == (2, 3, 0, 32)
    q = torch.randn(2, 4, 3, 32, device="cuda")
    assert not tokens.held_attention(q, held, 0).any()
    held = _held(2, 64, 3, 32, 18)
    assert not tokens.held_attention(q, held, 0).any()
    assert tokens.held_attention(q[:, :0], held, 64).shape == (2, 0, 3, 32)
    before = [t.clone() for t in held]
    none = torch.zeros(2, 0, 3, 32, device="cuda")
    tokens.hold_tokens(held, none, none, start=128)
    for a, b in zip(held, before):
        assert torch.equal(a, b)
    assert tokens.read_held(held, torch.float16, first=3, count=0)[0].shape == (2, 0, 3, 32)


def test_another_stream_and_graphs(device):
    """A step of a point, captured and replayed with other inputs, against the eager one; two graphs that
    share their memory."""
    held = _held(2, 300, 2, 64, 19)
    q = torch.randn(2, 1, 4, 64, generator=_gen(20)).to(torch.bfloat16).cuda()
    k, v = (torch.randn(2, 1, 2, 64, generator=_gen(i)).to(torch.bfloat16).cuda() for i in (21, 22))
    at, lengths = _int32(300, 130), _int32(301, 131)

    def step():
        tokens.hold_tokens(held, k, v, start=at)
        return tokens.held_attention(q, held, lengths), *tokens.read_held(held, torch.bfloat16)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    pool = torch.cuda.graph_pool_handle()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            results = step()
        graphs.append((graph, results))
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=_gen(30 + i)))
        k.copy_(torch.randn(k.shape, generator=_gen(40 + i)))
        at.add_(1)
        lengths.add_(1)
        graph, results = graphs[i % 2]
        graph.replay()
        kept = [r.clone() for r in results]
        torch.cuda.synchronize()
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_repeats(device):
    """The same call gives the same bits."""
    held = _held(2, 3001, 2, 64, 23)
    for queries in (1, 50):
        q = torch.randn(2, queries, 8, 64, generator=_gen(24)).to(torch.bfloat16).cuda()
        want = tokens.held_attention(q, held, 3001)
        for _ in range(5):
            assert torch.equal(tokens.held_attention(q, held, 3001), want)


def test_gradients_are_refused(device):
    held = _held(1, 64, 2, 32, 25)
    q = torch.randn(1, 3, 2, 32, device="cuda", requires_grad=True)
    got = tokens.held_attention(q, held, 64)
    assert torch.equal(got.detach(), tokens.held_attention(q.detach(), held, 64))
    with pytest.raises(ContractError, match="forward only"):
        got.sum().backward()


def test_refusals(device):
    held = _held(2, 64, 2, 32, 26)
    q, k = torch.randn(2, 3, 4, 32, device="cuda"), torch.randn(2, 3, 2, 32, device="cuda")
    bad = [
        lambda: tokens.hold_tokens(held, k, k, start=126),
        lambda: tokens.hold_tokens(held, k, k, start=-1),
        lambda: tokens.hold_tokens(held, k, k.half()),
        lambda: tokens.hold_tokens(held, k, k[:, :2]),
        lambda: tokens.hold_tokens(held, k[:1], k[:1]),
        lambda: tokens.hold_tokens(held, k[..., :16], k[..., :16]),
        lambda: tokens.hold_tokens(held, k.int(), k.int()),
        lambda: tokens.hold_tokens(held, k.cpu(), k.cpu()),
        lambda: tokens.hold_tokens(held, k, k, start=torch.zeros(2, device="cuda", dtype=torch.int64)),
        lambda: tokens.hold_tokens(held, k, k, lengths=torch.zeros(3, device="cuda", dtype=torch.int32)),
        lambda: tokens.hold_tokens(held._replace(v_codes=held.v_codes[..., :32]), k, k),
        lambda: tokens.hold_tokens(held._replace(k_codes=held.k_codes.transpose(1, 2)), k, k),
        lambda: tokens.hold_tokens(tokens.HeldTokens(*(t.expand(2, *t.shape[1:]) for t in _held(1, 64, 2, 32, 1))), k, k),
        lambda: tokens.hold_tokens(tokens.held_tokens(2, 64, 2, 24), k[..., :24], k[..., :24]),
        lambda: tokens.read_held(held, torch.int8),
        lambda: tokens.read_held(held, torch.float32, first=128, count=1),
        lambda: tokens.read_held(held, torch.float32, first=-1),
        lambda: tokens.read_held(held, torch.float32, count=129),
        lambda: tokens.read_held(held, torch.float32, out=(k, k)),
        lambda: tokens.read_held(held, torch.float16, count=3, out=(k, k)),
        lambda: tokens.held_attention(q, held, 129),
        lambda: tokens.held_attention(q, held, -1),
        lambda: tokens.held_attention(q, held, torch.tensor(5)),
        lambda: tokens.held_attention(q[:, :, :3], held, 64),
        lambda: tokens.held_attention(q[:1], held, 64),
        lambda: tokens.held_attention(q, held, 64, scale=math.inf),
        lambda: tokens.held_attention(q, held, 64, key_mask=torch.ones(2, 129, device="cuda", dtype=torch.bool)),
        lambda: tokens.held_attention(q, held, 64, key_mask=torch.ones(2, 64, device="cuda")),
        lambda: tokens.held_attention(q, held, 64, out=q[:, :2]),
        lambda: tokens.held_attention(q, held, 64, start=torch.zeros(2, device="cuda")),
        lambda: tokens.held_attention(q.double(), held, 64),
        lambda: tokens.held_tokens(1, -1, 2, 32),
    ]
    before = [t.clone() for t in held]
    for call in bad:
        with pytest.raises(ContractError):
            call()
    for a, b in zip(held, before):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [(3000, 1, 0, 900, 2999), (0, 0, 0), (5000, 5000), (1,) * 64, (700,) * 65 + (0,)])
def test_items_that_share_the_parts(device, dtype, lengths):
    """Items of very different lengths, whose parts of the work go by what they hold: each as if it were alone."""
    batch, n = len(lengths), 5000
    held = _held(batch, n, 1, 128, 27)
    q = torch.randn(batch, 2, 3, 128, generator=_gen(28)).to(dtype).cuda()
    for causal, start in ((False, None), (True, [max(0, length - 40) for length in lengths])):
        starts = None if start is None else _int32(*start)
        got = tokens.held_attention(q, held, _int32(*lengths), causal=causal, start=starts)
        for b in range(0, batch, 1 if batch < 10 else 13):
            alone = tokens.HeldTokens(*(t[b:b + 1].clone() for t in held))
            _attend_check(q[b:b + 1], alone, n, dtype, lengths=lengths[b:b + 1], causal=causal,
                          start=None if start is None else start[b:b + 1], got=got[b:b + 1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_operands_of_a_weight_belong_together(device, dtype):
    """Of 16 million weights some lie next to half a step of their first operand's type.  Logits below 1 err by less
    than (16 + 4) u, weights by twice that and 4 u, the operands and sums of 8 slots by 10 u: 58 u of the mean
    |v| in all; an operand that is a step off, by 2^-11 / 8, a hundred times that."""
    held = _held(1, 8, 4, 16, 29)
    q = (0.05 * torch.randn(1, 500000, 4, 16, generator=_gen(30))).to(dtype).cuda()
    got = tokens.held_attention(q, held, 8).double()
    k, v = (x.double()[0].permute(1, 2, 0).contiguous() for x in tokens.read_held(held, torch.float32, count=8))
    logits = torch.matmul(q.double()[0].permute(1, 0, 2).contiguous(), k) / 4  # (heads, queries, 8)
    assert float(logits.abs().max()) < 1
    p = torch.softmax(logits, -1)
    want = torch.matmul(p, v.transpose(1, 2).contiguous()).permute(1, 0, 2)
    size = torch.matmul(p, v.abs().amax(1)[..., None])[..., 0].t()[..., None]
    assert bool(((got[0] - want).abs() <= U[dtype] * want.abs() + 58 * 2.0**-24 * size).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_that_others_wrote(device, dtype):
    """Codes and scales may come from elsewhere: -128 is a code, a scale may be negative, values may lie far apart, and
    past float16's end (127 * 1e4 is 20 times that)."""
    held = _filled(2, 128, 2, 48, 31)
    held.v_scales[0] *= -1e4
    held.v_scales[1, :, 60:] *= 2.0**-40
    held.k_scales.mul_(0.01)
    held.k_codes[:, :, 5] = -128
    held.v_codes[..., 7] = -128
    for queries in (1, 37):
        q = torch.randn(2, queries, 4, 48, generator=_gen(32)).to(dtype).cuda()
        _attend_check(q, held, 128, dtype, lengths=(128, 100), got=tokens.held_attention(q, held, _int32(128, 100)))
