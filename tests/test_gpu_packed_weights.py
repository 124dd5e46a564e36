"""Products with 4-bit weights against the float64 oracle.

Codes and scales are elementwise float32 steps and compare exactly; an unpacked weight is one float32
product and one rounding.  A product of K inputs, u = 2^-24, U the type's unit roundoff: the float32 sum
is off by at most (K + 8) u times the sum of its terms' magnitudes, the gate's activation adds 8 u of
its value (its derivative is at most 1.1), and the result is rounded once.  In relative L2 errors do
not agree in sign, and K roundings of a sum's size make sqrt(K) of them: twice that for a product, four
times for a gated one, whose two sums are off, and 10 more roundings."""

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


def _matrix(seed, outputs, inputs, dtype=torch.float32):
    gen = _gen(seed)
    return (torch.randn(outputs, inputs, generator=gen) * torch.exp(torch.randn(outputs, 1, generator=gen))).to(dtype).cuda()


# ---- packing ------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,group", [((1, 1), 32), ((16, 128), 64), ((17, 129), 128), ((5, 300), 32), ((40, 64), 64),
                                         ((33, 257), 64)])
def test_pack(device, shape, group, dtype):
    w = _matrix(sum(shape), shape[0], shape[1] + 3, dtype)[:, 2:-1]
    packed = tokens.pack_weight(w, group)
    codes, scales, stands = ot.pack(_np32(w), group)
    assert packed[2:] == (*shape, group)
    assert np.array_equal(packed.codes.cpu().numpy(), codes)
    assert np.array_equal(packed.scales.cpu().numpy(), scales)
    back = tokens.unpack_weight(packed, torch.float32)
    assert np.array_equal(back.cpu().numpy(), stands.astype(np.float32))
    assert torch.equal(tokens.unpack_weight(packed, dtype), back.to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_pack_borders(device, dtype):
    """Half-way values, zeros, tiny groups, the type's end, what is not finite."""
    w = torch.zeros(2, 256)
    w[0, :16] = torch.tensor([6, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, -6, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5])
    w[0, 32] = 2.0**-61 if dtype != torch.float16 else 0.0
    w[0, 64] = math.inf
    w[0, 97] = math.nan
    w[0, 128:130] = torch.tensor([torch.finfo(dtype).max, -torch.finfo(dtype).max])
    w = w.to(dtype).cuda()
    packed = tokens.pack_weight(w, 32)
    back = tokens.unpack_weight(packed, torch.float32)
    assert back[0, :16].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -6, 0, -1, -1, -2, -2, -4, -4]
    assert not back[0, 16:64].any() and torch.isnan(back[0, 64:128]).all() and not back[1].any()
    assert torch.isfinite(back[0, 128:]).all()
    assert float((back[0, 128] - w[0, 128].float()).abs() / w[0, 128].float()) <= 2.0**-22
    assert not packed.codes[0, 0, 1].any()  # a row of zeros: no signs either


# ---- products -------------------------------------------------------------------------------

PRODUCTS = [
    # rows, inputs, outputs, group, bias, gated, activation
    (1, 1, 1, 32, True, False, "none"),
    (1, 320, 960, 64, True, False, "none"),
    (1, 128, 16, 128, False, True, "silu"),
    (3, 129, 17, 32, False, True, "sigmoid"),
    (16, 1000, 100, 64, False, False, "none"),
    (17, 333, 31, 128, True, True, "none"),
    (37, 1331, 70, 32, True, False, "none"),
    (64, 64, 64, 64, False, True, "silu"),
    (65, 640, 48, 32, False, False, "none"),
    (130, 96, 20, 64, True, True, "silu"),
    (2, 4100, 33, 128, False, False, "none"),
    (300, 257, 129, 128, True, False, "none"),
]


def _check_product(got, x, w, bias, gate, activation, dtype):
    xd, k, u = _f64(x).reshape(-1, x.shape[-1]), x.shape[-1], 2.0**-24
    product = xd @ w.T + (0 if bias is None else _f64(bias))
    off = (k + 8) * u * (np.abs(xd) @ np.abs(w.T) + (0 if bias is None else np.abs(_f64(bias))))
    if gate is not None:
        g = xd @ gate.T
        opened = ot.gated(np.ones_like(g), g, activation)
        slope = 1.1 if activation != "none" else 1.0
        off = off * np.abs(opened) + ((k + 8) * u * (np.abs(xd) @ np.abs(gate.T)) * slope + 8 * u * np.abs(opened)) * \
            (np.abs(product) + off)
        product = product * opened
    got = _f64(got).reshape(product.shape)
    # Below the type's least normal value tiny a result's steps no longer shrink with it: they stay tiny * eps, and a
    # rounding is off by up to half of one, tiny * U (float16: 2^-14 * 2^-11 = 2^-25).  The exact products of 8300 rows
    # by 17 with a gate, rounded to float16 by numpy, already pass U |product| in 4016 places, all of them below 2^-14.
    bound = U[dtype] * np.abs(product) + U[dtype] * torch.finfo(dtype).tiny + off + 1e-30
    assert (np.abs(got - product) <= bound).all(), (np.abs(got - product) / bound).max()
    rel = np.linalg.norm(got - product) / np.linalg.norm(product)
    assert rel <= U[dtype] + ((2 if gate is None else 4) * k**0.5 + 10) * u, rel


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", PRODUCTS)
def test_product(device, case, dtype):
    rows, inputs, outputs, group, with_bias, gated, activation = case
    seed = PRODUCTS.index(case)
    x = torch.randn(rows, inputs + 5, generator=_gen(seed)).to(dtype).cuda()[:, 3:-2]
    w = tokens.pack_weight(_matrix(seed, outputs, inputs) * inputs**-0.5, group)
    gate = tokens.pack_weight(_matrix(50 + seed, outputs, inputs) * inputs**-0.5, group) if gated else None
    bias = torch.randn(outputs, generator=_gen(seed)).cuda() if with_bias else None
    got = tokens.packed_linear(x, w, bias=bias, gate=gate, gate_activation=activation)
    assert got.shape == (rows, outputs) and got.dtype == dtype and got.is_contiguous()
    _check_product(got, x, _f64(tokens.unpack_weight(w, torch.float32)), bias,
                   None if gate is None else _f64(tokens.unpack_weight(gate, torch.float32)), activation, dtype)
    # nor does it matter how rows step
    assert torch.equal(tokens.packed_linear(x.contiguous(), w, bias=bias, gate=gate, gate_activation=activation), got)
    got = tokens.packed_linear(x[None, ::2], w, bias=bias, gate=gate, gate_activation=activation)
    assert got.shape == (1, (rows + 1) // 2, outputs)
    _check_product(got, x[::2], _f64(tokens.unpack_weight(w, torch.float32)), bias,
                   None if gate is None else _f64(tokens.unpack_weight(gate, torch.float32)), activation, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 20, 200])
def test_not_a_number(device, dtype, rows):
    """Of a row or of an output's group: in that row or output alone; of what lies behind a row, nowhere."""
    wide = torch.full((rows, 340), math.nan, dtype=dtype, device="cuda")
    x = wide[:, 4:337]
    x.copy_(torch.randn(rows, 333, generator=_gen(1)))
    m = _matrix(2, 50, 333)
    want = tokens.packed_linear(x, tokens.pack_weight(m))
    assert torch.isfinite(want).all()
    m[7, 300] = math.inf
    got = tokens.packed_linear(x, tokens.pack_weight(m))
    assert torch.isnan(got[:, 7]).all()
    got[:, 7] = want[:, 7]
    assert torch.equal(got, want)
    m[7, 300] = 0.5
    for odd in (math.nan, math.inf):
        x[rows - 1, 332] = odd
        got = tokens.packed_linear(x, tokens.pack_weight(m))
        assert not torch.isfinite(got[-1]).any()
        assert torch.isfinite(got[:-1]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sizes_of_rows(device, dtype):
    """Elements of very different size in one row keep their own precision."""
    x = torch.randn(5, 256, generator=_gen(3)) * 10.0 ** torch.arange(-6, 10).repeat(16)
    x[:, 130:] *= 1e20
    x = x.to(dtype).cuda()
    m = torch.eye(256).cuda()
    w = tokens.pack_weight(m, 32)
    got = tokens.packed_linear(x, w)
    assert float(((got - x).abs() / x.abs()).max()) <= 8 * 2.0**-24 if dtype == torch.float32 else torch.equal(got, x)


def test_offsets_beyond_32_bits(device):
    rows = (1 << 20) + 3
    x = torch.zeros(rows, 2050, dtype=torch.bfloat16, device="cuda")[:, 1:2049]
    x[-3:] = torch.randn(3, 2048, generator=_gen(4)).to(torch.bfloat16).cuda()
    w = tokens.pack_weight(_matrix(5, 40, 2048), 128)
    got = tokens.packed_linear(x, w)
    assert not got[:-3].any()
    _check_product(got[-3:], x[-3:], _f64(tokens.unpack_weight(w, torch.float32)), None, None, "none", torch.bfloat16)


def test_streams_and_graphs(device):
    w, gate = (tokens.pack_weight(_matrix(i, 300, 200), 64) for i in (6, 7))
    x = torch.randn(2, 3, 200, generator=_gen(8)).to(torch.float16).cuda()

    def step():
        return tokens.packed_linear(x, w, gate=gate, gate_activation="silu")

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert got.shape == (2, 3, 300) and torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=_gen(9 + i)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, step())


def test_nothing_to_do(device):
    w = tokens.pack_weight(_matrix(1, 7, 40))
    assert tokens.packed_linear(torch.zeros(0, 40, device="cuda"), w).shape == (0, 7)
    assert tokens.packed_linear(torch.zeros(40, device="cuda"), w).shape == (7,)


def test_gradients_are_refused(device):
    w = tokens.pack_weight(_matrix(1, 7, 40))
    x, bias = (torch.randn(n, device="cuda", requires_grad=True) for n in (40, 7))
    for kw in (dict(x=x), dict(x=x.detach(), bias=bias)):
        got = tokens.packed_linear(kw.pop("x"), w, **kw)
        with pytest.raises(ContractError, match="forward only"):
            got.sum().backward()


def test_refusals(device):
    w, other = tokens.pack_weight(_matrix(1, 30, 200)), tokens.pack_weight(_matrix(1, 30, 200), 32)
    x = torch.randn(4, 200, device="cuda")
    bad = [
        lambda: tokens.pack_weight(x, 48),
        lambda: tokens.pack_weight(x[0]),
        lambda: tokens.pack_weight(x.cpu()),
        lambda: tokens.pack_weight(x.double()),
        lambda: tokens.pack_weight(x.t()),
        lambda: tokens.pack_weight(x[:0]),
        lambda: tokens.pack_weight(x, torch.tensor(32)),
        lambda: tokens.unpack_weight(w, torch.int8),
        lambda: tokens.unpack_weight(w._replace(outputs=33), torch.float32),
        lambda: tokens.packed_linear(x[:, :100], w),
        lambda: tokens.packed_linear(x.double(), w),
        lambda: tokens.packed_linear(x.t(), w),
        lambda: tokens.packed_linear(x.cpu(), w),
        lambda: tokens.packed_linear(x, w, gate=other),
        lambda: tokens.packed_linear(x, w, gate_activation="silu"),
        lambda: tokens.packed_linear(x, w, gate=w, gate_activation="tanh"),
        lambda: tokens.packed_linear(x, w, bias=torch.zeros(31, device="cuda")),
        lambda: tokens.packed_linear(x, w, bias=torch.zeros(30, device="cuda").half()),
        lambda: tokens.packed_linear(x, w._replace(codes=w.codes[:1])),
        lambda: tokens.packed_linear(x, w._replace(scales=w.scales.transpose(1, 2))),
        lambda: tokens.packed_linear(x, w._replace(group=128)),
        lambda: tokens.packed_linear(x, w._replace(inputs=200.0)),
        lambda: tokens.packed_linear(x, w._replace(inputs=torch.tensor(200))),
    ]
    for call in bad:
        with pytest.raises(ContractError):
            call()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 100])
def test_ends_of_the_type(device, dtype, rows):
    """x near its type's end times small weights does not overflow on the way.  Weights of 6 codes' size, all equal:
    each output is the row's sum times the weight, whose float32 sum of 256 errs by less than 256 u."""
    top = torch.finfo(dtype).max
    x = ((torch.rand(rows, 256, generator=_gen(12)) * 0.1 + 0.9) * top).to(dtype).cuda()
    w = tokens.pack_weight(torch.full((40, 256), 2.0**-9, device="cuda"), 128)
    got = tokens.packed_linear(x, w).double()
    want = (x.double().sum(1, keepdim=True) * 2.0**-9).expand(rows, 40)
    assert bool(((got - want).abs() <= (U[dtype] + 258 * 2.0**-24) * want).all())
    assert torch.isfinite(tokens.packed_linear(x, w, gate=w)).logical_not().all()  # the product itself passes the end
    assert torch.isfinite(tokens.packed_linear(x, w, gate=w, gate_activation="sigmoid")).all()


def test_large_matrix(device):
    """More weights than a launch has threads."""
    outputs, inputs = 8192, 600000
    w = torch.zeros(outputs, inputs, dtype=torch.float16, device="cuda")
    w[-1, -40:] = torch.arange(40, device="cuda") / 40
    w[0, 0], w[-2, inputs // 2] = 3.0, -1.0
    packed = tokens.pack_weight(w, 32)
    back = tokens.unpack_weight(packed, torch.float16)
    small = tokens.unpack_weight(tokens.pack_weight(w[-1:, -64:].contiguous(), 32), torch.float16)  # the same groups
    assert torch.equal(back[-1, -64:], small[0])
    assert float(back[0, 0]) == 3.0 and float(back[-2, inputs // 2]) == -1.0
    assert int(torch.count_nonzero(back)) == 2 + int(torch.count_nonzero(small))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", [
    # rows, inputs, outputs, group, bias, gated, activation: enough pieces for waves that take one each
    (1000, 257, 530, 128, True, False, "none"),
    (2100, 333, 250, 64, True, True, "silu"),
    (8300, 31, 17, 32, False, True, "sigmoid"),
    (4161, 128, 130, 32, False, False, "none"),
    (1025, 900, 513, 64, True, True, "none"),
])
def test_many_rows(device, case, dtype):
    rows, inputs, outputs, group, with_bias, gated, activation = case
    x = torch.randn(rows, inputs + 5, generator=_gen(rows)).to(dtype).cuda()[:, 3:-2]
    w = tokens.pack_weight(_matrix(rows, outputs, inputs) * inputs**-0.5, group)
    gate = tokens.pack_weight(_matrix(50 + rows, outputs, inputs) * inputs**-0.5, group) if gated else None
    bias = torch.randn(outputs, generator=_gen(rows)).cuda() if with_bias else None
    got = tokens.packed_linear(x, w, bias=bias, gate=gate, gate_activation=activation)
    _check_product(got, x, _f64(tokens.unpack_weight(w, torch.float32)), bias,
                   None if gate is None else _f64(tokens.unpack_weight(gate, torch.float32)), activation, dtype)
    assert torch.equal(tokens.packed_linear(x.contiguous(), w, bias=bias, gate=gate, gate_activation=activation), got)
    # what is not a number stays in its row, what lies behind a row stays out
    wide = torch.full((rows, inputs + 5), math.nan, dtype=dtype, device="cuda")
    wide[:, 3:-2] = x
    wide[rows - 1, inputs + 2] = math.inf
    odd = tokens.packed_linear(wide[:, 3:-2], w, bias=bias, gate=gate, gate_activation=activation)
    assert torch.equal(odd[:-1], got[:-1]) and not torch.isfinite(odd[-1]).any()
