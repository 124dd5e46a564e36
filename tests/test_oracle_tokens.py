"""The token operators' oracle against torch in float64, and the rotary plan's steps."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from nnunet_mlx.errors import ContractError
from nnunet_mlx.model import tokens
from oracle import tokens as ot


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_norm(kind):
    rng = np.random.default_rng(0)
    u, w, b = rng.standard_normal((7, 33)), rng.standard_normal(33), rng.standard_normal(33)
    tu, tw, tb = map(torch.from_numpy, (u, w, b))
    if kind == "layer":
        want = torch.nn.functional.layer_norm(tu, (33,), tw, tb, 1e-5)
    else:
        want = torch.nn.functional.rms_norm(tu, (33,), tw, 1e-5) + tb
    np.testing.assert_allclose(ot.norm(u, (w, b), kind, 1e-5), want.numpy(), rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotation_keeps_products_by_distance(layout):
    """The product of a rotated query and key depends on the distance of their positions alone,
    and the inverse undoes the rotation."""
    rng = np.random.default_rng(1)
    freq, axes = 100.0 ** (-np.arange(6) / 6), np.zeros(6, int)
    x = rng.standard_normal((1, 2, 1, 16))

    def product(p0, p1):
        y = ot.rotate(x, np.array([[[p0], [p1]]]), freq, axes, 1.0, layout, False)
        return (y[0, 0, 0, :12] * y[0, 1, 0, :12]).sum()

    assert product(3, 11) == pytest.approx(product(1003, 1011), abs=1e-9)
    assert abs(product(3, 11) - product(3, 14)) > 1e-3
    pos = np.array([[[5], [900]]])
    back = ot.rotate(ot.rotate(x, pos, freq, axes, 1.0, layout, False), pos, freq, axes, 1.0, layout, True)
    np.testing.assert_allclose(back, x, atol=1e-13)


def test_attention_over_every_block_is_plain_attention():
    rng = np.random.default_rng(2)
    q, k, v = (rng.standard_normal((2, 40, h, 8)) for h in (4, 2, 2))
    ids = np.broadcast_to(np.arange(3, dtype=np.int32), (2, 40, 2, 3))
    for causal in (False, True):
        see = ot.seen(ids, 40, 16, np.ones((2, 40), bool), causal=causal)
        got, _ = ot.attention(q, k, v, see, 0.3)
        tq, tk, tv = (torch.from_numpy(a).transpose(1, 2) for a in (q, k, v))
        want = torch.nn.functional.scaled_dot_product_attention(
            tq, tk.repeat_interleave(2, 1), tv.repeat_interleave(2, 1), is_causal=causal, scale=0.3)
        np.testing.assert_allclose(got, want.transpose(1, 2).numpy(), rtol=1e-11, atol=1e-12)


def test_summaries_are_the_means_of_valid_keys_in_8_bits():
    rng = np.random.default_rng(3)
    k = rng.standard_normal((1, 50, 1, 24)).astype(np.float32)
    valid = rng.random((1, 50)) < 0.6
    valid[0, 16:32] = False
    codes, scales = ot.summarize(k, 16, valid)
    assert scales[0, 0, 1] == -1 and codes[0, 0, 1].max() == 0
    for j in (0, 2, 3):
        part = slice(16 * j, 16 * j + 16)
        mean = k[0, part, 0][valid[0, part]].mean(0, dtype=np.float64)
        step = np.abs(mean).max() / 127
        np.testing.assert_allclose(codes[0, 0, j] * float(scales[0, 0, j]), mean, atol=0.5 * step + 1e-3 * step)


def test_selection_is_the_best_blocks_and_ties_go_low():
    codes = np.zeros((1, 1, 6, 8), np.int8)
    codes[0, 0, :, 0] = [5, 9, 9, -3, 9, 1]
    scales = np.array([[[1, 1, 1, 1, -1, 1]]], np.float32)
    q = np.zeros((1, 1, 1, 8), np.float32)
    q[..., 0] = 2
    assert ot.select(q, codes, scales, 16, 2, local=0)[0, 0, 0].tolist() == [1, 2]
    assert ot.select(q, codes, scales, 16, 1, local=0)[0, 0, 0].tolist() == [1]
    assert ot.select(q, codes, scales, 16, 6, local=0)[0, 0, 0].tolist() == [0, 1, 2, 3, 5, -1]
    assert ot.select(q, codes, scales, 16, 2, first=1, local=1, start=[50])[0, 0, 0].tolist() == [0, 3]
    assert ot.select(q, codes, scales, 16, 3, local=0, causal=True, start=[31])[0, 0, 0].tolist() == [0, 1, -1]


def test_rotary_plan_steps():
    """Steps are the frequencies in 2^-64 turns; the axes share the pairs; scaled contexts."""
    def frequencies(plan):
        return np.array([(s % (1 << 64)) / 2.0**64 * 2 * math.pi for s in plan.steps.tolist()])

    plan = tokens.rotary_plan(20, axes=3, device="cpu")
    assert plan.axes.tolist() == [0] * 4 + [1] * 3 + [2] * 3 and plan.amplitude == 1.0
    np.testing.assert_allclose(frequencies(plan)[4:7], 10000.0 ** (-np.arange(3) / 3), rtol=1e-12)
    plain = frequencies(tokens.rotary_plan(64, device="cpu"))
    linear = frequencies(tokens.rotary_plan(64, scaling="linear", factor=4.0, device="cpu"))
    np.testing.assert_allclose(linear, plain / 4, rtol=1e-12)
    based = frequencies(tokens.rotary_plan(64, scaling="base", factor=4.0, device="cpu"))
    assert based[0] == plain[0] and based[-1] == pytest.approx(plain[-1] / 4, rel=1e-9)
    ramp = tokens.rotary_plan(64, scaling="ramp", factor=4.0, trained_length=1000, device="cpu")
    got, turns = frequencies(ramp), 1000 * plain / (2 * math.pi)
    np.testing.assert_allclose(got[turns > 32], plain[turns > 32], rtol=1e-12)
    np.testing.assert_allclose(got[turns < 1], plain[turns < 1] / 4, rtol=1e-12)
    assert ramp.amplitude == pytest.approx(0.1 * math.log(4) + 1)


@pytest.mark.parametrize("arguments", [
    dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, axes=5), dict(rotary_dim=8, axes=0),
    dict(rotary_dim=8, scaling="wide"), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=0.5),
    dict(rotary_dim=8, scaling="ramp", factor=2.0, low=4.0, high=4.0)])
def test_rotary_plan_refusals(arguments):
    with pytest.raises(ContractError):
        tokens.rotary_plan(device="cpu", **arguments)
