"""Gradients that held tokens and packed weights cannot keep are refused, whichever argument asks for them.  On a
host without a device: launches are left out."""

from __future__ import annotations

import pytest
import torch

from nnunet_mlx.errors import ContractError
from nnunet_mlx.model import tokens


@pytest.fixture
def launches(monkeypatch):
    told = []
    monkeypatch.setattr(tokens, "_check", lambda *args: None)
    monkeypatch.setattr(tokens, "_launch", lambda device, entry, config, *rest: told.append(entry))
    monkeypatch.setattr(tokens, "_checked", {})
    return told


def _packed(requires_grad=False):
    codes, scales = tokens._packed_shapes(5, 32, 32)
    return tokens.PackedWeight(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, requires_grad=requires_grad),
                               5, 32, 32)


def test_what_is_held_keeps_no_gradient(launches):
    """Codes are written into place: keys or values that ask for a gradient are refused at once, as often as asked."""
    held, x = tokens.held_tokens(2, 100, 2, 32, device="cpu"), torch.zeros(2, 3, 2, 32)
    leaf = x.clone().requires_grad_()
    part = (leaf * 2)[:, :, :, :]
    asked = held._replace(k_scales=held.k_scales.clone().requires_grad_())
    for _ in range(2):
        for call in (lambda: tokens.hold_tokens(held, leaf, x), lambda: tokens.hold_tokens(held, x, part, start=5),
                     lambda: tokens.hold_tokens(asked, x, x),
                     lambda: tokens.read_held(asked, torch.float32, count=3, out=(x, x))):
            with pytest.raises(ContractError, match="forward only"):
                call()
    assert not launches
    with torch.no_grad():
        tokens.hold_tokens(held, leaf, part)
        tokens.hold_tokens(asked, x, x)
    tokens.hold_tokens(held, leaf.detach(), part.detach())
    assert launches == ["nnx_hold_tokens"] * 3


def test_gradients_of_scales_and_weights(launches):
    """Results that depend on them refuse their gradient when it is asked for."""
    held, x = tokens.held_tokens(2, 100, 2, 32, device="cpu"), torch.zeros(2, 3, 2, 32)
    k_asked = held._replace(k_scales=held.k_scales.clone().requires_grad_())
    v_asked = held._replace(v_scales=held.v_scales.clone().requires_grad_())
    weight = torch.nn.Parameter(torch.randn(5, 32))
    for call in (lambda: tokens.held_attention(x, k_asked, 100), lambda: tokens.held_attention(x, v_asked, 100),
                 lambda: tokens.read_held(k_asked, torch.float32)[0], lambda: tokens.read_held(v_asked, torch.float32)[1],
                 lambda: tokens.packed_linear(x, _packed(True)), lambda: tokens.packed_linear(x, _packed(), gate=_packed(True)),
                 lambda: tokens.pack_weight(weight, 32).scales,
                 lambda: tokens.packed_linear(x, tokens.pack_weight(weight, 32))):
        with pytest.raises(ContractError, match="forward only"):
            call().sum().backward()
        with torch.no_grad():
            assert not call().requires_grad
    assert weight.grad is None
    packed = tokens.pack_weight(weight, 32)
    assert not packed.codes.requires_grad and packed[2:] == (5, 32, 32)
    for call in (lambda: tokens.packed_linear(x, _packed(), gate=_packed()), lambda: tokens.held_attention(x, held, 100),
                 lambda: tokens.pack_weight(weight.detach(), 32).scales):
        assert not call().requires_grad
