"""Gradients that held tokens and packed weights cannot keep: refused, and the results without them as they are."""

from __future__ import annotations

import pytest
import torch

from nnunet_mlx.errors import ContractError
from nnunet_mlx.model import tokens

pytestmark = pytest.mark.gpu


def test_a_trained_projection(device):
    """Keys and values of a layer that is trained, and its weights packed, beside the same without gradients."""
    gen = torch.Generator().manual_seed(1)
    weight = torch.nn.Parameter(torch.randn(96, 40, generator=gen).cuda())
    x = torch.randn(2, 7, 40, generator=gen).cuda()
    k, v, q = torch.nn.functional.linear(x, weight).unflatten(-1, (3, 1, 32)).unbind(2)
    held = tokens.held_tokens(2, 7, 1, 32)
    for call in (lambda: tokens.hold_tokens(held, k, v.detach()), lambda: tokens.hold_tokens(held, k.detach(), v)):
        with pytest.raises(ContractError, match="forward only"):
            call()
    assert not any(t.any() for t in held)
    with torch.no_grad():
        tokens.hold_tokens(held, k, v)
    want = tokens.hold_tokens(tokens.held_tokens(2, 7, 1, 32), k.detach(), v.detach())
    assert all(torch.equal(a, b) for a, b in zip(held, want))

    packed, plain = tokens.pack_weight(weight, 32), tokens.pack_weight(weight.detach(), 32)
    assert torch.equal(packed.codes, plain.codes) and torch.equal(packed.scales.detach(), plain.scales)
    asked = held._replace(v_scales=held.v_scales.clone().requires_grad_())
    for call, same in (
            (lambda: tokens.unpack_weight(packed, torch.float32), lambda: tokens.unpack_weight(plain, torch.float32)),
            (lambda: tokens.packed_linear(x, packed), lambda: tokens.packed_linear(x, plain)),
            (lambda: tokens.held_attention(q.detach(), asked, 7), lambda: tokens.held_attention(q.detach(), held, 7)),
            (lambda: tokens.read_held(asked, torch.float32, count=7)[1],
             lambda: tokens.read_held(held, torch.float32, count=7)[1])):
        got = call()
        assert torch.equal(got.detach(), same()) and not same().requires_grad
        with pytest.raises(ContractError, match="forward only"):
            got.sum().backward()
        with torch.no_grad():
            assert torch.equal(call(), same())
