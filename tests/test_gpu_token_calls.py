"""How the token operators take their arguments: views, numbers and positions, on the device."""

from __future__ import annotations

import pytest
import torch

from nnunet_mlx.errors import ContractError
from nnunet_mlx.model import tokens

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("cut", [
    lambda x: x[:, :1, 2:3], lambda x: x[:1, 3:4], lambda x: x[1:2, 2:3, ::2], lambda x: x[:, :, 4], lambda x: x[:1, :1],
    lambda x: x[:, -1:, -1:, 5:]])
def test_residual_norm_of_views_with_single_elements(device, cut):
    """Axes of one element at any place: the rows are the view's own, for x, residual and gate."""
    x, residual, gate = (cut(torch.randn(3, 5, 8, 24, generator=_gen(seed)).cuda()) for seed in range(3))
    got = tokens.residual_norm(x, residual, gate=gate, post=(None, None), pre=(None, None))
    want = tokens.residual_norm(x.contiguous(), residual.contiguous(), gate=gate.contiguous(), post=(None, None),
                                pre=(None, None))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert torch.equal(tokens.residual_norm(x, residual)[0], residual + x)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_a_scaled_turn_is_undone(device, layout):
    """By the opposite turn under the amplitude's reciprocal.  Each turn errs by 2e-6 of a pair's size."""
    x = torch.randn(1, 50, 3, 96, generator=_gen(3)).cuda()
    positions = torch.randint(0, 1 << 20, (50, 1), generator=_gen(4), dtype=torch.int32).cuda()
    plan = tokens.rotary_plan(96, scaling="ramp", factor=8.0)
    turned, _ = tokens.rotate(x, None, positions, plan, layout=layout)
    back, _ = tokens.rotate(turned, None, positions, plan._replace(amplitude=1 / plan.amplitude), layout=layout, inverse=True)
    assert plan.amplitude > 1.2
    assert float((back - x).abs().max()) <= 4e-6 * float(x.abs().max()) * 2**0.5
    again, _ = tokens.rotate(turned, None, positions, plan, layout=layout, inverse=True)
    assert float((again - plan.amplitude**2 * x).abs().max()) <= 4e-6 * plan.amplitude**2 * float(x.abs().max()) * 2**0.5


@pytest.mark.parametrize("block", [16, 128])
def test_a_causal_selection_does_not_see_later_keys(device, block):
    """With the query's own block kept for every query, what later keys hold changes neither the kept blocks
    nor the result."""
    k, v = (torch.randn(1, 700, 2, 32, generator=_gen(seed)).cuda() for seed in (5, 6))
    q = torch.randn(1, 700, 4, 32, generator=_gen(7)).cuda()
    want, ids = tokens.sparse_attention(q, k, v, block, 3, causal=True, local=1)
    for at in (1, 130, 255, 256, 500):
        later = k.clone()
        later[:, at:] = torch.randn(1, 700 - at, 2, 32, generator=_gen(at)).cuda() * 5
        got, again = tokens.sparse_attention(q, later, v, block, 3, causal=True, local=1)
        assert torch.equal(again[:, :at], ids[:, :at])
        # the same operations on the same numbers: the order of rows in a tile does not show
        assert torch.equal(got[:, :at], want[:, :at])


def test_one_position_for_all_items_and_each_its_own(device):
    q, k, v = (torch.randn(2, n, 2, 16, generator=_gen(n)).cuda() for n in (6, 90, 90))
    for start in (0, 7, 77):
        each = torch.full((2,), start, dtype=torch.int32, device="cuda")
        for a, b in zip(tokens.sparse_attention(q, k, v, 16, 2, causal=True, start=start),
                        tokens.sparse_attention(q, k, v, 16, 2, causal=True, start=each)):
            assert torch.equal(a, b)


def test_results_of_inputs_that_require_a_gradient(device):
    """The same results, whose backward pass is refused."""
    q, k, v = (torch.randn(1, n, 2, 16, generator=_gen(n)).cuda() for n in (6, 90, 91))
    v = v[:, :90]
    weight = torch.ones(32, device="cuda")
    plan, positions = tokens.rotary_plan(16), torch.arange(6, dtype=torch.int32, device="cuda")[:, None].contiguous()

    def run(q, v, weight):
        turned, _ = tokens.rotate(q, None, positions, plan)
        mixed, _ = tokens.sparse_attention(turned, k, v, 16, 3)
        return tokens.residual_norm(mixed.flatten(2), None, pre=(weight, None))[1]

    want = run(q, v, weight)
    for which in range(3):
        inputs = [t.clone().requires_grad_(i == which) for i, t in enumerate((q, v, weight))]
        got = run(*inputs)
        assert torch.equal(got.detach(), want)
        with pytest.raises(ContractError, match="forward only"):
            got.sum().backward()
        with torch.no_grad():
            assert torch.equal(run(*inputs), want)
