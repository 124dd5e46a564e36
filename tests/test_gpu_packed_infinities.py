"""Infinite inputs of products with 4-bit weights: what float32 sums of the products make of them."""

from __future__ import annotations

import math

import pytest
import torch

from nnunet_mlx.model import tokens

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 20, 200, 4100])
@pytest.mark.parametrize("inputs", [40, 333, 640])
def test_infinite_inputs(device, inputs, rows, dtype):
    """One infinite input: infinite of the weight's sign, NaN where the weight is 0; two of other signs NaN as well."""
    m = torch.randn(60, inputs, generator=_gen(1)).cuda()
    w = tokens.pack_weight(m, 32)
    signs = torch.sign(tokens.unpack_weight(w, torch.float32)).double()
    x = torch.randn(rows, inputs, generator=_gen(2)).to(dtype).cuda()
    want = tokens.packed_linear(x, w)
    at, row = [0, 17, 31, inputs - 1], rows - 1
    for i in at:
        for odd in (math.inf, -math.inf):
            y = x.clone()
            y[row, i] = odd
            got = tokens.packed_linear(y, w)
            assert torch.equal(got[row].double().nan_to_num(7.0, 8.0, -8.0), (odd * signs[:, i]).nan_to_num(7.0, 8.0, -8.0))
            assert torch.equal(got[:row], want[:row])
    y = x.clone()
    y[row, at[0]], y[row, at[1]] = math.inf, -math.inf
    both = math.inf * signs[:, at[0]] - math.inf * signs[:, at[1]]
    got = tokens.packed_linear(y, w)
    assert torch.equal(got[row].double().nan_to_num(7.0, 8.0, -8.0), both.nan_to_num(7.0, 8.0, -8.0))
    y[row, at[2]] = math.nan
    assert torch.isnan(tokens.packed_linear(y, w)[row]).all()
    # a NaN whose last bits alone say so
    if dtype == torch.float32:
        y = x.clone()
        y.view(torch.int32)[row, at[1]] = 0x7F800001
        assert torch.isnan(tokens.packed_linear(y, w)[row]).all()
