"""How the token operators take their arguments, as far as no device is needed."""

from __future__ import annotations

import itertools

import pytest
import torch

from nnunet_mlx.errors import ContractError
from nnunet_mlx.model import tokens

# ---- rows of a (..., channels) tensor -------------------------------------------------


def _row_views():
    """Views whose rows step evenly, with axes of one element at every place."""
    base = torch.arange(4 * 6 * 10 * 8, dtype=torch.float32).reshape(4, 6, 10, 8)
    yield base[0, 0, 0]
    yield base[0, 0, 3:4]
    yield base[:, :, 2]
    yield base[:, ::2, 2, 1:7]
    yield base[0, :, :, 3:]
    yield base[:1, 2:5]
    yield base[:, :1, :1]
    yield base[:, 1:2, 4:5, :5]
    yield base[:, 5:, 7]
    yield base[1:2, :1, :3]
    yield base[1:2, 2:3, ::4]
    yield base[2:3, ::5, 9:]
    yield base[::3, 3:4, 9:]
    yield base[:1, :1, :1]
    yield base[:, 0, 0][:, None, None]
    yield base[0, 0, 0].expand(3, 5, 8)
    for shape in itertools.product((1, 3), repeat=4):
        yield torch.arange(float(torch.Size(shape).numel() * 8)).reshape(*shape, 8)


@pytest.mark.parametrize("view", _row_views(), ids=lambda v: f"{tuple(v.shape)}-{v.stride()}")
def test_rows_that_step_evenly(view):
    step = tokens._rows("x", view)
    rows = view.numel() // view.shape[-1]
    assert torch.equal(view.as_strided((rows, view.shape[-1]), (step, 1), view.storage_offset()),
                       view.reshape(rows, view.shape[-1]))


def test_rows_that_do_not():
    base = torch.zeros(4, 6, 10, 8)
    for view in (base[:, :1, :3], base[:, :, :3], base[:, ::3], base[:, ::5, :1], base.transpose(0, 1),
                 base.transpose(1, 2)[:, :, :1, :], torch.zeros(2, 1, 10, 8)[:, :, :3], torch.zeros(4, 3, 5, 8)[:, ::3],
                 base[0].expand(4, 6, 10, 8), base[:, :, :, :4].transpose(0, 2)):
        with pytest.raises(ContractError, match="evenly"):
            tokens._rows("x", view)
