"""Arguments of held attention whose product with a constant of the kernel's leaves float32: refused by the C entry."""

from __future__ import annotations

import pytest

from nnunet_mlx import _native


@pytest.mark.parametrize("scale", [2.4e38, 3e38, -3e38, 3.4028234e38, float("inf")])
@pytest.mark.parametrize("kind", [_native.NNX_TYPE_F32, _native.NNX_TYPE_F16, _native.NNX_TYPE_BF16])
def test_scales_past_float32_in_octaves(kind, scale):
    """Logits are in units of log 2: a scale is multiplied by log2 e, 1.4427."""
    lib = _native.load()
    config = _native.NnxHeldConfig(kind, 1, 4, 4096, 4096, 4, 2, 64, 0, scale, 0)
    assert lib.nnx_held_attention(config, *[None] * 10, 0, None) == _native.NNX_ERR_INVALID
    assert "scale" in lib.nnx_last_error().decode()
    assert lib.nnx_held_attention_workspace(config) == 0


def test_the_largest_scales():
    """Up to float32's end over log2 e a scale is no reason to refuse."""
    lib = _native.load()
    for scale in (2.35e38, -2.35e38, 0.0):
        config = _native.NnxHeldConfig(0, 1, 4, 4096, 4096, 4, 2, 64, 0, scale, 0)
        assert lib.nnx_held_attention(config, *[None] * 10, 0, None) == _native.NNX_ERR_INVALID
        assert "null pointer" in lib.nnx_last_error().decode()
