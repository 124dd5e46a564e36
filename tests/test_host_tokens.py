"""Argument checks of the token operators' C entry points on a CPU host: every refusal comes
before any device call, and a size query answers 0 for what its entry refuses."""

from __future__ import annotations

import ctypes

import pytest

from nnunet_mlx import _native


def _rotary(**kw):
    c = _native.NnxRotaryConfig(0, 1, 1, (1, 0), 64, 64, 1, 0, 0, 1.0)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def _norm(**kw):
    c = _native.NnxResidualNormConfig(0, 0, 4, 64, 0, 0, 0, 1.0, 1e-5)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def _block(**kw):
    c = _native.NnxBlockConfig(0, 1, 4, 100, 4, 2, 64, 16, 3, 0, 1, 0, 0, 0.125)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def _refused(status, text):
    assert status == _native.NNX_ERR_INVALID
    assert text in _native.load().nnx_last_error().decode(), _native.load().nnx_last_error()


@pytest.mark.parametrize("change,text", [
    (dict(type=3), "type"), (dict(batch=0), "positive"), (dict(tokens=-1), "positive"),
    (dict(heads=(0, 0)), "heads"), (dict(heads=(-1, 2)), "heads"), (dict(head_dim=1025), "head_dim"),
    (dict(rotary_dim=7), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"), (dict(axes=9), "axes"),
    (dict(amplitude=float("inf")), "amplitude"), ({}, "null pointer")])
def test_rotary(change, text):
    _refused(_native.load().nnx_rotary(_rotary(**change), *[None] * 8), text)


@pytest.mark.parametrize("change,text", [
    (dict(type=-1), "type"), (dict(type=1, residual_type=2), "float32"), (dict(rows=0), "rows"),
    (dict(rows=1 << 31), "rows"), (dict(channels=0), "channels"), (dict(channels=16385), "channels"),
    (dict(kind=2), "norm"), (dict(gate_activation=3), "gate"), (dict(eps=-1e-3), "eps"),
    (dict(residual_scale=float("nan")), "scale"), ({}, "null pointer")])
def test_residual_norm(change, text):
    _refused(_native.load().nnx_residual_norm(_norm(**change), *[None] * 11), text)


@pytest.mark.parametrize("change,text", [
    (dict(type=9), "type"), (dict(batch=0), "items"), (dict(batch=65536), "items"), (dict(keys=0), "items"),
    (dict(kv_heads=0), "key heads"), (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(block=48), "block"), (dict(keys=32768 * 16 + 1), "32768"), (dict(queries=0), "queries"),
    (dict(heads=5), "multiple"), (dict(heads=2 * 1025), "share"), (dict(keep=0), "keep"), (dict(keep=257), "keep"),
    (dict(queries=1 << 30, keep=2), "2^31"), (dict(scale=float("inf")), "scale"), (dict(start=-1), "start"),
    (dict(first=-1), "first"), ({}, "null pointer")])
def test_blocks(change, text):
    lib, config = _native.load(), _block(**change)
    _refused(lib.nnx_block_select(config, *[None] * 6, 0, None), text)
    _refused(lib.nnx_block_attention(config, *[None] * 9, 0, None), text)
    if change:
        assert lib.nnx_block_attention_workspace(config) == 0
    else:
        assert lib.nnx_block_attention_workspace(config) > 0


def test_summaries():
    lib = _native.load()
    for first, count in ((-1, 1), (0, 8), (7, 1), (0, -1), (8, 0)):
        _refused(lib.nnx_block_summarize(_block(), None, None, None, first, count, None, None, None), "blocks")
    _refused(lib.nnx_block_summarize(_block(), None, None, None, 0, 7, None, None, None), "null pointer")


def test_selection_places():
    """Codes and workspaces that do not fit are refused before anything runs on a device."""
    lib = _native.load()
    few, many = _block(), _block(keys=32 * 3000)
    assert lib.nnx_block_select_workspace(few) == 0
    size = lib.nnx_block_select_workspace(many)
    assert size > 0
    assert lib.nnx_block_select_workspace(_block(keys=32 * 3000, keep=0)) == 0
    assert lib.nnx_block_select_workspace(ctypes.POINTER(_native.NnxBlockConfig)()) == 0
    place = 1 << 20
    for codes, scales in ((place + 4, place), (place, place + 2)):
        _refused(lib.nnx_block_select(few, place, codes, scales, None, place, None, 0, None), "aligned")
    for work, given in ((None, size), (place, size - 1), (place + 8, size)):
        _refused(lib.nnx_block_select(many, place, place, place, None, place, work, given, None), "workspace")
    size = lib.nnx_block_attention_workspace(many)
    for work, given in ((place, size - 1), (place + 8, size)):
        _refused(lib.nnx_block_attention(many, *[place] * 4, None, None, None, place, work, given, None), "workspace")


def test_null_configs():
    lib = _native.load()
    none = ctypes.POINTER(_native.NnxBlockConfig)()
    _refused(lib.nnx_block_select(none, *[None] * 6, 0, None), "null config")
    assert lib.nnx_block_attention_workspace(none) == 0
