"""Tokens held in 8 bits and packed weights as far as no device is needed: the C entry points' refusals, and
how calls take their arguments."""

from __future__ import annotations

import ctypes
import struct
from pathlib import Path

import numpy as np
import pytest
import torch

from nnunet_mlx import _native
from nnunet_mlx.errors import ContractError
from nnunet_mlx.model import tokens
from oracle import tokens as ot


def _held(**kw):
    c = _native.NnxHeldConfig(0, 1, 4, 128, 100, 4, 2, 64, 0, 0.125, 0)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def _weight(**kw):
    c = _native.NnxPackedConfig(0, 300, 50, 64, 0, 4, 300, 50)
    for name, value in kw.items():
        setattr(c, name, value)
    return c


def _refused(status, text):
    assert status == _native.NNX_ERR_INVALID
    assert text in _native.load().nnx_last_error().decode(), _native.load().nnx_last_error()


PLACE = 1 << 20


@pytest.mark.parametrize("change,text", [
    (dict(type=3), "type"), (dict(batch=0), "items"), (dict(batch=65536), "items"), (dict(tokens=0), "items"),
    (dict(slots=0), "slots"), (dict(slots=100), "slots"), (dict(slots=-64), "slots"), (dict(kv_heads=0), "key heads"),
    (dict(kv_heads=65537), "key heads"), (dict(head_dim=24), "head_dim"), (dict(head_dim=144), "head_dim"),
    (dict(head_dim=0), "head_dim"), (dict(start=-1), "start"), (dict(start=1 << 40), "start"), ({}, "null pointer")])
def test_held(change, text):
    lib, config = _native.load(), _held(**change)
    _refused(lib.nnx_hold_tokens(config, *[None] * 9), text)
    _refused(lib.nnx_held_attention(config, *[None] * 10, 0, None), text)
    _refused(lib.nnx_read_held(config, *[None] * 7), text)
    if change:
        assert lib.nnx_held_attention_workspace(config) == 0


@pytest.mark.parametrize("change,text", [
    (dict(keys=0), "keys"), (dict(keys=129), "keys"), (dict(heads=0), "multiple"), (dict(heads=5), "multiple"),
    (dict(heads=1 << 17), "multiple"), (dict(tokens=1 << 30), "2^31"), (dict(scale=float("nan")), "scale")])
def test_held_attention(change, text):
    lib, config = _native.load(), _held(**change)
    _refused(lib.nnx_held_attention(config, *[None] * 10, 0, None), text)
    assert lib.nnx_held_attention_workspace(config) == 0


def test_held_places():
    lib = _native.load()
    for off in range(4):
        held = [PLACE + (8 if i == off else 0) for i in range(4)]
        _refused(lib.nnx_hold_tokens(_held(), PLACE, PLACE, None, None, *held, None), "aligned")
        _refused(lib.nnx_read_held(_held(), *held, PLACE, PLACE, None), "aligned")
        _refused(lib.nnx_held_attention(_held(), PLACE, *held, None, None, None, PLACE, None, 0, None), "aligned")
    _refused(lib.nnx_read_held(_held(start=125), *[None] * 7), "slots")
    _refused(lib.nnx_hold_tokens(_held(tokens=1 << 30), *[None] * 9), "2^30")
    # long caches of many queries, whose partial results need memory
    large = _held(slots=1 << 20, keys=1 << 20, tokens=1)
    size = lib.nnx_held_attention_workspace(large)
    if size:
        for work, given in ((None, size), (PLACE, size - 1), (PLACE + 8, size)):
            _refused(lib.nnx_held_attention(large, *[PLACE] * 5, None, None, None, PLACE, work, given, None), "workspace")
    assert lib.nnx_held_attention_workspace(_held(slots=1 << 20, keys=1 << 20, tokens=1, start=77)) == size


@pytest.mark.parametrize("change,text", [
    (dict(type=-1), "type"), (dict(inputs=0), "inputs"), (dict(inputs=(1 << 20) + 1), "inputs"), (dict(outputs=0), "inputs"),
    (dict(outputs=(1 << 20) + 1), "inputs"), (dict(group=16), "group"), ({}, "null pointer")])
def test_packed(change, text):
    lib, config = _native.load(), _weight(**change)
    _refused(lib.nnx_pack_weight(config, *[None] * 4), text)
    _refused(lib.nnx_unpack_weight(config, *[None] * 4), text)
    _refused(lib.nnx_packed_linear(config, *[None] * 8), text)


def test_packed_linear():
    lib = _native.load()
    for change, text in ((dict(rows=0), "rows"), (dict(rows=1 << 31), "rows"), (dict(gate_activation=3), "gate")):
        _refused(lib.nnx_packed_linear(_weight(**change), *[None] * 8), text)
    for gate in ((PLACE, None), (None, PLACE)):
        _refused(lib.nnx_packed_linear(_weight(), PLACE, PLACE, PLACE, None, *gate, PLACE, None), "null pointer")
    for i in range(4):
        sides = [PLACE + (4 if j == i else 0) for j in range(4)]
        _refused(lib.nnx_packed_linear(_weight(), PLACE, *sides[:2], None, *sides[2:], PLACE, None), "aligned")


def test_null_configs():
    lib = _native.load()
    held, packed = (ctypes.POINTER(c)() for c in (_native.NnxHeldConfig, _native.NnxPackedConfig))
    _refused(lib.nnx_hold_tokens(held, *[None] * 9), "null config")
    _refused(lib.nnx_read_held(held, *[None] * 7), "null config")
    _refused(lib.nnx_held_attention(held, *[None] * 10, 0, None), "null config")
    assert lib.nnx_held_attention_workspace(held) == 0
    _refused(lib.nnx_pack_weight(packed, *[None] * 4), "null config")
    _refused(lib.nnx_unpack_weight(packed, *[None] * 4), "null config")
    _refused(lib.nnx_packed_linear(packed, *[None] * 8), "null config")


@pytest.mark.parametrize("structure,layout", [(_native.NnxHeldConfig, tokens._HELD), (_native.NnxPackedConfig, tokens._PACKED)])
def test_layouts(structure, layout):
    """A structure packed at once has its fields where setting them one by one puts them."""
    assert ctypes.sizeof(structure) == layout.size
    count = len(layout.unpack(bytes(layout.size)))
    packed = _native.packed(structure, layout, *range(1, count + 1))
    one, value = structure(), 1
    for name, kind in structure._fields_:
        if issubclass(kind, ctypes.Array):
            setattr(one, name, kind(*range(value, value + kind._length_)))
            value += kind._length_
        else:
            setattr(one, name, value)
            value += 1
    assert layout.unpack(bytes(packed)) == layout.unpack(bytes(one)) and struct.calcsize(layout.format) == layout.size


# ---- calls ----------------------------------------------------------------------------


@pytest.fixture
def launches(monkeypatch):
    """What the library would be told, on a host without a device."""
    told = []
    monkeypatch.setattr(tokens, "_check", lambda *args: None)
    monkeypatch.setattr(tokens, "_launch", lambda device, entry, config, *rest: told.append((entry, config, rest)))
    monkeypatch.setattr(tokens, "_checked", {})
    return told


def _some():
    return tokens.held_tokens(2, 100, 2, 32, device="cpu"), torch.zeros(2, 3, 2, 32)


def test_slots_that_move(launches):
    held, x = _some()
    assert held.k_scales.shape == (2, 2, 128)
    for at in (0, 5, np.int64(125), 7):
        tokens.hold_tokens(held, x, x, start=at)
        assert launches[-1][1].start == at
        tokens.read_held(held, torch.float32, first=at, count=3)
        assert launches[-1][1].start == at and launches[-1][1].tokens == 3
    for n in (1, 128, np.int32(64)):
        for at in (None, 3):
            tokens.held_attention(x, held, n, start=at)
            assert launches[-1][1].keys == n and launches[-1][1].start == (at or 0)
    tokens.held_attention(x, held, torch.zeros(2, dtype=torch.int32))
    assert launches[-1][1].keys == 128
    mask = torch.zeros(2, 70, dtype=torch.bool)
    for n, keys in ((torch.zeros(2, dtype=torch.int32), 70), (128, 70), (20, 20)):
        tokens.held_attention(x, held, n, key_mask=mask)
        assert launches[-1][1].keys == keys
    assert len(tokens._checked) == 6
    before = len(launches)
    for call in (lambda: tokens.hold_tokens(held, x, x, start=126), lambda: tokens.hold_tokens(held, x, x, start=-1),
                 lambda: tokens.hold_tokens(held, x, x, start=1.0), lambda: tokens.hold_tokens(held, x, x, start=None),
                 lambda: tokens.read_held(held, torch.float32, first=126, count=3),
                 lambda: tokens.read_held(held, torch.float32, first=1.0),
                 lambda: tokens.read_held(held, torch.float32, count=torch.tensor(3)),
                 lambda: tokens.held_attention(x, held, 129), lambda: tokens.held_attention(x, held, -1),
                 lambda: tokens.held_attention(x, held, 5.0), lambda: tokens.held_attention(x, held, None),
                 lambda: tokens.held_attention(x, held, 5, causal=torch.tensor(True)),
                 lambda: tokens.held_attention(x, held, 5, scale=torch.tensor(0.5)),
                 lambda: tokens.held_attention(x, held, 5, start=0.5)):
        with pytest.raises(ContractError):
            call()
    assert len(launches) == before


def test_rows_of_a_product(launches):
    codes, scales = tokens._packed_shapes(50, 300, 64)
    w = tokens.PackedWeight(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales), 50, 300, 64)
    for shape in ((300,), (4, 300), (2, 3, 300), (1, 1, 300), (0, 300)):
        assert tokens.packed_linear(torch.zeros(shape), w).shape == (*shape[:-1], 50)
    assert [config.rows for _, config, _ in launches] == [1, 4, 6, 1]
    tokens.packed_linear(torch.zeros(4, 8, 300)[:, 3], w, gate=w, gate_activation="silu")
    assert (launches[-1][1].x_stride, launches[-1][1].rows, launches[-1][1].gate_activation) == (2400, 4, 2)
    for call in (lambda: tokens.packed_linear(torch.zeros(4, 8, 300)[:, ::3], w),
                 lambda: tokens.packed_linear(torch.zeros(4, 299), w),
                 lambda: tokens.packed_linear(torch.zeros(4, 300), w._replace(group=torch.tensor(64))),
                 lambda: tokens.packed_linear(torch.zeros(4, 300), w, gate=w._replace(outputs=49))):
        with pytest.raises(ContractError):
            call()


def test_gradients(launches):
    held, x = _some()
    codes, scales = tokens._packed_shapes(5, 32, 32)
    w = tokens.PackedWeight(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales), 5, 32, 32)
    q = x.clone().requires_grad_()
    for call in (lambda: tokens.held_attention(q, held, 100), lambda: tokens.packed_linear(q, w),
                 lambda: tokens.packed_linear(x, w, bias=torch.zeros(5, requires_grad=True))):
        with pytest.raises(ContractError, match="forward only"):
            call().sum().backward()
        with torch.no_grad():
            assert not call().requires_grad
    with pytest.raises(ContractError, match="forward only"):
        tokens.held_attention(q, held, 100, out=x)
    with pytest.raises(ContractError, match="forward only"):
        tokens.read_held(held, torch.float32, count=3, out=(q, x))


# ---- the oracle's own formulas ----------------------------------------------------------


def test_oracle_quantisation():
    """Held rows are within half a step of what was held, packed weights at the nearest value."""
    x = np.random.default_rng(0).standard_normal((50, 32)).astype(np.float32)
    codes, scales = ot.hold(x)
    assert np.abs(codes).max(-1).min() == 127
    assert (np.abs(codes * scales[:, None].astype(np.float64) - x) <= 0.5001 * scales[:, None]).all()
    stands = ot.pack(x, 32)[2]
    size = np.abs(x).max(1, keepdims=True) / 6
    levels = np.concatenate([-ot.LEVELS[::-1], ot.LEVELS])
    nearest = np.abs(x[..., None] / size[..., None] - levels).min(-1) * size
    assert (np.abs(stands - x) <= nearest + 1e-6).all()


def test_oracle_places():
    codes = np.arange(2 * 1 * 128 * 16, dtype=np.int64).reshape(2, 1, 128, 16)
    placed = ot.place_values((codes % 251 - 125).astype(np.int8))
    for s in (0, 1, 5, 17, 63):
        assert np.array_equal(placed[1, 0, 1, :, 16 * (s // 4 % 4) + 4 * (s // 16) + s % 4],
                              (codes[1, 0, 64 + s] % 251 - 125).astype(np.int8))


def test_no_exception_leaves_the_size_query():
    """Refusals are built as strings, which may fail to be allocated: everything is caught."""
    source = (Path(__file__).resolve().parents[1] / "nnunet-mlx_amd" / "csrc" / "nnx_held.hip").read_text()
    query = source[source.index("size_t held_attention_workspace("):]
    assert "catch (...)" in query[:query.index("\n}\n")]


def test_arguments_of_the_wrong_kind(launches, monkeypatch):
    held, x = _some()
    for mask in (torch.tensor(True), torch.ones(5, dtype=torch.bool), torch.ones(2, 129, dtype=torch.bool),
                 torch.ones(2, 2, 5, dtype=torch.bool), torch.ones(2, 5)):
        with pytest.raises(ContractError, match="key_mask"):
            tokens.held_attention(x, held, 5, key_mask=mask)
    for lengths in (3, [1, 2], 1.0):
        with pytest.raises(ContractError, match="lengths"):
            tokens.hold_tokens(held, x, x, lengths=lengths)
    monkeypatch.undo()
    for call in (lambda: tokens.read_held(held, torch.float32), lambda: tokens.hold_tokens(held, x, x),
                 lambda: tokens.held_attention(x, held, 5)):  # nothing of a host's memory reaches a kernel
        with pytest.raises(ContractError, match="device"):
            call()
    assert not launches
