"""How the token operators take their arguments, as far as no device is needed."""

from __future__ import annotations

import itertools
import threading

import numpy as np
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


# ---- numbers and positions ------------------------------------------------------------


@pytest.fixture
def launches(monkeypatch):
    """What the library would be told, on a host without a device."""
    told = []
    monkeypatch.setattr(tokens, "_check", lambda *args: None)
    monkeypatch.setattr(tokens, "_launch", lambda device, entry, config, *rest: told.append((entry, config, rest)))
    monkeypatch.setattr(tokens, "_checked", {})
    return told


def _selection():
    return torch.zeros(1, 4, 2, 16), tokens.BlockSummary(torch.zeros(1, 2, 8, 16, dtype=torch.int8), torch.zeros(1, 2, 8))


@pytest.mark.parametrize("order", list(itertools.permutations((40, np.int64(40), None, 7))))
def test_start_whatever_was_called_before(launches, order):
    q, summary = _selection()
    k, ids = torch.zeros(1, 128, 2, 16), torch.zeros(1, 4, 2, 1, dtype=torch.int32)
    for start in order:
        tokens.select_blocks(q, summary, 16, 1, start=start)
        tokens.block_attention(q, k, k, ids, 16, start=start)
        for _, config, _ in launches[-2:]:
            assert config.start == (0 if start is None else int(start))
    assert len(tokens._checked) == 2  # a position that moves is checked once


@pytest.mark.parametrize("start", [40.0, "x", np.float64(3), 1 << 40, -1, -(1 << 63), 1 << 64])
def test_start_that_is_no_position(launches, start):
    q, summary = _selection()
    for known in (False, True):
        with pytest.raises(ContractError, match="start"):
            tokens.select_blocks(q, summary, 16, 1, start=start)
        if not known:
            tokens.select_blocks(q, summary, 16, 1, start=40)
    assert [config.start for _, config, _ in launches] == [40]


def _norm(**kw):
    x = torch.zeros(3, 8)
    return tokens.residual_norm(x, x, **kw)


def _rotate(**kw):
    plan = tokens.rotary_plan(16, device="cpu")._replace(amplitude=kw.pop("amplitude", 1.0))
    return tokens.rotate(torch.zeros(1, 4, 2, 16), None, torch.zeros(4, 1, dtype=torch.int32), plan, **kw)


def _select(**kw):
    q, summary = _selection()
    return tokens.select_blocks(q, summary, kw.pop("block", 16), kw.pop("keep", 1), **kw)


def _attend(**kw):
    k, ids = torch.zeros(1, 128, 2, 16), torch.zeros(1, 4, 2, 1, dtype=torch.int32)
    return tokens.block_attention(_selection()[0], k, k, ids, kw.pop("block", 16), **kw)


def _summarize(**kw):
    return tokens.summarize_blocks(torch.zeros(1, 128, 2, 16), kw.pop("block", 16), out=_selection()[1], **kw)


@pytest.mark.parametrize("call,name,value", [
    (_norm, "residual_scale", 0.5), (_norm, "eps", 0.25), (_rotate, "amplitude", 1.5), (_attend, "scale", 0.125),
    (_rotate, "inverse", True), (_select, "causal", True), (_attend, "causal", True), (_select, "block", 16),
    (_select, "keep", 3), (_select, "first", 2), (_select, "local", 2), (_attend, "block", 16), (_summarize, "block", 16),
    (_summarize, "first", 2), (_summarize, "count", 3)])
def test_numbers_that_tensors_hold(launches, call, name, value):
    """A tensor's value can change behind a remembered call and would have to be waited for; a NumPy number is
    as good as Python's."""
    with pytest.raises(ContractError, match=name):
        call(**{name: torch.tensor(value)})
    call(**{name: value})
    call(**{name: np.array([value])[0]})
    one, two = ((entry, bytes(config), [a for a in rest if isinstance(a, int) and a < 1 << 20])
                for entry, config, rest in launches)
    assert one == two and len(tokens._checked) == 1


@pytest.mark.parametrize("call,kw", [
    (_norm, dict(residual_scale="1")), (_norm, dict(residual_scale=1e39)), (_norm, dict(eps=None)), (_rotate, dict(amplitude=-1e40)),
    (_attend, dict(scale=1e300)), (_attend, dict(scale="0.1")), (_select, dict(keep=1.0)), (_select, dict(keep=1 << 32)),
    (_select, dict(first=1 << 31)), (_select, dict(local=1.5)), (_summarize, dict(first=1 << 32, count=1)),
    (_summarize, dict(first=0, count=1 << 32)), (_summarize, dict(first=0.0)), (_summarize, dict(count=9)),
    (_summarize, dict(first=-1, count=2))])
def test_numbers_that_are_none_or_do_not_fit(launches, call, kw):
    with pytest.raises(ContractError):
        call(**kw)
    assert not launches


# ---- what a call cannot do ------------------------------------------------------------


def test_positions_of_too_few_axes(launches):
    """A plan knows how many position axes its pairs turn by."""
    q, plan = torch.zeros(1, 4, 2, 16), tokens.rotary_plan(12, axes=3, device="cpu")
    made = tokens.RotaryPlan(plan.steps, plan.axes, 1.0)
    for known in (made, plan):  # the check of one plan does not stand for another of the same shapes
        for axes in (3, 4):
            tokens.rotate(q, None, torch.zeros(4, axes, dtype=torch.int32), known)
    tokens.rotate(q, None, torch.zeros(4, 2, dtype=torch.int32), made)
    for axes in (1, 2):
        with pytest.raises(ContractError, match="axes"):
            tokens.rotate(q, None, torch.zeros(4, axes, dtype=torch.int32), plan)
    assert len(launches) == 5


@pytest.mark.parametrize("call", [
    lambda x, w: tokens.rotate(x, None, torch.zeros(4, 1, dtype=torch.int32), tokens.rotary_plan(16, device="cpu"))[0],
    lambda x, w: tokens.residual_norm(x, None, pre=(w, None))[1],
    lambda x, w: tokens.residual_norm(torch.zeros(3, 16), None, post=(None, w))[0],
    lambda x, w: tokens.residual_norm(torch.zeros_like(x), torch.zeros_like(x), gate=x)[0],
    lambda x, w: tokens.block_attention(torch.zeros_like(x), x, torch.zeros_like(x), torch.zeros(1, 4, 2, 1, dtype=torch.int32), 16),
    lambda x, w: tokens.sparse_attention(x, torch.zeros_like(x), torch.zeros_like(x), 16, 1)[0]])
def test_a_gradient_that_is_asked_for_is_refused(launches, call):
    """Forward only: results of inputs that require a gradient are there, but say so in the backward pass
    instead of losing it."""
    x, w = torch.zeros(1, 4, 2, 16, requires_grad=True), torch.zeros(16, requires_grad=True)
    y = call(x, w)
    with pytest.raises(ContractError, match="forward only"):
        (y + x.sum() + w.sum()).sum().backward()
    with torch.no_grad():
        assert not call(x, w).requires_grad
    assert not call(x.detach(), w.detach()).requires_grad


def test_no_results_into_place_where_a_gradient_is_kept(launches):
    q = torch.zeros(1, 4, 2, 16, requires_grad=True)
    plan, positions = tokens.rotary_plan(16, device="cpu"), torch.zeros(4, 1, dtype=torch.int32)
    ids, out = torch.zeros(1, 4, 2, 1, dtype=torch.int32), torch.zeros(1, 4, 2, 16)
    for call in (lambda: tokens.rotate(q, None, positions, plan, out=(q, None)),
                 lambda: tokens.rotate(out, None, positions, plan, out=(q, None)),
                 lambda: tokens.rotate(q, None, positions, plan, out=(out, None)),
                 lambda: tokens.block_attention(q, out, out, ids, 16, out=out)):
        with pytest.raises(ContractError, match="forward only"):
            call()
    assert not launches
    with torch.no_grad():
        assert tokens.rotate(q, None, positions, plan, out=(q, None))[0] is q
    assert len(launches) == 1


def test_threads_that_share_what_has_been_checked(launches):
    """Eight threads with more signatures than are remembered: every call is told its own shape."""
    def work(seed):
        for i in range(400):
            n = 1 + (seed * 400 + i) % 1500
            tokens.residual_norm(torch.zeros(n, 4), None)

    threads = [threading.Thread(target=work, args=(seed,)) for seed in range(8)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert sorted(config.rows for _, config, _ in launches) == sorted(1 + n % 1500 for n in range(3200))
    assert len(tokens._checked) <= 1024 + 8
