"""Token operators: the steps of a transformer block over the tokens of a volume.

A volume cut into cubes is a sequence of tokens.  Between a block's plain matrix products lie
rotary positions (``rotary_plan``, ``rotate``), attention over blocks of keys that a cheap
score selects for each query (``summarize_blocks``, ``select_blocks``, ``block_attention``, all
three in ``sparse_attention``) and the norms around the block with its gate and residual sum
(``residual_norm``).  Everything runs in libnnunet_hip.so on the current stream of the tensors'
device, forward only (a gradient asked of a result raises ``ContractError``; a selection has
none); float32, float16 and bfloat16 tensors with a contiguous last axis and any other strides.
No reference counterpart.
"""

from __future__ import annotations

import math
import numbers
import operator
import struct
from typing import NamedTuple

import torch

from nnunet_mlx import _native
from nnunet_mlx.errors import ContractError

_TYPES = {
    torch.float32: _native.NNX_TYPE_F32,
    torch.float16: _native.NNX_TYPE_F16,
    torch.bfloat16: _native.NNX_TYPE_BF16,
}
_KINDS = {"layer": _native.NNX_TOKEN_NORM_LAYER, "rms": _native.NNX_TOKEN_NORM_RMS}
_GATES = {
    "none": _native.NNX_GATE_NONE,
    "sigmoid": _native.NNX_GATE_SIGMOID,
    "silu": _native.NNX_GATE_SILU,
}
_LAYOUTS = {"half": 0, "interleaved": 1}
BLOCK_SIZES = (16, 32, 64, 128)

# native layouts of the library's configurations
_ROTARY = struct.Struct("@10if4x14q")
_NORM = struct.Struct("@2iq4i2f5q")
_BLOCK = struct.Struct("@12iqf4x13q")

# the current stream of a device index, as torch's own launches ask for it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ContractError(message)


def _whole(name: str, value) -> int:
    """The int of any whole number.  A tensor is none: its value would have to be waited for."""
    if type(value) is int:
        return value
    if not isinstance(value, torch.Tensor):
        try:
            return operator.index(value)
        except TypeError:
            pass
    raise ContractError(f"{name} must be a whole number, got {type(value).__name__}")


def _number(name: str, value) -> float:
    """The float of any real number in float32's range; of a tensor not, as above."""
    if type(value) is not float:
        if not isinstance(value, numbers.Real):
            raise ContractError(f"{name} must be a number, got {type(value).__name__}")
        value = float(value)
    if abs(value) <= 3.4028235e38:
        return value
    raise ContractError(f"{name} must be a finite float32, got {value}")


def _flag(name: str, value) -> bool:
    if type(value) is bool:
        return value
    if isinstance(value, torch.Tensor):
        raise ContractError(f"{name} must be true or false, got a tensor")
    return bool(value)


def _packed(structure, layout: struct.Struct, *values):
    try:
        return _native.packed(structure, layout, *values)
    except struct.error as error:
        raise ContractError(f"an argument does not fit its 32 or 64 bits: {error}") from error


def _check(name: str, tensor: torch.Tensor, dims: int, like: torch.Tensor | None = None) -> None:
    if tensor.dim() != dims:
        raise ContractError(f"{name} needs {dims} axes, got shape {tuple(tensor.shape)}")
    if not tensor.is_cuda:
        raise ContractError("the HIP path needs device tensors")
    if tensor.stride(-1) != 1 and tensor.shape[-1] > 1:
        raise ContractError(f"{name} needs a contiguous last axis")
    if like is None:
        if tensor.dtype not in _TYPES:
            raise ContractError(f"{name} must be float32, float16 or bfloat16, not {tensor.dtype}")
    elif tensor.device != like.device or tensor.dtype != like.dtype:
        raise ContractError(f"{name} is {tensor.dtype} on {tensor.device}, not {like.dtype} on {like.device}")


def _check_side(name: str, tensor: torch.Tensor, dtype: torch.dtype, shape: tuple[int, ...],
                device: torch.device) -> None:
    if tensor.dtype != dtype or tuple(tensor.shape) != shape or tensor.device != device:
        raise ContractError(f"{name} must be {dtype} {shape} on {device}, got {tensor.dtype} "
                            f"{tuple(tensor.shape)} on {tensor.device}")
    if not tensor.is_contiguous():
        raise ContractError(f"{name} must be contiguous")


def _address(tensor: torch.Tensor | None) -> int | None:
    return None if tensor is None else tensor.data_ptr()


# What calls have been checked and how the library is told of them, by the shapes, strides, types, devices
# and asked-for gradients of their tensors and their other arguments (never by what the tensors hold or where):
# checking again would be half of what the smallest calls cost.
_checked: dict = {}


def _signature(*tensors: torch.Tensor | None) -> tuple:
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.device, t.requires_grad) for t in tensors])


def _remember(key: tuple, value):
    if len(_checked) >= 1024:
        _checked.clear()
    _checked[key] = value
    return value


def _launch(device: torch.device, entry: str, *arguments) -> None:
    """Calls a library entry on the device's current stream, its last argument."""
    function = getattr(_native.load(), entry)
    if device.index == torch.cuda.current_device():
        status = function(*arguments, _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            status = function(*arguments, _raw_stream(device.index))
    if status:
        _native.check(status, entry)


class _ForwardOnly(torch.autograd.Function):
    """Results whose gradient is refused rather than lost."""

    @staticmethod
    def forward(ctx, name, results, *inputs):
        ctx.name = name
        return results

    @staticmethod
    def backward(ctx, *gradients):
        raise ContractError(f"{ctx.name} is forward only and has no gradient")


def _gradients(*tensors: torch.Tensor | None) -> bool:
    return any([t is not None and t.requires_grad for t in tensors])


def _without_gradient(name: str, results: tuple, given: bool, *inputs: torch.Tensor | None) -> tuple:
    """The results of inputs some of which require a gradient; ``given``: written into place."""
    if not torch.is_grad_enabled():
        return results
    if given:
        raise ContractError(f"{name} is forward only and writes no results into place where a gradient is kept")
    return _ForwardOnly.apply(name, results, *inputs)


# ---- rotary positions -----------------------------------------------------------------


class RotaryPlan(NamedTuple):
    """Rotation of the pairs of a head: ``steps`` int64 in 2^-64 turns a position, ``axes`` int32
    the position axis of each pair, ``amplitude`` the factor on the rotated elements and
    ``position_axes`` how many axes a position has at least (0: not checked; a pair whose axis a
    position lacks is turned by the last it has)."""

    steps: torch.Tensor
    axes: torch.Tensor
    amplitude: float
    position_axes: int = 0


def rotary_plan(rotary_dim: int, *, axes: int = 1, base: float = 10000.0, scaling: str | None = None,
                factor: float = 1.0, trained_length: int = 8192, low: float = 1.0, high: float = 32.0,
                device: torch.device | str = "cuda") -> RotaryPlan:
    """Frequencies base^(-i / n) for the n pairs of each position axis (the pairs are shared out
    evenly, the first axes taking one more), stretched for contexts ``factor`` times longer:

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"base"``: the base multiplied by factor^(n / (n - 1)), which divides the slowest frequency
      by ``factor`` and keeps the fastest;
    * ``"ramp"``: frequencies that turn fewer than ``low`` times over ``trained_length`` are divided
      by ``factor``, those above ``high`` turns kept, a linear ramp between; the amplitude is
      0.1 ln(factor) + 1.
    """
    _need(rotary_dim >= 2 and rotary_dim % 2 == 0, f"rotary_dim must be even and positive, got {rotary_dim}")
    pairs = rotary_dim // 2
    _need(1 <= axes <= min(8, pairs), f"axes must be 1 to min(8, {pairs}), got {axes}")
    _need(scaling in (None, "linear", "base", "ramp"), f"unknown scaling {scaling!r}")
    _need(math.isfinite(base) and base > 0, f"base must be positive, got {base}")
    _need(math.isfinite(factor) and factor >= 1, f"factor must be at least 1, got {factor}")
    _need(scaling != "ramp" or (high > low and trained_length > 0), "the ramp needs high > low and a length")
    steps, owners = [], []
    for axis in range(axes):
        n = pairs // axes + (axis < pairs % axes)
        stretched = base * factor ** (n / (n - 1)) if scaling == "base" and n > 1 else base
        for i in range(n):
            frequency = stretched ** (-i / n)
            if scaling == "linear":
                frequency /= factor
            elif scaling == "ramp":
                turns = trained_length * frequency / (2 * math.pi)
                kept = min(1.0, max(0.0, (turns - low) / (high - low)))
                frequency *= kept + (1 - kept) / factor
            step = round(frequency / (2 * math.pi) * 2.0**64) % (1 << 64)
            steps.append(step - (1 << 64) if step >= 1 << 63 else step)
            owners.append(axis)
    amplitude = 0.1 * math.log(factor) + 1.0 if scaling == "ramp" else 1.0
    return RotaryPlan(torch.tensor(steps, dtype=torch.int64, device=device),
                      torch.tensor(owners, dtype=torch.int32, device=device), amplitude, axes)


def rotate(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, plan: RotaryPlan, *,
           layout: str = "half", inverse: bool = False,
           out: tuple[torch.Tensor, torch.Tensor | None] | None = None,
           ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotary positions of ``q`` and ``k`` (batch, tokens, heads, head_dim) in one launch.

    ``positions`` is int32 (tokens, axes) or (batch, tokens, axes).  ``layout`` pairs element i
    with i + rotary_dim / 2 ("half") or 2i with 2i + 1 ("interleaved"); elements past the plan's
    pairs are copied.  ``inverse`` turns by the opposite angles, the amplitude included: it is the
    gradient of the forward turn, and undoes it where the amplitude is 1.  A scaled turn is undone with
    ``plan._replace(amplitude=1 / plan.amplitude)``.
    ``out`` may hold the results, ``(q, k)`` itself to rotate in place."""
    amplitude = plan.amplitude
    if type(amplitude) is not float or type(inverse) is not bool:
        amplitude, inverse = _number("plan.amplitude", amplitude), _flag("inverse", inverse)
    key = ("rotate", _signature(q, k, positions, plan.steps, plan.axes, *(out or (None,))), amplitude,
           plan.position_axes, layout, inverse)
    known = _checked.get(key)
    if known is None:
        known = _remember(key, (_rotary_config(q, k, positions, plan, amplitude, layout, inverse, out),
                                _gradients(q, k, *(out or ()))))
    config, gradients = known
    if out is None:
        yq = torch.empty_like(q, memory_format=torch.contiguous_format)
        yk = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        yq, yk = out
    results = (yq, yk)
    if gradients:
        results = _without_gradient("rotate", results, out is not None, q, k)
    if config:
        _launch(q.device, "nnx_rotary", config, q.data_ptr(), _address(k), positions.data_ptr(),
                plan.steps.data_ptr(), plan.axes.data_ptr(), yq.data_ptr(), _address(yk))
    return results


def _contiguous_strides(shape: torch.Size) -> tuple[int, int, int]:
    return (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3])


def _rotary_config(q, k, positions, plan, amplitude, layout, inverse, out):
    """The checked configuration of a rotation, False where there is nothing to do."""
    _number("plan.amplitude", amplitude)
    _check("q", q, 4)
    batch, tokens, heads, dim = q.shape
    rotary_dim = 2 * plan.steps.numel()
    _need(layout in _LAYOUTS, f"layout must be 'half' or 'interleaved', got {layout!r}")
    if k is not None:
        _check("k", k, 4, q)
        _need(k.shape[:2] == q.shape[:2] and k.shape[3] == dim,
              f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    _need(positions.dim() in (2, 3) and positions.dtype == torch.int32 and positions.device == q.device
          and positions.shape[-2] == tokens and positions.shape[:-2] in ((), (batch,)),
          f"positions must be int32 (tokens, axes) or (batch, tokens, axes) on {q.device}, got "
          f"{positions.dtype} {tuple(positions.shape)} on {positions.device}")
    axes = positions.shape[-1]
    _need(axes >= plan.position_axes, f"the plan turns by {plan.position_axes} position axes, positions have {axes}")
    _need(axes == 1 or positions.stride(-1) == 1, "positions need a contiguous last axis")
    _check_side("plan.steps", plan.steps, torch.int64, (rotary_dim // 2,), q.device)
    _check_side("plan.axes", plan.axes, torch.int32, (rotary_dim // 2,), q.device)
    none = (0, 0, 0)
    if out is None:
        strides = _contiguous_strides(q.shape), none if k is None else _contiguous_strides(k.shape)
    else:
        for name, x, y in (("out[0]", q, out[0]), ("out[1]", k, out[1])):
            _need((x is None) == (y is None), f"{name} does not match its input")
            if y is not None:
                _check(name, y, 4, q)
                _need(y.shape == x.shape, f"{name} {tuple(y.shape)} does not match its input {tuple(x.shape)}")
        strides = [none if y is None else y.stride()[:3] for y in out]
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return False
    return _packed(
        _native.NnxRotaryConfig, _ROTARY, _TYPES[q.dtype], batch, tokens, heads, 0 if k is None else k.shape[2],
        dim, rotary_dim, axes, _LAYOUTS[layout], int(inverse), amplitude,
        *q.stride()[:3], *(none if k is None else k.stride()[:3]), *strides[0], *strides[1],
        *((0, positions.stride(0)) if positions.dim() == 2 else positions.stride()[:2]))


# ---- the norms around a block ---------------------------------------------------------

Affine = tuple[torch.Tensor | None, torch.Tensor | None]


def _rows(name: str, tensor: torch.Tensor) -> int:
    """Stride of the rows of a (..., channels) tensor whose leading axes step evenly; an axis of one
    element takes no step, whatever its stride."""
    step, following = tensor.shape[-1], None  # of a single row, any
    for size, stride in zip(reversed(tensor.shape[:-1]), reversed(tensor.stride()[:-1])):
        if size == 1:
            continue
        if following is None:
            step = stride
        elif stride != following:
            raise ContractError(f"{name}: the axes before the last must step evenly")
        following = stride * size
    return step


def residual_norm(x: torch.Tensor, residual: torch.Tensor | None, *, kind: str = "layer",
                  post: Affine | None = None, pre: Affine | None = None,
                  gate: torch.Tensor | None = None, gate_activation: str = "none",
                  scale: torch.Tensor | None = None, residual_scale: float = 1.0, eps: float = 1e-6,
                  ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The residual sum between two blocks with the norms on both its sides, in one pass:

        u  = norm(x, post) if post is given, else x
        r' = residual_scale * residual + scale * activation(gate) * u
        y  = norm(r', pre) if pre is given

    Returns ``(r', y)``, y None without ``pre``.  ``x`` (..., channels) is a block's output;
    ``residual`` has its shape and dtype or is float32, and r' is like it (like x without one);
    ``gate`` is like x; ``scale`` float32 (channels,).  ``post`` and ``pre`` are (weight, bias),
    float32 (channels,) or None each.  ``kind`` is "layer" or "rms"; y is the norm of r' before
    it is rounded to its dtype."""
    if type(residual_scale) is not float or type(eps) is not float:
        residual_scale, eps = _number("residual_scale", residual_scale), _number("eps", eps)
    vectors = (scale, *(post or (None, None)), *(pre or (None, None)))
    key = ("norm", _signature(x, residual, gate, *vectors), kind, post is None, pre is None, gate_activation,
           residual_scale, eps)
    known = _checked.get(key)
    if known is None:
        known = _remember(key, (_norm_config(x, residual, gate, vectors, kind, post is not None, gate_activation,
                                             residual_scale, eps), _gradients(x, residual, gate, *vectors)))
    config, gradients = known
    total = torch.empty_like(x if residual is None else residual, memory_format=torch.contiguous_format)
    y = None if pre is None else torch.empty_like(x, memory_format=torch.contiguous_format)
    results = (total, y)
    if gradients:
        results = _without_gradient("residual_norm", results, False, x, residual, gate, *vectors)
    if config:
        _launch(x.device, "nnx_residual_norm", config, x.data_ptr(), _address(residual), _address(gate),
                *[None if v is None else v.data_ptr() for v in vectors], total.data_ptr(), _address(y))
    return results


def _norm_config(x, residual, gate, vectors, kind, post, gate_activation, residual_scale, eps):
    """The checked configuration of a residual norm, False where there is nothing to do."""
    _number("residual_scale", residual_scale), _number("eps", eps)
    _check("x", x, max(1, x.dim()))
    channels = x.shape[-1]
    rows = x.numel() // channels if channels else 0
    _need(kind in _KINDS, f"kind must be 'layer' or 'rms', got {kind!r}")
    _need(gate_activation in _GATES, f"unknown gate activation {gate_activation!r}")
    _need(gate is not None or gate_activation == "none", "a gate activation needs a gate")
    if residual is not None:
        _check("residual", residual, x.dim(), x if residual.dtype == x.dtype else None)
        _need(residual.shape == x.shape and residual.device == x.device
              and residual.dtype in (x.dtype, torch.float32),
              f"residual {residual.dtype} {tuple(residual.shape)} does not match x {x.dtype} {tuple(x.shape)}")
    if gate is not None:
        _check("gate", gate, x.dim(), x)
        _need(gate.shape == x.shape, f"gate {tuple(gate.shape)} does not match x {tuple(x.shape)}")
    for name, vector in zip(("scale", "post weight", "post bias", "pre weight", "pre bias"), vectors):
        if vector is not None:
            _check_side(name, vector, torch.float32, (channels,), x.device)
    if rows == 0:
        return False
    wide = _TYPES[x.dtype if residual is None else residual.dtype]
    return _packed(
        _native.NnxResidualNormConfig, _NORM, _TYPES[x.dtype], wide, rows, channels, _KINDS[kind], int(post),
        _GATES[gate_activation], residual_scale, eps, _rows("x", x),
        0 if residual is None else _rows("residual", residual), 0 if gate is None else _rows("gate", gate),
        channels, channels)


# ---- attention over selected blocks ---------------------------------------------------


class BlockSummary(NamedTuple):
    """Means of the blocks' valid keys in 8 bits: ``codes`` int8 (batch, kv_heads, blocks, head_dim)
    and ``scales`` float32 (batch, kv_heads, blocks), -1 for a block without valid keys."""

    codes: torch.Tensor
    scales: torch.Tensor


_NO_STRIDES = (0, 0, 0)


def _block_config(like: torch.Tensor, block: int, batch: int, queries: int, keys: int, heads: int,
                  kv_heads: int, *, keep: int = 1, first: int = 0, local: int = 0, causal: bool = False,
                  scale: float = 1.0, q=_NO_STRIDES, k=_NO_STRIDES, v=_NO_STRIDES,
                  out=_NO_STRIDES, mask_stride: int = 0) -> _native.NnxBlockConfig:
    if block not in BLOCK_SIZES:
        raise ContractError(f"block must be one of {BLOCK_SIZES}, got {block}")
    return _packed(_native.NnxBlockConfig, _BLOCK, _TYPES[like.dtype], batch, queries, keys, heads, kv_heads,
                   like.shape[-1], block, keep, first, local, causal, 0, scale, *q, *k, *v, *out, mask_stride)


def _one_start(start: int) -> int:
    """One position for all items."""
    at = _whole("start", start)
    _need(0 <= at < 1 << 40, f"start must be 0..2^40, got {at}")
    return at


def _placed(config: _native.NnxBlockConfig, start: int) -> _native.NnxBlockConfig:
    """The checked configuration for queries from ``start`` on.  A decoder moves it at every step, so it is
    no part of what is remembered."""
    config = _native.NnxBlockConfig.from_buffer_copy(config)
    config.start = start
    return config


def _check_lengths_mask(lengths: torch.Tensor | None, mask: torch.Tensor | None, batch: int, keys: int,
                        device: torch.device) -> int:
    """Checks both and returns the mask's stride."""
    if lengths is not None:
        _check_side("lengths", lengths, torch.int32, (batch,), device)
    if mask is None:
        return 0
    _need(mask.dtype in (torch.bool, torch.uint8) and tuple(mask.shape) == (batch, keys)
          and mask.device == device and (keys <= 1 or mask.stride(1) == 1),
          f"key_mask must be bool or uint8 ({batch}, {keys}) on {device} with a contiguous last axis, "
          f"got {mask.dtype} {tuple(mask.shape)} on {mask.device}")
    return mask.stride(0)


def summarize_blocks(k: torch.Tensor, block: int, *, lengths: torch.Tensor | None = None,
                     key_mask: torch.Tensor | None = None, first: int = 0, count: int | None = None,
                     out: BlockSummary | None = None) -> BlockSummary:
    """Summaries of the blocks of keys ``k`` (batch, keys, kv_heads, head_dim).

    ``lengths`` int32 (batch,) counts the keys each item has, ``key_mask`` (batch, keys) marks the
    ones that are seen.  ``first`` and ``count`` with ``out`` refresh those blocks of a summary
    that is kept, as after appending keys."""
    codes, scales = out or (None, None)
    if type(block) is not int or type(first) is not int:
        block, first = _whole("block", block), _whole("first", first)
    if count is not None and type(count) is not int:
        count = _whole("count", count)
    key = ("summarize", _signature(k, lengths, key_mask, codes, scales), block, first, count)
    known = _checked.get(key)
    if known is None:
        known = _remember(key, _summary_config(k, block, lengths, key_mask, first, count, out))
    config, blocks, count = known
    if out is None:
        batch, _, kv_heads, dim = k.shape
        out = BlockSummary(torch.empty((batch, kv_heads, blocks, dim), dtype=torch.int8, device=k.device),
                           torch.empty((batch, kv_heads, blocks), dtype=torch.float32, device=k.device))
    if config:
        _launch(k.device, "nnx_block_summarize", config, k.data_ptr(), _address(lengths), _address(key_mask),
                first, count, out.codes.data_ptr(), out.scales.data_ptr())
    return out


def _summary_config(k, block, lengths, key_mask, first, count, out):
    """The checked configuration (False where there is nothing to do), blocks in all and asked for."""
    _check("k", k, 4)
    batch, keys, kv_heads, dim = k.shape
    mask_stride = _check_lengths_mask(lengths, key_mask, batch, keys, k.device)
    config = _block_config(k, block, batch, 0, keys, kv_heads, kv_heads, k=k.stride()[:3],
                           mask_stride=mask_stride)
    blocks = -(-keys // block)
    if count is None:
        count = blocks - first
    if out is None:
        _need(first == 0 and count == blocks, "summaries of some blocks need the summary to refresh (out)")
    else:
        _check_side("out.codes", out.codes, torch.int8, (batch, kv_heads, blocks, dim), k.device)
        _check_side("out.scales", out.scales, torch.float32, (batch, kv_heads, blocks), k.device)
        _need(first >= 0 and count >= 0 and first + count <= blocks,
              f"blocks {first} to {first + count} are not blocks of the keys, which have {blocks}")
    return config if k.numel() else False, blocks, count


def select_blocks(q: torch.Tensor, summary: BlockSummary, block: int, keep: int, *, causal: bool = False,
                  start: torch.Tensor | int | None = None, first: int = 0, local: int = 1) -> torch.Tensor:
    """Blocks that each query (batch, queries, heads, head_dim) keeps for each key head: int32
    (batch, queries, kv_heads, keep), ascending, -1 behind the last.

    Kept are the ``first`` leading blocks, the ``local`` blocks ending at the query's own (its
    position is ``start``, an int or int32 (batch,), plus its index), and the best by the largest
    product of the summary with the query heads that share the key head; equal scores go to the
    lower index.  The scores are formed in whole numbers, so they do not depend on how the work is
    split.  ``causal`` leaves out the blocks behind the query's own.  A block's score is of all its
    valid keys, so with ``local`` 0 a causal query's own block is kept or not by keys behind the query
    too; with ``local`` 1 or more it is kept always, and no later key shows."""
    starts, at = start, 0
    if start is not None and not isinstance(start, torch.Tensor):
        starts, at = None, _one_start(start)
    if not type(block) is type(keep) is type(first) is type(local) is int or type(causal) is not bool:
        block, keep, causal = _whole("block", block), _whole("keep", keep), _flag("causal", causal)
        first, local = _whole("first", first), _whole("local", local)
    key = ("select", _signature(q, *summary, starts), block, keep, causal, first, local)
    known = _checked.get(key)
    if known is None:
        known = _remember(key, _selection_config(q, summary, block, keep, causal, starts, first, local))
    config, size = known
    ids = torch.empty((q.shape[0], q.shape[1], summary.codes.shape[1], keep), dtype=torch.int32, device=q.device)
    if config:
        work = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        _launch(q.device, "nnx_block_select", _placed(config, at) if at else config, q.data_ptr(),
                summary.codes.data_ptr(), summary.scales.data_ptr(), _address(starts), ids.data_ptr(), _address(work), size)
    elif ids.numel():
        ids.fill_(-1)
    return ids


def _selection_config(q, summary, block, keep, causal, starts, first, local):
    """The checked configuration of a selection (False where there is nothing to select from) and its workspace's
    bytes."""
    _check("q", q, 4)
    batch, queries, heads, dim = q.shape
    _need(summary.codes.dim() == 4, f"summary codes need 4 axes, got shape {tuple(summary.codes.shape)}")
    kv_heads, blocks = summary.codes.shape[1:3]
    _check_side("summary.codes", summary.codes, torch.int8, (batch, kv_heads, blocks, dim), q.device)
    _check_side("summary.scales", summary.scales, torch.float32, (batch, kv_heads, blocks), q.device)
    if starts is not None:
        _check_side("start", starts, torch.int32, (batch,), q.device)
    _need(keep >= 1, f"keep must be positive, got {keep}")
    config = _block_config(q, block, batch, queries, blocks * block, heads, kv_heads, keep=keep, first=first,
                           local=local, causal=causal, q=q.stride()[:3])
    if q.numel() == 0 or blocks == 0:
        return False, 0
    return config, _native.load().nnx_block_select_workspace(config)


def block_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ids: torch.Tensor, block: int, *,
                    scale: float | None = None, causal: bool = False,
                    start: torch.Tensor | int | None = None, lengths: torch.Tensor | None = None,
                    key_mask: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Softmax attention of q (batch, queries, heads, head_dim) over the keys k and values v
    (batch, keys, kv_heads, head_dim) of the blocks in ``ids`` (batch, queries, kv_heads, keep).

    ``scale`` defaults to head_dim^-0.5; ``causal``, ``start``, ``lengths`` and ``key_mask`` as in
    ``select_blocks`` and ``summarize_blocks``.  A query that sees no key gets zeros."""
    starts, at = start, 0
    if start is not None and not isinstance(start, torch.Tensor):
        starts, at = None, _one_start(start)
    if type(block) is not int or type(causal) is not bool:
        block, causal = _whole("block", block), _flag("causal", causal)
    if scale is not None and type(scale) is not float:
        scale = _number("scale", scale)
    key = ("attention", _signature(q, k, v, ids, starts, lengths, key_mask, out), block, scale, causal)
    known = _checked.get(key)
    if known is None:
        known = _remember(key, (*_attention_config(q, k, v, ids, block, scale, causal, starts, lengths, key_mask, out),
                                _gradients(q, k, v, out)))
    config, size, gradients = known
    given = out is not None
    if not given:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    results = (out,)
    if gradients:
        results = _without_gradient("block_attention", results, given, q, k, v)
    if config:
        work = torch.empty(size, dtype=torch.uint8, device=q.device)
        _launch(q.device, "nnx_block_attention", _placed(config, at) if at else config, q.data_ptr(), k.data_ptr(),
                v.data_ptr(), ids.data_ptr(), _address(starts), _address(lengths), _address(key_mask), out.data_ptr(),
                work.data_ptr(), size)
    elif out.numel():
        out.detach().zero_()
    return results[0]


def _attention_config(q, k, v, ids, block, scale, causal, starts, lengths, key_mask, out):
    """The checked configuration (False where there is nothing to attend to) and workspace bytes."""
    if scale is not None:
        _number("scale", scale)
    _check("q", q, 4)
    _check("k", k, 4, q)
    _check("v", v, 4, q)
    batch, queries, heads, dim = q.shape
    keys, kv_heads = k.shape[1:3]
    _need(k.shape == (batch, keys, kv_heads, dim) and v.shape == k.shape,
          f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match q {tuple(q.shape)}")
    _need(ids.dim() == 4, f"ids need 4 axes, got shape {tuple(ids.shape)}")
    keep = ids.shape[3]
    _check_side("ids", ids, torch.int32, (batch, queries, kv_heads, keep), q.device)
    if starts is not None:
        _check_side("start", starts, torch.int32, (batch,), q.device)
    mask_stride = _check_lengths_mask(lengths, key_mask, batch, keys, q.device)
    if out is not None:
        _check("out", out, 4, q)
        _need(out.shape == q.shape, f"out {tuple(out.shape)} does not match q {tuple(q.shape)}")
    config = _block_config(
        q, block, batch, queries, keys, heads, kv_heads, keep=keep, causal=causal,
        scale=dim**-0.5 if scale is None else scale,
        q=q.stride()[:3], k=k.stride()[:3], v=v.stride()[:3],
        out=_contiguous_strides(q.shape) if out is None else out.stride()[:3], mask_stride=mask_stride)
    if q.numel() == 0 or keys == 0:
        return False, 0
    # 0 for what the library refuses, with the reason, when it is called
    return config, max(1, _native.load().nnx_block_attention_workspace(config))


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, block: int, keep: int, *,
                     summary: BlockSummary | None = None, scale: float | None = None, causal: bool = False,
                     start: torch.Tensor | int | None = None, first: int = 0, local: int = 1,
                     lengths: torch.Tensor | None = None,
                     key_mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``summarize_blocks`` (unless a ``summary`` is held), ``select_blocks`` and ``block_attention``;
    returns the attention's output and the kept blocks."""
    if summary is None:
        summary = summarize_blocks(k, block, lengths=lengths, key_mask=key_mask)
    ids = select_blocks(q, summary, block, keep, causal=causal, start=start, first=first, local=local)
    return block_attention(q, k, v, ids, block, scale=scale, causal=causal, start=start, lengths=lengths,
                           key_mask=key_mask), ids
