"""Float64 restatement of the token operators (CPU, numpy).

The rotary angle comes from the frequency in float64, not from the plan's whole steps; the
block summaries and scores follow their definition step by step (float32 elementwise steps and
whole numbers), so kept blocks compare exactly; everything else is float64."""

from __future__ import annotations

import numpy as np

F32 = np.float32
TINY = F32(2.0**-60)


def rotate(x: np.ndarray, positions: np.ndarray, frequencies: np.ndarray, axes: np.ndarray,
           amplitude: float, layout: str, inverse: bool) -> np.ndarray:
    """x (B, T, H, D), positions (B, T, A) -> rotated, float64."""
    half = len(frequencies)
    angle = positions[..., axes].astype(np.float64) * frequencies  # (B, T, pairs)
    turn = amplitude * np.exp(1j * (-angle if inverse else angle))[:, :, None, :]
    y = x.astype(np.float64).copy()
    first, second = (slice(0, half), slice(half, 2 * half)) if layout == "half" else \
        (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z = (y[..., first] + 1j * y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def norm(u: np.ndarray, affine, kind: str, eps: float) -> np.ndarray:
    shift = u.mean(-1, keepdims=True) if kind == "layer" else 0.0
    u = (u - shift) / np.sqrt(((u - shift) ** 2).mean(-1, keepdims=True) + eps)
    weight, bias = affine
    if weight is not None:
        u = u * weight.astype(np.float64)
    return u if bias is None else u + bias.astype(np.float64)


def residual_norm(x, residual, *, kind="layer", post=None, pre=None, gate=None, activation="none",
                  scale=None, residual_scale=1.0, eps=1e-6):
    u = x.astype(np.float64)
    if post is not None:
        u = norm(u, post, kind, eps)
    if gate is not None:
        g = gate.astype(np.float64)
        open_ = 1.0 / (1.0 + np.exp(-g))
        u = u * {"none": g, "sigmoid": open_, "silu": g * open_}[activation]
    if scale is not None:
        u = u * scale.astype(np.float64)
    if residual is not None:
        u = u + residual_scale * residual.astype(np.float64)
    return u, None if pre is None else norm(u, pre, kind, eps)


def _codes(values: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """8-bit codes of the last axis and the largest magnitudes (1 where all but zero)."""
    values = np.where(np.isfinite(values), values, F32(0)).astype(F32)
    top = np.abs(values).max(-1, keepdims=True)
    small = top < TINY
    top = np.where(small, F32(1), top)
    codes = np.rint(values * (F32(127) / top)).astype(np.int64)
    return np.where(small, 0, codes), top


def summarize(k: np.ndarray, block: int, valid: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """k (B, S, G, D) float32, valid (B, S) -> codes (B, G, nb, D) int8, scales (B, G, nb)."""
    batch, keys, heads, dim = k.shape
    blocks = -(-keys // block)
    codes = np.zeros((batch, heads, blocks, dim), np.int8)
    scales = np.full((batch, heads, blocks), -1, F32)
    for b in range(batch):
        for g in range(heads):
            for j in range(blocks):
                part = slice(j * block, min((j + 1) * block, keys))
                rows = k[b, part, g][valid[b, part]].astype(F32)
                if not len(rows):
                    continue
                rows = np.where(np.isfinite(rows), rows, F32(0))
                top = np.abs(rows).max()
                scales[b, g, j] = 0
                if top < TINY:
                    continue
                total = np.rint(rows * (F32(32767) / top)).astype(np.int64).sum(0)
                most = np.abs(total).max()
                if most == 0:
                    continue
                codes[b, g, j] = np.rint(total.astype(F32) * (F32(127) / F32(most)))
                scales[b, g, j] = top / (F32(4161409) * F32(len(rows))) * F32(most)
    return codes, scales


def select(q: np.ndarray, codes: np.ndarray, scales: np.ndarray, block: int, keep: int, *,
           causal=False, start=None, first=0, local=1) -> np.ndarray:
    """Kept blocks (B, T, G, keep) int32, ascending, -1 behind the last."""
    batch, queries, heads, _ = q.shape
    kv_heads, blocks = codes.shape[1:3]
    group = heads // kv_heads
    ids = np.full((batch, queries, kv_heads, keep), -1, np.int32)
    whole, top = _codes(q)
    index = np.arange(blocks)
    for b in range(batch):
        for g in range(kv_heads):
            mine = slice(g * group, (g + 1) * group)
            dots = whole[b, :, mine] @ codes[b, g].astype(np.int64).T  # (T, group, blocks)
            with np.errstate(over="ignore"):
                score = (dots.astype(F32) * top[b, :, mine] * scales[b, g]).max(1)
            score = np.clip(score, np.finfo(F32).min, np.finfo(F32).max)
            for t in range(queries):
                own = ((0 if start is None else int(start[b])) + t) // block
                row = score[t].copy()
                row[(index < first) | ((index <= own) & (index > own - local))] = np.inf
                row[scales[b, g] < 0] = -np.inf
                if causal:
                    row[index > own] = -np.inf
                order = [j for j in np.argsort(-row, kind="stable")[:keep] if row[j] != -np.inf]
                ids[b, t, g, :len(order)] = np.sort(order)
    return ids


def seen(ids: np.ndarray, keys: int, block: int, valid: np.ndarray, *, causal=False,
         start=None) -> np.ndarray:
    """Which keys each query and key head sees: (B, T, G, S) booleans."""
    batch, queries, kv_heads, _ = ids.shape
    out = np.zeros((batch, queries, kv_heads, keys), bool)
    blocks = -(-keys // block)
    for b, t, g in np.ndindex(batch, queries, kv_heads):
        for j in ids[b, t, g]:
            if 0 <= j < blocks:
                out[b, t, g, j * block:(j + 1) * block] = True
        if causal:
            out[b, t, g, (0 if start is None else int(start[b])) + t + 1:] = False
    return out & valid[:, None, None, :]


def attention(q: np.ndarray, k: np.ndarray, v: np.ndarray, see: np.ndarray,
              scale: float) -> tuple[np.ndarray, np.ndarray]:
    """Softmax attention over the seen keys, float64, and per query row the mean over its weights
    of the largest |v| of each key (what an error of the weights can move an output by)."""
    batch, queries, heads, dim = q.shape
    group = heads // see.shape[2]
    out = np.zeros((batch, queries, heads, dim))
    size = np.zeros((batch, queries, heads))
    for b, t, h in np.ndindex(batch, queries, heads):
        rows = np.flatnonzero(see[b, t, h // group])
        if not len(rows):
            continue
        kk, vv = (a[b, rows, h // group].astype(np.float64) for a in (k, v))
        logits = kk @ q[b, t, h].astype(np.float64) * scale
        p = np.exp(logits - logits.max())
        p /= p.sum()
        out[b, t, h] = p @ vv
        size[b, t, h] = p @ np.abs(vv).max(1)
    return out, size


# ---- tokens held in 8 bits, weights in 4 -----------------------------------------------


def _scales(top: np.ndarray, steps: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Of largest magnitudes: the factor to codes of up to ``steps``, the scale, and where codes are zero."""
    zero = ~np.isfinite(top) | (top < TINY)
    safe = np.where(zero, F32(1), top).astype(F32)
    scale = np.minimum(safe, F32(3.4028233e38)) / F32(steps)
    scale = np.where(zero, np.where(np.isfinite(top), F32(0), F32(np.nan)), scale)
    return F32(steps) / safe, scale.astype(F32), zero


def hold(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """Rows (..., D) float32 -> codes int8 (..., D) and scales (...)."""
    up, scale, zero = _scales(np.abs(x).max(-1, keepdims=True), 127)
    with np.errstate(invalid="ignore", over="ignore"):
        codes = np.where(zero, F32(0), np.rint(x * up))
    return codes.astype(np.int8), scale[..., 0]


def place_values(codes: np.ndarray) -> np.ndarray:
    """Codes (B, G, slots, D) in the order in which values are held, slot by slot."""
    b, g, slots, d = codes.shape
    out = np.zeros((b, g, slots // 64, d, 64), np.int8)
    for s in range(64):
        out[..., 16 * (s // 4 % 4) + 4 * (s // 16) + s % 4] = codes[:, :, s::64]
    return out


LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def pack(w: np.ndarray, group: int) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """A matrix (O, I) float32 -> packed codes and scales and the matrix that they stand for, weight by weight."""
    outputs, inputs = w.shape
    tiles, blocks = -(-outputs // 16), -(-inputs // 128)
    codes = np.zeros((tiles, blocks, 64, 16), np.uint8)
    scales = np.zeros((tiles, blocks * 128 // group, 16), F32)
    stands = np.zeros(w.shape)
    for o in range(outputs):
        for i0 in range(0, inputs, group):
            part = w[o, i0:i0 + group]
            up, scale, zero = _scales(np.abs(part).max(), 6)
            scales[o // 16, i0 // group, o % 16] = scale
            for n, x in enumerate(part):
                size, i = 0.0 if zero else float(F32(abs(x)) * up), i0 + n
                # the nearest value, of two as near the one with the even code
                code = min(range(8), key=lambda c: (abs(LEVELS[c] - size), c % 2))
                stands[o, i] = np.copysign(LEVELS[code], x) * float(scale)
                if code and x < 0:
                    code += 8
                place, byte = i % 32 // 8 * 16 + o % 16, i % 128 // 32 * 4 + i % 8 // 2
                codes[o // 16, i // 128, place, byte] |= code << (4 if i % 2 else 0)
    return codes, scales, stands


def gated(u: np.ndarray, g: np.ndarray | None, activation: str) -> np.ndarray:
    if g is None:
        return u
    open_ = 1.0 / (1.0 + np.exp(-g))
    return u * {"none": g, "sigmoid": open_, "silu": g * open_}[activation]
