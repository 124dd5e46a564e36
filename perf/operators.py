"""The token operators' workloads: rotary positions, the norm around a block and block-sparse attention.

A volume cut into cubes is a sequence of tokens; these are the steps of a transformer block
over them outside its plain matrix products.  ``listed`` and ``draw`` give cases, ``prepare`` a
case's inputs on the GPU, ``run`` one pass, with ``own`` through ``nnunet_mlx.model.tokens`` and
else in elementary float32 torch operations, ``exact`` the result in float64 and ``work`` the
bytes and operations of one pass.

Token counts are those of the networks' patches (a 128^3 patch is 4096 cubes of 8^3 voxels and
32768 of 4^3, a 128 x 160 x 160 patch 6400 of 8^3); 320 channels, five heads of 64, is the width
of the networks' bottom stages.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parents[1] / "nnunet-mlx_amd")
_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}


# ---- the cases ------------------------------------------------------------------------


def _rotate(**kw):
    base = dict(op="rotate", type="bf16", batch=1, tokens=1, heads=5, kv_heads=5, dim=64, rotary=60,
                axes=3, layout="half", factor=1.0, inverse=False)
    return {**base, **kw}


def _norm(**kw):
    base = dict(op="norm", type="bf16", residual="bf16", rows=1, channels=320, kind="layer",
                post=False, pre=True, gate="none", activation="none", residual_scale=1.0)
    return {**base, **kw}


def _attend(**kw):
    base = dict(op="attend", type="bf16", batch=1, queries=1, keys=1, heads=5, kv_heads=5, dim=64,
                block=64, keep=16, first=0, local=1, causal=False, ragged=False, masked=False,
                held=False)
    return {**base, **kw}


def listed():
    return [
        # one prompted point against a volume: the position of a single token
        _rotate(name="rotate_point"),
        # a 128 x 160 x 160 patch in float32, as the networks' default precision; adjacent pairs, and
        # the inverse rotation (positions taken out again)
        _rotate(name="rotate_patch_fp32", type="fp32", tokens=6400, layout="interleaved", inverse=True),
        # two whole volumes as one line of tokens each, far beyond the trained length
        _rotate(name="rotate_long", type="fp16", batch=2, tokens=65536, heads=16, kv_heads=4, dim=128,
                rotary=96, axes=1, factor=8.0),
        # a single token between two blocks
        _norm(name="norm_point", post=True),
        # one 128^3 patch: block output scaled per channel and added, next norm
        _norm(name="norm_patch", rows=4096, gate="channel"),
        # odd rows and channels in float32; norm on both sides and a gate for every token
        _norm(name="norm_odd_fp32", type="fp32", residual="fp32", rows=6399, channels=331, kind="rms",
              post=True, gate="token", activation="sigmoid", residual_scale=0.8),
        # a batch of eight patches in fine cubes, the residual stream in float32
        _norm(name="norm_batch", residual="fp32", rows=262144, kind="rms", post=True, gate="channel"),
        # one prompted point against one coarse patch that is held
        _attend(name="attend_point", keys=4096, held=True),
        # prompts against three held volumes of different sizes, eight heads to a key head
        _attend(name="attend_prompts", type="fp16", batch=3, queries=4, keys=131072, heads=16, kv_heads=2,
                dim=128, keep=64, ragged=True, held=True),
        # two coarse patches over themselves, background tokens masked
        _attend(name="attend_patch", batch=2, queries=4096, keys=4096, masked=True),
        # an ordered sequence of slices' tokens in float32: odd sizes, ragged, one item empty
        _attend(name="attend_order_fp32", type="fp32", batch=4, queries=2501, keys=2501, heads=6, kv_heads=3,
                dim=80, block=32, keep=12, first=1, local=2, causal=True, ragged=True),
        # a fine patch over itself
        _attend(name="attend_fine", queries=32768, keys=32768, keep=32),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_rotate(rng):
    dim = rng.choice([32, 48, 64, 80, 96, 128])
    axes = rng.choice([1, 2, 3])
    kv = rng.randint(1, 8)
    return _rotate(type=rng.choice(list(_TYPES)), batch=rng.randint(1, 4), tokens=_log(rng, 1, 65536),
                   heads=kv * rng.choice([1, 2, 4]), kv_heads=kv, dim=dim,
                   rotary=2 * rng.randint(axes, dim // 2), axes=axes,
                   layout=rng.choice(["half", "interleaved"]),
                   factor=rng.choice([1.0, 4.0, 8.0]) if axes == 1 else 1.0,
                   inverse=rng.random() < 0.3)


def _draw_norm(rng):
    kind = rng.choice(list(_TYPES))
    gate = rng.choice(["none", "channel", "token"])
    post = rng.random() < 0.5
    return _norm(type=kind, residual=rng.choice([kind, "fp32"]), rows=_log(rng, 1, 262144),
                 channels=_log(rng, 33, 4096), kind=rng.choice(["layer", "rms"]), post=post,
                 pre=(not post) or rng.random() < 0.8, gate=gate,
                 activation=rng.choice(["none", "sigmoid", "silu"]) if gate == "token" else "none",
                 residual_scale=rng.choice([1.0, 0.8]))


def _draw_attend(rng):
    kv = rng.randint(1, 6)
    held = rng.random() < 0.4
    keys = _log(rng, 500, 131072 if held else 32768)
    queries = rng.randint(1, 8) if held else keys
    block = rng.choice([16, 32, 64, 128])
    causal = not held and rng.random() < 0.4
    batch = rng.randint(1, 4)
    return _attend(type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), batch=batch, queries=queries, keys=keys,
                   heads=kv * rng.choice([1, 1, 2, 4, 8]), kv_heads=kv, dim=rng.choice([32, 64, 80, 128]),
                   block=block, keep=rng.randint(4, 64), first=rng.randint(0, 1),
                   local=rng.randint(0, 2) if held else rng.randint(1, 2), causal=causal,
                   ragged=batch > 1 and rng.random() < 0.5, masked=not causal and rng.random() < 0.4, held=held)


def draw(rng):
    make = rng.choice([_draw_rotate, _draw_norm, _draw_attend, _draw_attend])
    while True:
        case = make(rng)
        most = [(work(c), _cost(c)) for c in listed() if c["op"] == case["op"]]
        asked = work(case)
        if (asked["bytes"] <= max(w["bytes"] for w, _ in most) and asked["flops"] <= max(w["flops"] for w, _ in most)
                and _cost(case) <= max(c for _, c in most)):
            return case


def _cost(case):
    """Elements that the plain form holds at once."""
    if case["op"] == "attend":
        return case["batch"] * case["heads"] * case["queries"] * case["keys"]
    if case["op"] == "norm":
        return case["rows"] * case["channels"]
    return case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]


# ---- the inputs -----------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _frequencies(case):
    """Radians per position of every pair in float64, its position axis, and the amplitude."""
    pairs = case["rotary"] // 2
    share = [pairs // case["axes"] + (a < pairs % case["axes"]) for a in range(case["axes"])]
    freqs, axes = [], []
    for axis, n in enumerate(share):
        freqs += [10000.0 ** (-i / n) for i in range(n)]
        axes += [axis] * n
    factor, amplitude = case["factor"], 1.0
    if factor != 1.0:  # slow pairs stretched by the factor, fast ones kept, a ramp between
        for i, f in enumerate(freqs):
            ramp = min(1.0, max(0.0, (8192 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)))
            freqs[i] = f * (ramp + (1.0 - ramp) / factor)
        amplitude = 0.1 * math.log(factor) + 1.0
    return freqs, axes, amplitude


def _prepare_rotate(case, gen):
    b, t, h, g, d = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
    # queries, keys and values of one projection, side by side
    qkv = _randn(gen, b, t, h + 2 * g, d).to(_TYPES[case["type"]])
    side = max(1, math.ceil(t ** (1.0 / case["axes"])))
    index = torch.arange(t, device="cuda")
    positions = torch.stack([(index // side ** a) % side if case["axes"] > 1 else index
                             for a in range(case["axes"])], 1)
    positions = positions + torch.randint(0, 512, (1, case["axes"]), generator=gen, device="cuda")
    freqs, axes, amplitude = _frequencies(case)
    steps = [round(f / (2 * math.pi) * 2.0 ** 64) for f in freqs]  # turns in units of 2^-64
    steps = [s - (1 << 64) if s >= 1 << 63 else s for s in steps]
    return {"case": case, "q": qkv[:, :, :h], "k": qkv[:, :, h:h + g],
            "positions": positions.to(torch.int32).contiguous(),
            "steps": torch.tensor(steps, dtype=torch.int64, device="cuda"),
            "axes": torch.tensor(axes, dtype=torch.int32, device="cuda"), "amplitude": amplitude}


def _prepare_norm(case, gen):
    n, c = case["rows"], case["channels"]
    kind, wide = _TYPES[case["type"]], _TYPES[case["residual"]]
    # a residual stream has channels of very different size and a mean
    sizes = torch.exp(_randn(gen, c))
    state = {"case": case, "x": (_randn(gen, n, c) * 0.5 + 0.1).to(kind),
             "residual": (_randn(gen, n, c) * sizes + 0.3).to(wide), "gate": None, "scale": None,
             "post": None, "pre": None}

    def weights():
        w = 1.0 + 0.1 * _randn(gen, c)
        return (w, 0.1 * _randn(gen, c) if case["kind"] == "layer" else None)

    if case["post"]:
        state["post"] = weights()
    if case["pre"]:
        state["pre"] = weights()
    if case["gate"] == "token":
        state["gate"] = _randn(gen, n, c).to(kind)
    elif case["gate"] == "channel":
        state["scale"] = 0.1 + 0.05 * _randn(gen, c)
    return state


def _lengths(case):
    """Valid keys of each item: the whole, or falling by an odd step down to an empty item."""
    n, b = case["keys"], case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [n] + [max(0, n - i * (n // (b - 1)) - 7) if b > 3 else n - i * (n // 4) - 7 for i in range(1, b)]


def _tissue(gen, batch, tokens, heads, dim):
    """Token features: runs of 32 prototypes that recur along the volume, and noise."""
    kinds = _randn(gen, 32, heads, dim)
    runs = torch.randint(0, 32, (batch, tokens // 96 + 1), generator=gen, device="cuda")
    at = torch.arange(tokens, device="cuda") // 96
    return kinds[runs[:, at]] + 0.7 * _randn(gen, batch, tokens, heads, dim)


def _prepare_attend(case, gen):
    b, t, n, h, g, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    kind = _TYPES[case["type"]]
    k = _tissue(gen, b, n, g, d)
    v = _randn(gen, b, n, g, d)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    at = torch.randint(0, n, (b, t), generator=gen, device="cuda") if case["held"] else \
        torch.arange(n, device="cuda").expand(b, n)
    # a query resembles keys like those at its own place
    near = torch.gather(k, 1, at[:, :, None, None].expand(b, t, g, d)).repeat_interleave(h // g, 2)
    q = 0.6 * near + 0.8 * _randn(gen, b, t, h, d)
    mask = None
    if case["masked"]:  # background in runs
        runs = torch.rand((b, n // 48 + 1), generator=gen, device="cuda") < 0.7
        mask = runs[:, torch.arange(n, device="cuda") // 48].contiguous()
    if case["ragged"]:  # what lies behind an item's end was never written
        behind = torch.arange(n, device="cuda")[None, :] >= lengths[:, None]
        k = k.masked_fill(behind[:, :, None, None], float("nan"))
        v = v.masked_fill(behind[:, :, None, None], float("nan"))
    state = {"case": case, "q": q.to(kind), "k": k.to(kind), "v": v.to(kind), "lengths": lengths,
             "mask": mask, "start": at[:, 0].to(torch.int32).contiguous(), "codes": None, "scales": None}
    if case["held"]:
        state["codes"], state["scales"] = _summaries(case, state["k"], lengths, mask)
    return state


def prepare(case, seed):
    gen = _generator(seed)
    make = {"rotate": _prepare_rotate, "norm": _prepare_norm, "attend": _prepare_attend}[case["op"]]
    return make(case, gen)


# ---- the plain forms ------------------------------------------------------------------


def _plain_rotate(s):
    case, half = s["case"], s["case"]["rotary"] // 2
    phase = s["positions"].long()[:, s["axes"].long()] * s["steps"]  # wraps at whole turns
    angle = (phase >> 40).float() * (2 * math.pi / 2 ** 24)
    cos = (torch.cos(angle) * s["amplitude"])[:, None, :]
    sin = (torch.sin(angle) * s["amplitude"])[:, None, :]
    if case["inverse"]:
        sin = -sin

    def turn(x):
        part, rest = x[..., :2 * half].float(), x[..., 2 * half:]
        if case["layout"] == "half":
            a, b = part[..., :half], part[..., half:]
            part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([part.to(x.dtype), rest], -1)

    return turn(s["q"]), turn(s["k"])


def _plain_norm(s):
    case = s["case"]

    def norm(u, weights):
        if case["kind"] == "layer":
            u = u - u.mean(1, keepdim=True)
        u = u * torch.rsqrt((u * u).mean(1, keepdim=True) + 1e-6) * weights[0]
        return u if weights[1] is None else u + weights[1]

    u = s["x"].float()
    if s["post"] is not None:
        u = norm(u, s["post"])
    if s["gate"] is not None:
        gate = s["gate"].float()
        if case["activation"] != "none":
            open_ = 1.0 / (1.0 + torch.exp(-gate))
            gate = open_ if case["activation"] == "sigmoid" else gate * open_
        u = u * gate
    if s["scale"] is not None:
        u = u * s["scale"]
    r = case["residual_scale"] * s["residual"].float() + u
    out = {"residual": r.to(s["residual"].dtype)}
    if s["pre"] is not None:
        out["y"] = norm(r, s["pre"]).to(s["x"].dtype)
    return out


def _valid(case, lengths, mask):
    valid = torch.arange(case["keys"], device=lengths.device)[None, :] < lengths[:, None]
    return valid if mask is None else valid & mask


def _summaries(case, k, lengths, mask):
    """Codes (batch, kv_heads, blocks, dim) and scales of the keys' block means."""
    block = case["block"]
    valid = _valid(case, lengths, mask)
    k = torch.where(valid[:, :, None, None] & torch.isfinite(k), k.float(), 0.0)
    pad = -k.shape[1] % block
    k = torch.nn.functional.pad(k, (0, 0, 0, 0, 0, pad)).unflatten(1, (-1, block))
    count = torch.nn.functional.pad(valid, (0, pad)).unflatten(1, (-1, block)).sum(2).float()[:, :, None]
    top = k.abs().amax((2, 4))  # (batch, blocks, kv_heads)
    tiny = top < 2.0 ** -60
    safe = torch.where(tiny, 1.0, top)
    up = torch.div(torch.full_like(safe, 32767.0), safe)
    # whole numbers below 2^24: exact in float32 in any order
    total = torch.round(k * up[:, :, None, :, None]).sum(2)
    total = torch.where(tiny[..., None], 0.0, total)
    most = total.abs().amax(3)
    few = torch.where(most == 0, 1.0, most)
    codes = torch.round(total * torch.div(torch.full_like(few, 127.0), few)[..., None])
    scales = torch.div(safe, 4161409.0 * torch.clamp(count, min=1.0)) * most
    scales = torch.where(count == 0, -1.0, scales)
    return codes.to(torch.int8).transpose(1, 2).contiguous(), scales.transpose(1, 2).contiguous()


def _select(case, q, codes, scales, start):
    """The kept blocks of every query and key head, ascending, -1 behind them."""
    b, t, h, d = q.shape
    g, blocks, keep = case["kv_heads"], codes.shape[2], case["keep"]
    q = torch.where(torch.isfinite(q), q.float(), 0.0)
    top = q.abs().amax(3, keepdim=True)
    safe = torch.where(top < 2.0 ** -60, 1.0, top)
    whole = torch.where(top < 2.0 ** -60, 0.0, torch.round(q * torch.div(torch.full_like(safe, 127.0), safe)))
    whole = whole.view(b, t, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(b, g, (h // g) * t, d)
    # whole numbers below 2^24 again
    score = torch.matmul(whole, codes.float().transpose(2, 3).contiguous()).view(b, g, h // g, t, blocks)
    top = safe.view(b, t, g, h // g).permute(0, 2, 3, 1)[..., None]
    score = (score * top * scales[:, :, None, None, :]).amax(2)  # (batch, kv_heads, queries, blocks)
    index = torch.arange(blocks, device=q.device)
    at = (start[:, None] + torch.arange(t, device=q.device)[None, :]) // case["block"]  # (batch, queries)
    at = at[:, None, :, None]
    usable = (scales >= 0)[:, :, None, :]
    if case["causal"]:
        usable = usable & (index <= at)
    forced = (index < case["first"]) | ((index <= at) & (index > at - case["local"]))
    score = torch.where(forced, float("inf"), score)
    score = torch.where(usable, score, -float("inf"))
    best, order = torch.sort(score, dim=3, descending=True, stable=True)
    order = torch.where(best == -float("inf"), blocks, order)[..., :keep]
    order = torch.sort(order, dim=3).values
    order = torch.nn.functional.pad(order, (0, keep - order.shape[3]), value=blocks)
    return torch.where(order == blocks, -1, order).to(torch.int32).transpose(1, 2).contiguous()


def _plain_attend(s):
    case, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, t, h, d = q.shape
    n, g = case["keys"], case["kv_heads"]
    codes, scales = s["codes"], s["scales"]
    if not case["held"]:
        codes, scales = _summaries(case, k, s["lengths"], s["mask"])
    ids = _select(case, q, codes, scales, s["start"])
    blocks = codes.shape[2]
    kept = torch.zeros((b, g, t, blocks + 1), dtype=torch.bool, device=q.device)
    kept.scatter_(3, torch.where(ids < 0, blocks, ids).long().transpose(1, 2), True)
    kept = kept[..., :blocks].repeat_interleave(case["block"], 3)[..., :n]
    valid = _valid(case, s["lengths"], s["mask"])
    kept &= valid[:, None, None, :]
    if case["causal"]:
        at = s["start"][:, None] + torch.arange(t, device=q.device)
        kept &= torch.arange(n, device=q.device) <= at[:, None, :, None]
    k = torch.where(valid[:, :, None, None], k.float(), 0.0).permute(0, 2, 3, 1).contiguous()
    v = torch.where(valid[:, :, None, None], v.float(), 0.0).permute(0, 2, 1, 3).contiguous()
    q = q.float().view(b, t, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(b, g, (h // g) * t, d)
    p = torch.matmul(q * d ** -0.5, k).view(b, g, h // g, t, n)
    p.masked_fill_(~kept[:, :, None], -float("inf"))
    p -= p.amax(4, keepdim=True).clamp_(min=-1e30)
    p.exp_()
    total = p.sum(4).clamp_(min=1e-30)
    out = torch.matmul(p.view(b, g, (h // g) * t, n), v).view(b, g, h // g, t, d) / total[..., None]
    out = out.permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(s["q"].dtype)
    return {"out": out, "ids": ids}


# ---- the framework's ------------------------------------------------------------------


def _tokens():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from nnunet_mlx.model import tokens

    return tokens


def _own_rotate(s):
    tokens, case = _tokens(), s["case"]
    plan = tokens.RotaryPlan(s["steps"], s["axes"], s["amplitude"])
    return tokens.rotate(s["q"], s["k"], s["positions"], plan, layout=case["layout"], inverse=case["inverse"])


def _own_norm(s):
    tokens, case = _tokens(), s["case"]
    residual, y = tokens.residual_norm(
        s["x"], s["residual"], kind=case["kind"], post=s["post"], pre=s["pre"], gate=s["gate"],
        gate_activation=case["activation"], scale=s["scale"], residual_scale=case["residual_scale"], eps=1e-6)
    return {"residual": residual} if y is None else {"residual": residual, "y": y}


def _own_attend(s):
    tokens, case = _tokens(), s["case"]
    if case["held"]:
        summary = tokens.BlockSummary(s["codes"], s["scales"])
    else:
        summary = tokens.summarize_blocks(s["k"], case["block"], lengths=s["lengths"], key_mask=s["mask"])
    ids = tokens.select_blocks(s["q"], summary, case["block"], case["keep"], causal=case["causal"],
                               start=s["start"], first=case["first"], local=case["local"])
    out = tokens.block_attention(s["q"], s["k"], s["v"], ids, case["block"], causal=case["causal"],
                                 start=s["start"], lengths=s["lengths"], key_mask=s["mask"])
    return {"out": out, "ids": ids}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotate": _own_rotate, "norm": _own_norm, "attend": _own_attend}[op](state)
    return {"rotate": _plain_rotate, "norm": _plain_norm, "attend": _plain_attend}[op](state)


# ---- bytes and operations -------------------------------------------------------------


def work(case):
    if case["op"] == "rotate":
        heads = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * heads * case["dim"] * _BYTES[case["type"]] + 4 * case["tokens"] * case["axes"],
                "flops": 6 * heads * case["rotary"] // 2}
    if case["op"] == "norm":
        n = case["rows"] * case["channels"]
        each = _BYTES[case["type"]] * (1 + case["pre"] + (case["gate"] == "token")) + 2 * _BYTES[case["residual"]]
        return {"bytes": n * each, "flops": n * (3 + 7 * case["post"] + 7 * case["pre"] + 4 * (case["gate"] == "token"))}
    size, block, keep = _BYTES[case["type"]], case["block"], case["keep"]
    t, h, g, d = case["queries"], case["heads"], case["kv_heads"], case["dim"]
    moved = flops = 0
    for n in _lengths(case):
        blocks = -(-n // block)
        if case["causal"]:  # query i sees i + 1 keys
            full = max(0, min(t, n) - keep * block)
            pairs = full * keep * block + sum(range(1, min(t, n) - full + 1)) + (t - min(t, n)) * min(keep * block, n)
            scored = t * blocks / 2
        else:
            pairs, scored = t * min(keep * block, n), t * blocks
        touched = min(n, t * keep * block)
        moved += 2 * t * h * d * size + 4 * t * g * keep + 2 * touched * g * d * size + blocks * g * (d + 4)
        flops += 4 * pairs * h * d + 2 * scored * h * d
    return {"bytes": int(moved), "flops": int(flops)}


# ---- 64 bits --------------------------------------------------------------------------


def _exact_rotate(case, s):
    freqs, axes, amplitude = _frequencies(case)
    freqs = torch.tensor(freqs, dtype=torch.float64, device="cuda")
    angle = s["positions"].double()[:, axes] * freqs
    turn = torch.polar(torch.full_like(angle, amplitude), -angle if case["inverse"] else angle)[:, None, :]
    r = case["rotary"]

    def one(x):
        y = x.double().clone()
        if case["layout"] == "half":
            z = torch.complex(y[..., :r // 2].clone(), y[..., r // 2:r].clone()) * turn
            y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
        else:
            z = torch.complex(y[..., 0:r:2].clone(), y[..., 1:r:2].clone()) * turn
            y[..., 0:r:2], y[..., 1:r:2] = z.real, z.imag
        return y

    return one(s["q"]), one(s["k"])


def _exact_norm(case, s):
    def norm(u, weights):
        shift = u.mean(1, keepdim=True) if case["kind"] == "layer" else 0.0
        spread = ((u - shift) ** 2).mean(1, keepdim=True)
        u = (u - shift) / torch.sqrt(spread + 1e-6) * weights[0].double()
        return u + weights[1].double() if weights[1] is not None else u

    branch = s["x"].double()
    if case["post"]:
        branch = norm(branch, s["post"])
    if case["gate"] == "token":
        gate = s["gate"].double()
        branch = branch * {"none": lambda z: z, "sigmoid": torch.sigmoid,
                           "silu": lambda z: z * torch.sigmoid(z)}[case["activation"]](gate)
    elif case["gate"] == "channel":
        branch = branch * s["scale"].double()
    total = s["residual"].double() * case["residual_scale"] + branch
    return {"residual": total, "y": norm(total, s["pre"])} if case["pre"] else {"residual": total}


def _exact_ids(case, q, k, valid, start):
    """One item and key head: kept blocks of each query, from q (queries, group, dim) and k (keys, dim)."""
    block, n = case["block"], k.shape[0]
    blocks = -(-n // block)
    f32 = np.float32
    codes, scales = np.zeros((blocks, k.shape[1]), np.int64), np.full(blocks, -1, f32)
    for j in range(blocks):
        rows = k[j * block:(j + 1) * block][valid[j * block:(j + 1) * block]]
        if not len(rows):
            continue
        rows = np.where(np.isfinite(rows), rows, f32(0))
        top = np.abs(rows).max()
        scales[j] = 0
        if top < 2.0 ** -60:
            continue
        total = np.rint(rows * (f32(32767) / top)).astype(np.int64).sum(0)
        most = np.abs(total).max()
        if most:
            codes[j] = np.rint(total.astype(f32) * (f32(127) / f32(most)))
            scales[j] = top / (f32(4161409) * f32(len(rows))) * f32(most)
    q = np.where(np.isfinite(q), q, f32(0))
    top = np.abs(q).max(2, keepdims=True)
    top[top < 2.0 ** -60] = 1
    whole = np.rint(q * (f32(127) / top))
    dots = whole.astype(np.float64) @ codes.T.astype(np.float64)  # whole numbers, exact
    score = ((dots.astype(f32) * top) * scales).max(1)
    place = (start + np.arange(q.shape[0])) // block
    index = np.arange(blocks)
    behind = place[:, None] - index[None, :]
    score[(index[None, :] < case["first"]) | ((behind >= 0) & (behind < case["local"]))] = np.inf
    score[:, scales < 0] = -np.inf
    if case["causal"]:
        score[behind < 0] = -np.inf
    order = np.argsort(-score, axis=1, kind="stable")[:, :case["keep"]]
    order[np.take_along_axis(score, order, 1) == -np.inf] = blocks
    order.sort(1)
    ids = np.full((q.shape[0], case["keep"]), -1, np.int32)
    ids[:, :order.shape[1]] = np.where(order == blocks, -1, order)
    return ids


def _exact_attend(case, s):
    b, t, h, d = s["q"].shape
    n, g, block, keep = case["keys"], case["kv_heads"], case["block"], case["keep"]
    blocks = -(-n // block)
    if b * g * t * blocks > 1e8 or b * h * t * keep * block * d > 1e12:
        return None
    valid = np.zeros((b, n), bool)
    for i, length in enumerate(_lengths(case)):
        valid[i, :length] = True
    if s["mask"] is not None:
        valid &= s["mask"].cpu().numpy()
    out = torch.zeros((b, t, h, d), dtype=torch.float64, device="cuda")
    ids = np.zeros((b, t, g, keep), np.int32)
    start = s["start"].cpu().numpy()
    for i in range(b):
        for j in range(g):
            heads = slice(j * (h // g), (j + 1) * (h // g))
            q32, k32 = s["q"][i, :, heads].float().cpu().numpy(), s["k"][i, :, j].float().cpu().numpy()
            ids[i, :, j] = _exact_ids(case, q32, k32, valid[i], start[i])
            keys = torch.from_numpy(ids[i, :, j].astype(np.int64)).cuda()[:, :, None] * block
            keys = torch.where(keys < 0, n, keys + torch.arange(block, device="cuda")).clamp_(max=n).flatten(1)
            ok = torch.cat([torch.from_numpy(valid[i]).cuda(), torch.zeros(1, dtype=torch.bool, device="cuda")])
            zero = torch.zeros((1, d), dtype=torch.float64, device="cuda")
            k64 = torch.cat([s["k"][i, :, j].double(), zero])
            v64 = torch.cat([s["v"][i, :, j].double(), zero])
            k64[~ok], v64[~ok] = 0, 0
            step = max(1, int(2e8) // (keep * block * d))
            for lo in range(0, t, step):
                rows = keys[lo:lo + step]
                see = ok[rows]
                if case["causal"]:
                    at = int(start[i]) + torch.arange(lo, lo + len(rows), device="cuda")
                    see &= rows <= at[:, None]
                logits = torch.bmm(s["q"][i, lo:lo + step, heads].double() * d ** -0.5,
                                   k64[rows].transpose(1, 2).contiguous())
                logits = logits.masked_fill(~see[:, None], -math.inf)
                top = logits.amax(2, keepdim=True)
                weight = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
                total = weight.sum(2, keepdim=True)
                out[i, lo:lo + step, heads] = torch.bmm(weight, v64[rows]) / torch.where(total == 0, 1.0, total)
    return {"out": out, "ids": torch.from_numpy(ids).cuda()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "norm": _exact_norm, "attend": _exact_attend}[case["op"]](case, s)
