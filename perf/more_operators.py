"""The workloads of a volume that is held in 8 bits and of products with 4-bit weights.

A prompted point is answered against the tokens of a volume that stays on the GPU: new tokens
are quantised into it and read back ("hold"), the point's queries attend to it ("attend"), and
the point's own products use weights of 4 bits ("linear").  ``listed`` and ``draw`` give cases,
``prepare`` a case's inputs on the GPU, ``run`` one pass, with ``own`` through
``nnunet_mlx.model.tokens`` and else in elementary float32 torch operations, ``exact`` the
result in float64 and ``work`` the bytes and operations of one pass.

Token counts are those of the networks' patches (a 128^3 patch is 4096 cubes of 8^3 voxels and
32768 of 4^3, a 128 x 160 x 160 patch 6400 of 8^3); 320 channels, five heads of 64, is the width
of the networks' bottom stages.

Held tokens lie in slots, a multiple of 64 for an item.  Keys: codes int8 (batch, kv_heads,
slots, dim); values: codes int8 (batch, kv_heads, slots / 64, dim, 64), where slot 16 t + 4 g + i
of 64 stands at place 16 g + 4 t + i; scales float32 (batch, kv_heads, slots) of both.

Packed weights (outputs, inputs): codes uint8 (ceil(outputs / 16), ceil(inputs / 128), 64, 16):
byte 4 j + b of place 16 g + n holds inputs 32 j + 8 g + 2 b (low four bits) and the next of
output n of 16; scales float32 (ceil(outputs / 16), ceil(inputs / 128) * 128 / group, 16).
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
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # of a 4-bit code's low three bits; the fourth is the sign


# ---- the cases ------------------------------------------------------------------------


def _hold(**kw):
    base = dict(op="hold", type="bf16", batch=1, tokens=1, slots=64, heads=5, dim=64, ragged=False)
    return {**base, **kw}


def _attend(**kw):
    base = dict(op="attend", type="bf16", batch=1, queries=1, keys=1, heads=5, kv_heads=5, dim=64,
                causal=False, ragged=False, masked=False)
    return {**base, **kw}


def _linear(**kw):
    base = dict(op="linear", type="bf16", rows=1, inputs=320, outputs=320, group=64, bias=False, gated=False,
                activation="none")
    return {**base, **kw}


def listed():
    return [
        # one more token of a coarse patch that is held
        _hold(name="hold_point", slots=4160),
        # batches of slices' tokens of different lengths in float32, behind what is held already; one item empty
        _hold(name="hold_ragged_fp32", type="fp32", batch=4, tokens=2501, slots=4096, heads=3, dim=80, ragged=True),
        # a fine patch, held at once and read back for the operators that take it whole
        _hold(name="hold_volume", tokens=32768, slots=32768),
        # one prompted point against one coarse patch
        _attend(name="attend_point", keys=4096),
        # prompts against three held volumes of different sizes, eight heads to a key head
        _attend(name="attend_prompts", type="fp16", batch=3, queries=4, keys=131072, heads=16, kv_heads=2,
                dim=128, ragged=True),
        # two sets of clicked points in float32 against odd numbers of tokens, background masked
        _attend(name="attend_points_fp32", type="fp32", batch=2, queries=37, keys=6399, heads=6, kv_heads=3,
                dim=80, masked=True),
        # an ordered sequence of slices' tokens over itself: ragged, one item empty
        _attend(name="attend_order", batch=4, queries=2501, keys=2501, heads=6, kv_heads=3, dim=96, causal=True,
                ragged=True),
        # a coarse patch's tokens against the held fine ones
        _attend(name="attend_fine", queries=4096, keys=32768),
        # a point's queries, keys and values
        _linear(name="linear_point", outputs=960, bias=True),
        # the gated half of a wide point's feed-forward
        _linear(name="linear_gated_point", inputs=4096, outputs=16384, group=128, gated=True, activation="silu"),
        # odd sizes in float32
        _linear(name="linear_points_fp32", type="fp32", rows=37, inputs=1331, outputs=1000, group=32, bias=True),
        # the narrowing half of a feed-forward over a coarse patch
        _linear(name="linear_patch", type="fp16", rows=4096, inputs=1280, outputs=320),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_hold(rng):
    tokens = _log(rng, 1, 32768)
    batch = rng.randint(1, 4)
    return _hold(type=rng.choice(list(_TYPES)), batch=batch, tokens=tokens, heads=rng.randint(1, 8),
                 slots=64 * (-(-tokens // 64) + rng.choice([0, 1, 1, rng.randint(1, 64)])), dim=16 * rng.randint(1, 8),
                 ragged=batch > 1 and rng.random() < 0.6)


def _draw_attend(rng):
    kv = rng.randint(1, 6)
    few = rng.random() < 0.6
    keys = _log(rng, 60, 131072 if few else 8192)
    queries = _log(rng, 1, 64) if few else keys if rng.random() < 0.5 else _log(rng, 64, 4096)
    batch = rng.randint(1, 4)
    return _attend(type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), batch=batch, queries=queries, keys=keys,
                   heads=kv * rng.choice([1, 1, 2, 4, 8]), kv_heads=kv, dim=16 * rng.randint(1, 8),
                   causal=queries <= keys and rng.random() < 0.3, ragged=batch > 1 and rng.random() < 0.5,
                   masked=rng.random() < 0.4)


def _draw_linear(rng):
    gated = rng.random() < 0.4
    return _linear(type=rng.choice(["bf16", "bf16", "fp16", "fp32"]), rows=_log(rng, 1, 4096),
                   inputs=_log(rng, 33, 16384), outputs=_log(rng, 17, 16384), group=rng.choice([32, 64, 128]),
                   bias=rng.random() < 0.5, gated=gated,
                   activation=rng.choice(["none", "sigmoid", "silu"]) if gated else "none")


def draw(rng):
    make = rng.choice([_draw_hold, _draw_attend, _draw_attend, _draw_linear, _draw_linear])
    while True:
        case = make(rng)
        most = [(work(c), _cost(c)) for c in listed() if c["op"] == case["op"]]
        asked = work(case)
        if (asked["bytes"] <= max(w["bytes"] for w, _ in most) and asked["flops"] <= max(w["flops"] for w, _ in most)
                and _cost(case) <= max(c for _, c in most)):
            return case


def _cost(case):
    """Elements that the plain form holds at once."""
    if case["op"] == "hold":
        return case["batch"] * case["slots"] * case["heads"] * case["dim"]
    if case["op"] == "attend":
        return case["batch"] * case["heads"] * case["queries"] * case["keys"]
    return (1 + case["gated"]) * (case["inputs"] + case["rows"]) * case["outputs"] + case["rows"] * case["inputs"]


# ---- the inputs -----------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _quantise(x):
    """Codes (whole numbers in float32) and scales of the last axis."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    odd, tiny = ~torch.isfinite(top), top < 2.0 ** -60
    safe = torch.where(odd | tiny, 1.0, top)
    up = torch.div(torch.full_like(safe, 127.0), safe)
    codes = torch.where(odd | tiny, 0.0, torch.round(x * up))
    scales = torch.div(torch.clamp(safe, max=3.4028233e38), torch.full_like(safe, 127.0))
    return codes, torch.where(tiny, 0.0, torch.where(odd, float("nan"), scales))[..., 0]


def _tile(codes):
    """Values' codes (batch, heads, slots, dim) in the order in which they are held."""
    return codes.unflatten(2, (-1, 4, 4, 4)).permute(0, 1, 2, 6, 4, 3, 5).flatten(4).contiguous()


def _untile(codes):
    return codes.unflatten(4, (4, 4, 4)).permute(0, 1, 2, 5, 4, 6, 3).flatten(2, 5)


def _held(case, k, v, slots):
    """The held form of k and v (batch, tokens, heads, dim); what lies behind them is zero."""
    out = []
    for x in (k, v):
        codes, scales = _quantise(x.transpose(1, 2))
        codes = torch.nn.functional.pad(codes, (0, 0, 0, slots - x.shape[1])).to(torch.int8)
        out += [codes.contiguous(), torch.nn.functional.pad(scales, (0, slots - x.shape[1])).contiguous()]
    return {"k_codes": out[0], "k_scales": out[1], "v_codes": _tile(out[2]), "v_scales": out[3]}


def _prepare_hold(case, gen):
    b, t, s, h, d = (case[k] for k in ("batch", "tokens", "slots", "heads", "dim"))
    # keys and values of one projection, side by side; channels of very different size
    sizes = torch.exp(_randn(gen, 2 * h, d))
    kv = (_randn(gen, b, t, 2 * h, d) * sizes).to(_TYPES[case["type"]])
    lengths = torch.tensor(_lengths(case, t), dtype=torch.int32, device="cuda")
    start = torch.randint(0, s - t + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
    before = _randn(gen, 2, b, s, h, d)
    return {"case": case, "k": kv[:, :, :h], "v": kv[:, :, h:], "lengths": lengths, "start": start,
            **_held(case, before[0], before[1], s)}


def _lengths(case, n):
    """Tokens of each item: the whole, or falling by an odd step down to an empty item."""
    b = case["batch"]
    if not case["ragged"]:
        return [n] * b
    return [n] + [max(0, n - i * (n // (b - 1)) - 7) if b > 3 else max(0, n - i * (n // 4) - 7) for i in range(1, b)]


def _prepare_attend(case, gen):
    b, t, n, h, g, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "dim"))
    slots = -(-n // 64) * 64
    # token features: runs of 32 prototypes that recur along the volume, and noise
    kinds = _randn(gen, 32, g, d)
    runs = torch.randint(0, 32, (b, n // 96 + 1), generator=gen, device="cuda")
    k = kinds[runs[:, torch.arange(n, device="cuda") // 96]] + 0.7 * _randn(gen, b, n, g, d)
    v = _randn(gen, b, n, g, d)
    # a query resembles keys like those at some place
    at = torch.arange(t, device="cuda").expand(b, t) if case["causal"] and t == n else \
        torch.randint(0, n, (b, t), generator=gen, device="cuda")
    near = torch.gather(k, 1, at[:, :, None, None].expand(b, t, g, d)).repeat_interleave(h // g, 2)
    q = 0.6 * near + 0.8 * _randn(gen, b, t, h, d)
    mask = None
    if case["masked"]:  # background in runs
        runs = torch.rand((b, n // 48 + 1), generator=gen, device="cuda") < 0.7
        mask = runs[:, torch.arange(n, device="cuda") // 48].contiguous()
    lengths = torch.tensor(_lengths(case, n), dtype=torch.int32, device="cuda")
    held = _held(case, k, v, slots)
    if case["ragged"]:  # what lies behind an item's end is another's that was held there before
        behind = torch.arange(slots, device="cuda")[None, :] >= lengths[:, None]
        held["k_scales"].masked_fill_(behind[:, None], float("nan"))
        held["v_scales"].masked_fill_(behind[:, None], float("nan"))
    # a causal sequence's queries are its last tokens
    start = torch.full((b,), n - t, dtype=torch.int32, device="cuda") if case["causal"] else None
    return {"case": case, "q": q.to(_TYPES[case["type"]]), "lengths": lengths, "mask": mask, "start": start, **held}


def _pack(case, gen, outputs, inputs):
    """Codes and scales of a random matrix in their packed order."""
    group, padded, blocks = case["group"], -(-outputs // 16) * 16, -(-inputs // 128)
    w = _randn(gen, outputs, inputs) * torch.exp(0.5 * _randn(gen, outputs, 1)) * inputs ** -0.5
    w = torch.nn.functional.pad(w, (0, blocks * 128 - inputs, 0, padded - outputs)).unflatten(1, (-1, group))
    top = w.abs().amax(2, keepdim=True)
    safe = torch.where(top < 2.0 ** -60, 1.0, top)
    size = w.abs() * torch.div(torch.full_like(safe, 6.0), safe)
    code = torch.zeros_like(size, dtype=torch.uint8)
    # half-way values go to the even code
    for i, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):
        code += (size >= border) if i % 2 else (size > border)
    code = code | ((w < 0) & (code > 0)).to(torch.uint8) << 3
    scales = torch.where(top < 2.0 ** -60, 0.0, torch.div(safe, torch.full_like(safe, 6.0)))[..., 0]
    code = code.view(padded // 16, 16, blocks, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)
    codes = (code[..., 0] | code[..., 1] << 4).flatten(4).flatten(2, 3).contiguous()
    return codes, scales.view(padded // 16, 16, -1).transpose(1, 2).contiguous()


def _prepare_linear(case, gen):
    n, i, o = case["rows"], case["inputs"], case["outputs"]
    state = {"case": case, "x": (_randn(gen, n, i) + 0.1).to(_TYPES[case["type"]]), "w": _pack(case, gen, o, i),
             "gate": None, "bias": None}
    if case["gated"]:
        state["gate"] = _pack(case, gen, o, i)
    if case["bias"]:
        state["bias"] = 0.1 * _randn(gen, o)
    return state


def prepare(case, seed):
    gen = _generator(seed)
    make = {"hold": _prepare_hold, "attend": _prepare_attend, "linear": _prepare_linear}[case["op"]]
    return make(case, gen)


# ---- the plain forms ------------------------------------------------------------------


def _plain_hold(s):
    case, t = s["case"], s["case"]["tokens"]
    token = torch.arange(t, device="cuda")
    slot = (s["start"][:, None] + token).long()
    written = (token < s["lengths"][:, None])[:, None, :]
    out = {}
    for name in ("k", "v"):
        codes, scales = s[name + "_codes"], s[name + "_scales"]
        rows = codes if name == "k" else _untile(codes)
        new_codes, new_scales = _quantise(s[name].transpose(1, 2))
        at = slot[:, None, :].expand(new_scales.shape)
        new_scales = torch.where(written, new_scales, torch.gather(scales, 2, at))
        scales.scatter_(2, at, new_scales)
        at = at[..., None].expand(new_codes.shape)
        new_codes = torch.where(written[..., None], new_codes.to(torch.int8), torch.gather(rows, 2, at))
        rows = rows.scatter(2, at, new_codes)
        codes.copy_(rows if name == "k" else _tile(rows))
        out[name] = (rows.float() * scales[..., None]).transpose(1, 2).to(_TYPES[case["type"]]).contiguous()
    return out


def _plain_attend(s):
    case, q = s["case"], s["q"]
    b, t, h, d = q.shape
    n, g = case["keys"], case["kv_heads"]
    seen = torch.arange(n, device="cuda")[None, :] < s["lengths"][:, None]
    if s["mask"] is not None:
        seen = seen & s["mask"]
    k = torch.where(seen[:, None, :, None], s["k_codes"][:, :, :n].float() * s["k_scales"][:, :, :n, None], 0.0)
    v = torch.where(seen[:, None, :, None], _untile(s["v_codes"])[:, :, :n].float() * s["v_scales"][:, :, :n, None], 0.0)
    seen = seen[:, None, None, None, :]
    if case["causal"]:
        at = s["start"][:, None] + torch.arange(t, device="cuda")
        seen = seen & (torch.arange(n, device="cuda") <= at[:, None, None, :, None])
    q = q.float().view(b, t, g, h // g, d).permute(0, 2, 3, 1, 4).reshape(b, g, (h // g) * t, d)
    p = torch.matmul(q * d ** -0.5, k.transpose(2, 3).contiguous()).view(b, g, h // g, t, n)
    p.masked_fill_(~seen, -float("inf"))
    p -= p.amax(4, keepdim=True).clamp_(min=-1e30)
    p.exp_()
    total = p.sum(4).clamp_(min=1e-30)
    out = torch.matmul(p.view(b, g, (h // g) * t, n), v).view(b, g, h // g, t, d) / total[..., None]
    return out.permute(0, 3, 1, 2, 4).reshape(b, t, h, d).to(s["q"].dtype)


def _matrix(case, codes, scales):
    """The matrix (outputs, inputs) that packed codes and scales stand for."""
    tiles, blocks = codes.shape[:2]
    code = torch.stack([codes & 15, codes >> 4], -1).view(tiles, blocks, 4, 16, 4, 4, 2).permute(0, 3, 1, 4, 2, 5, 6)
    levels = torch.tensor(_LEVELS + tuple(-x for x in _LEVELS), device="cuda")
    w = levels[code.reshape(tiles * 16, -1, case["group"]).int()]
    w = w * scales.transpose(1, 2).reshape(tiles * 16, -1, 1)
    return w.flatten(1)[:case["outputs"], :case["inputs"]]


def _plain_linear(s):
    case, x = s["case"], s["x"].float()
    y = torch.matmul(x, _matrix(case, *s["w"]).t())
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["gate"] is not None:
        gate = torch.matmul(x, _matrix(case, *s["gate"]).t())
        if case["activation"] != "none":
            open_ = 1.0 / (1.0 + torch.exp(-gate))
            gate = open_ if case["activation"] == "sigmoid" else gate * open_
        y = gate * y
    return y.to(s["x"].dtype)


# ---- the framework's ------------------------------------------------------------------


def _tokens():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from nnunet_mlx.model import tokens

    return tokens


def _own_hold(s):
    tokens = _tokens()
    held = tokens.HeldTokens(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    tokens.hold_tokens(held, s["k"], s["v"], start=s["start"], lengths=s["lengths"])
    k, v = tokens.read_held(held, s["k"].dtype)
    return {"k": k, "v": v}


def _own_attend(s):
    tokens = _tokens()
    held = tokens.HeldTokens(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    return tokens.held_attention(s["q"], held, s["lengths"], causal=s["case"]["causal"], start=s["start"],
                                 key_mask=s["mask"])


def _own_linear(s):
    tokens, case = _tokens(), s["case"]
    w, gate = (None if p is None else tokens.PackedWeight(*p, case["outputs"], case["inputs"], case["group"])
               for p in (s["w"], s["gate"]))
    return tokens.packed_linear(s["x"], w, bias=s["bias"], gate=gate, gate_activation=case["activation"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"hold": _own_hold, "attend": _own_attend, "linear": _own_linear}[op](state)
    return {"hold": _plain_hold, "attend": _plain_attend, "linear": _plain_linear}[op](state)


# ---- bytes and operations -------------------------------------------------------------


def work(case):
    size = _BYTES[case["type"]]
    if case["op"] == "hold":
        each = case["heads"] * case["dim"]
        new = sum(_lengths(case, case["tokens"]))
        moved = new * (each * (size + 1) + 4 * case["heads"])
        moved += case["batch"] * case["slots"] * (each * (size + 1) + 4 * case["heads"])
        return {"bytes": 2 * moved, "flops": 8 * new * each + 2 * case["batch"] * case["slots"] * each}
    if case["op"] == "attend":
        t, h, g, d = case["queries"], case["heads"], case["kv_heads"], case["dim"]
        moved = flops = 0
        for n in _lengths(case, case["keys"]):
            pairs = t * n
            if case["causal"]:  # the i-th query sees keys - queries + i + 1 keys, no more than there are
                first = case["keys"] - t + 1
                whole = max(0, t - max(0, n - first))
                pairs = whole * n + (t - whole) * first + (t - whole) * (t - whole - 1) // 2
            moved += 2 * t * h * d * size + 2 * n * g * (d + 4) + n * case["masked"]
            flops += 4 * pairs * h * d
        return {"bytes": int(moved), "flops": int(flops)}
    n, i, o = case["rows"], case["inputs"], case["outputs"]
    weights = (1 + case["gated"]) * (o * i // 2 + 4 * o * -(-i // case["group"]))
    return {"bytes": weights + n * (i + o) * size + 4 * o * case["bias"],
            "flops": 2 * (1 + case["gated"]) * n * i * o}


# ---- 64 bits --------------------------------------------------------------------------


def _exact_hold(case, s):
    f32 = np.float32
    token = np.arange(case["tokens"])
    lengths, start = _lengths(case, case["tokens"]), s["start"].cpu().numpy()
    places = [int(16 * (j // 4 % 4) + 4 * (j // 16) + j % 4) for j in range(64)]  # of slot j among 64
    out = {}
    for name in ("k", "v"):
        codes = s[name + "_codes"].cpu().numpy()
        if name == "v":
            codes = codes[..., places].swapaxes(3, 4).reshape(s["k_codes"].shape)
        value = codes.astype(np.float64) * s[name + "_scales"].double().cpu().numpy()[..., None]
        value = np.ascontiguousarray(value.transpose(0, 2, 1, 3))  # (batch, slots, heads, dim)
        x = s[name].float().cpu().numpy()
        top = np.abs(x).max(-1, keepdims=True)
        with np.errstate(divide="ignore", over="ignore"):
            code = np.where(top < 2.0 ** -60, f32(0), np.rint(x * (f32(127) / top)))
        new = code.astype(np.float64) * np.where(top < 2.0 ** -60, f32(0), top / f32(127)).astype(np.float64)
        for b, length in enumerate(lengths):
            value[b, start[b] + token[:length]] = new[b, :length]
        out[name] = torch.from_numpy(value)
    return out


def _exact_attend(case, s):
    b, t, h, d = s["q"].shape
    n, g = case["keys"], case["kv_heads"]
    if b * h * t * n * d > 1e11:
        return None
    place = torch.arange(64, device="cuda").view(4, 4, 4).transpose(0, 1).reshape(64)  # of each slot of 64
    out = torch.zeros((b, t, h, d), dtype=torch.float64, device="cuda")
    for item, length in enumerate(_lengths(case, n)):
        see = torch.zeros(n, dtype=torch.bool, device="cuda")
        see[:length] = True
        if s["mask"] is not None:
            see &= s["mask"][item]
        see = torch.nonzero(see)[:, 0]
        if not len(see):
            continue
        for j in range(g):
            k = s["k_codes"][item, j].double()[see] * s["k_scales"][item, j].double()[see, None]
            v = s["v_codes"][item, j].double()[:, :, place].transpose(1, 2).reshape(-1, d)[see]
            v = v * s["v_scales"][item, j].double()[see, None]
            for head in range(j * (h // g), (j + 1) * (h // g)):
                step = max(1, int(2e8) // len(see))
                for lo in range(0, t, step):
                    logits = s["q"][item, lo:lo + step, head].double() @ k.t() / math.sqrt(d)
                    if case["causal"]:
                        at = n - t + torch.arange(lo, lo + len(logits), device="cuda")
                        logits = logits.masked_fill(see > at[:, None], -math.inf)
                    top = logits.amax(1, keepdim=True)
                    weight = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
                    total = weight.sum(1, keepdim=True)
                    out[item, lo:lo + step, head] = weight @ v / torch.where(total == 0, 1.0, total)
    return out


def _exact_matrix(case, codes, scales):
    """By the definition of the packed order, an output and a place of 128 inputs at a time."""
    o, i = case["outputs"], case["inputs"]
    levels = np.array(_LEVELS + tuple(-x for x in _LEVELS))
    row, column = np.arange(o)[:, None], np.arange(i)[None, :]
    at = column % 128
    byte = codes.cpu().numpy()[row // 16, column // 128, 16 * (at % 32 // 8) + row % 16, 4 * (at // 32) + at % 8 // 2]
    code = np.where(at % 2 == 1, byte >> 4, byte & 15)
    return torch.from_numpy(levels[code] * scales.double().cpu().numpy()[row // 16, column // case["group"], row % 16])


def _exact_linear(case, s):
    x = s["x"].double()
    y = x @ _exact_matrix(case, *s["w"]).cuda().t()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if s["gate"] is None:
        return y
    gate = x @ _exact_matrix(case, *s["gate"]).cuda().t()
    return y * {"none": lambda z: z, "sigmoid": torch.sigmoid, "silu": lambda z: z * torch.sigmoid(z)}[case["activation"]](gate)


def exact(case, seed):
    s = prepare(case, seed)
    return {"hold": _exact_hold, "attend": _exact_attend, "linear": _exact_linear}[case["op"]](case, s)
