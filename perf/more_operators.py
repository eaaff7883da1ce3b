"""What stands around the experts of a block, as cases that can be timed and compared.

Three operators, each in its plain form (``own`` false: elementary torch operations in 32 bits, in 64 where an order or
an 8-bit border hangs on it, rounded once at the end) and as calls of ``veymoe`` (``own`` true):

* ``route``   from a router's logits to experts (``routing.select_experts``): softmax or sigmoid scores, a balance bias
              that decides the choice but not the weight, groups of experts of which the best are kept, top-k, weights
              renormalised and scaled;
* ``block``   the norm behind a block, its gate and scale, the residual's addition and the norm in front of the next
              block (``norm.block_norm``): output in the input's type or in MX (e4m3 values, e8m0 scales per 32);
* ``linear``  a matrix product with bias, activation and residual in its epilogue (``linear.linear``): bf16 or MX
              operands, output in bf16 or fp32.

Widths: the small layer (hidden 1024, intermediate 256, 64 experts top-4), the full-size layer (2048 / 512, 512 experts
top-10) and the checkpoint's widths (2560 / 640, the same routing), and odd sizes around them.  Activations are N(0, 1),
weights N(0, 1/in), router logits N(0, 1.5^2).
"""
from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

EPS = 1e-6
GROUP = 32          # values that share one scale
E4M3_MAX = 448.0
ACTIVATIONS = (None, "relu", "silu", "gelu", "gelu_tanh", "sigmoid", "swiglu")


def _route(name, rows, experts, top_k, scoring="softmax", dtype="fp32", bias=False, groups=1, top_groups=1, group_top=1,
           renormalize=True, scale=1.0, closed=0):
    return {"name": name, "op": "route", "rows": rows, "experts": experts, "top_k": top_k, "scoring": scoring,
            "dtype": dtype, "bias": bias, "groups": groups, "top_groups": top_groups, "group_top": group_top,
            "renormalize": renormalize, "scale": scale, "closed": closed}


def _block(name, rows, width, dtype="bf16", residual="bf16", post=True, gate="none", sigmoid=False, scale=1.0,
           residual_scale=1.0, quantize=False, pad=0, centered=True):
    return {"name": name, "op": "block", "rows": rows, "width": width, "dtype": dtype, "residual": residual,
            "post": post, "gate": gate, "sigmoid": sigmoid, "scale": scale, "residual_scale": residual_scale,
            "quantize": quantize, "pad": pad, "centered": centered}


def _linear(name, rows, k, n, fmt="bf16", activation="none", bias=False, residual="none", out="bf16"):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "format": fmt, "activation": activation,
            "bias": bias, "residual": residual, "out": out}


def listed():
    return [
        # one decode token over all experts: latency
        _route("route_token", 1, 512, 10),
        # batched decode with a balance bias and groups, logits of a bf16 projection
        _route("route_batch_37", 37, 256, 8, "sigmoid", "bf16", True, 8, 4, 2, scale=2.5),
        # a window of prefill chunks, biased, of which some experts are closed
        _route("route_window_8192", 8192, 512, 10, "sigmoid", bias=True, scale=2.5, closed=9),
        # between two blocks of one decode token: latency
        _block("block_token", 1, 2560),
        # a short prompt, residual stream in fp32, the branch under its row's sigmoid gate
        _block("block_prompt_333", 333, 2048, residual="fp32", gate="row", sigmoid=True, pad=64),
        # a window of prefill chunks, scaled branch, 8 bits out for the next products
        _block("block_window_8192", 8192, 2560, scale=0.22, quantize=True, centered=False),
        # a projection of one decode token with its residual
        _linear("linear_token", 1, 2560, 2560, residual="bf16"),
        # gate/up of the shared expert in batched decode, 8 bits
        _linear("linear_batch_mx_32", 32, 2560, 640, "mx8", "swiglu"),
        # an odd prompt through an odd projection
        _linear("linear_prompt_333", 333, 1000, 1333, activation="gelu", bias=True),
        # router logits of a prefill chunk, kept in fp32
        _linear("linear_logits_2048", 2048, 2048, 512, out="fp32"),
        # gate/up of the shared expert over a window, 8 bits
        _linear("linear_window_mx_8192", 8192, 2560, 640, "mx8", "swiglu"),
        # a full projection over a window, with everything in its epilogue
        _linear("linear_window_8192", 8192, 2560, 2560, activation="silu", bias=True, residual="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_route(rng):
    if rng.random() < 0.5:
        experts, groups = rng.choice(((64, 1), (64, 4), (256, 8), (256, 1), (512, 1), (512, 8)))
    else:
        groups = rng.choice((1, 1, 1, 2, 3, 5, 8, 16))
        experts = groups * rng.randint(max(2, 8 // groups), max(2, 640 // groups))
    top_groups = rng.randint(1, groups)
    top_k = min(rng.choice((1, 2, 4, 6, 8, 10, 16)), top_groups * (experts // groups))
    scoring = rng.choice(("softmax", "sigmoid"))
    rows = _log(rng, 1, 8192 if experts <= 512 else 6000)
    return _route("", rows, experts, top_k, scoring, rng.choice(("fp32", "fp32", "bf16")), rng.random() < 0.6, groups,
                  top_groups, rng.choice((1, 2)), rng.random() < 0.8, rng.choice((1.0, 1.0, 2.5)),
                  rng.choice((0, 0, rng.randint(0, experts // 8))))


def _draw_block(rng):
    quantize = rng.random() < 0.4
    dtype = "fp32" if rng.random() < 0.25 else "bf16"
    if rng.random() < 0.6:
        width = rng.choice((1024, 2048, 2560, 4096, 8192))
    else:
        width = 32 * rng.randint(2, 200) if quantize else rng.randint(33, 6500)
    gate = rng.choice(("none", "none", "row", "channel", "value"))
    residual = rng.choice(("bf16", "fp32"))
    size = (4 if dtype == "fp32" else 2) * (3 if gate == "value" else 2) + (8 if residual == "fp32" else 4)
    rows = _log(rng, 1, max(2, min(8192, 8192 * 2560 * 7 // (width * size))))
    return _block("", rows, width, dtype, residual, rng.random() < 0.8, gate, rng.random() < 0.5,
                  rng.choice((1.0, 1.0, 0.22)), rng.choice((1.0, 1.0, 1.41)), quantize, rng.choice((0, 0, 8, 40)),
                  rng.random() < 0.6)


def _draw_linear(rng):
    fmt = rng.choice(("bf16", "bf16", "mx8"))
    unit = 32 if fmt == "mx8" else 8
    k = rng.choice((512, 640, 1024, 2048, 2560, unit * rng.randint(64 // unit, 2560 // unit)))
    n = rng.choice((256, 512, 640, 1024, 2048, 2560, rng.randint(33, 2560), rng.randint(33, 2560)))
    activation = rng.choice(ACTIVATIONS) or "none"
    if activation == "swiglu":
        n = min(n, 1280)
    return _linear("", _log(rng, 1, 8192), k, n, fmt, activation, rng.random() < 0.5, rng.choice(("none", "bf16", "fp32")),
                   rng.choice(("bf16", "bf16", "fp32")))


def draw(rng):
    c = rng.choices((_draw_route, _draw_block, _draw_linear), (3, 3, 5))[0](rng)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs --

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(shape, gen, scale=1.0, dtype=torch.bfloat16):
    x = torch.empty(shape, device="cuda", dtype=dtype)
    return x.normal_(0.0, scale, generator=gen)


def _to_mx(v):
    """(e4m3 values, e8m0 scales) of rows whose width divides into groups, in the values' own precision: the scale is the
    least power of two that keeps the group's largest value within e4m3's range."""
    g = v.reshape(*v.shape[:-1], -1, GROUP)
    big = g.abs().amax(-1, keepdim=True)
    m, x = torch.frexp(big)                                # big = m 2^x, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(big > 0, torch.where(m <= 0.875, x - 9, x - 8), -127).clamp(min=-127)
    v8 = g * torch.ldexp(torch.ones_like(big), -e)
    step = torch.ldexp(torch.ones_like(v8), torch.frexp(v8).exponent.clamp(min=-5) - 4)
    q = (torch.round(v8 / step) * step).to(torch.float8_e4m3fn)
    return q.reshape(v.shape), (e + 127).squeeze(-1).to(torch.uint8).view(torch.float8_e8m0fnu)


def _from_mx(values, scales):
    e = scales.view(torch.uint8).to(torch.int32) - 127
    s = torch.ldexp(torch.ones(e.shape, device=e.device), e)
    return (values.float().reshape(*scales.shape, GROUP) * s[..., None]).reshape(values.shape)


def prepare(case, seed):
    gen = _gen(seed)
    s = {"op": case["op"], "case": dict(case)}
    rows = case["rows"]
    if case["op"] == "route":
        s["logits"] = _normal((rows, case["experts"]), gen, 1.5, _TYPES[case["dtype"]])
        if case["closed"]:       # experts that no token may take
            s["logits"][:, torch.randperm(case["experts"], device="cuda", generator=gen)[:case["closed"]]] = -math.inf
        s["bias"] = _normal((case["experts"],), gen, 0.05, torch.float32) if case["bias"] else None
    elif case["op"] == "block":
        width, dtype = case["width"], _TYPES[case["dtype"]]
        wide = (rows, width + case["pad"])
        s["x"] = _normal(wide, gen, dtype=dtype)[:, :width]
        s["residual"] = _normal(wide, gen, 2.0, _TYPES[case["residual"]])[:, :width]
        shape = {"none": None, "row": (rows, 1), "channel": (width,), "value": (rows, width)}[case["gate"]]
        s["gate"] = None if shape is None else _normal(shape, gen, dtype=dtype)
        at = 1.0 if case["centered"] else 0.0
        s["weight"], post = (at + 0.2 * torch.randn((2, width), device="cuda", generator=gen)).to(dtype)
        s["post"] = post if case["post"] else None
    else:
        k, n = case["k"], case["n"] * (2 if case["activation"] == "swiglu" else 1)
        x, w = _normal((rows, k), gen), _normal((n, k), gen, k ** -0.5)
        s["x"], s["weight"] = (_to_mx(x.float()), _to_mx(w.float())) if case["format"] == "mx8" else (x, w)
        s["bias"] = _normal((n,), gen, 0.5) if case["bias"] else None
        s["residual"] = None if case["residual"] == "none" else _normal((rows, case["n"]), gen, 1.0, _TYPES[case["residual"]])
    return s


# ------------------------------------------------------------ plain forms --

def _route_plain(s):
    case = s["case"]
    l, b = s["logits"].double(), s["bias"]          # 64 bits: the order of close choices
    rows, experts = l.shape
    closed = l == -math.inf
    if case["scoring"] == "softmax":
        top = l.amax(-1, keepdim=True)
        e = torch.exp(l - torch.where(top == -math.inf, 0.0, top))
        score = torch.where(closed, 0.0, e / e.sum(-1, keepdim=True))
    else:
        score = 1.0 / (1.0 + torch.exp(-l))
    # without a bias the logits order the experts as their scores do, even where scores are too small to differ
    choice = l if b is None else torch.where(closed, -math.inf, score + b.double())
    if case["groups"] > 1:
        per = experts // case["groups"]
        rank = choice if case["group_top"] == 1 else torch.where(closed, -math.inf, score if b is None else choice)
        best = rank.reshape(rows, case["groups"], per).sort(dim=-1, descending=True).values[..., :case["group_top"]]
        rank = torch.where(best[..., 0] == -math.inf, -math.inf, torch.where(best == -math.inf, 0.0, best).sum(-1))
        kept = rank.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros((rows, case["groups"]), device=l.device, dtype=torch.bool).scatter_(1, kept, True)
        choice = torch.where(keep.repeat_interleave(per, 1), choice, -math.inf)
    best, inds = choice.sort(dim=-1, descending=True, stable=True)
    best, inds = best[:, :case["top_k"]], inds[:, :case["top_k"]]
    none = best == -math.inf
    w = torch.where(none, 0.0, score.gather(1, inds))
    if case["renormalize"]:
        total = w.sum(-1, keepdim=True)
        w = torch.where(total == 0.0, 0.0, w / total)
    return [torch.where(none, -1, inds).to(torch.int32), (w * case["scale"]).float()]


def _block_plain(s):
    case = s["case"]
    wide = torch.float64 if case["quantize"] else torch.float32      # 64 bits: values next to e4m3's borders
    x, r = s["x"].to(wide), s["residual"].to(wide)
    gain = lambda w: w.to(wide) + (0.0 if case["centered"] else 1.0)  # noqa: E731
    if s["post"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gain(s["post"])
    if s["gate"] is not None:
        g = s["gate"].to(wide)
        x = x * (1.0 / (1.0 + torch.exp(-g)) if case["sigmoid"] else g)
    h = r * case["residual_scale"] + x * case["scale"]
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * gain(s["weight"])
    return [*(_to_mx(y) if case["quantize"] else [y.to(s["x"].dtype)]), h.to(s["residual"].dtype)]


def _activated(y, name):
    if name == "relu":
        return y.clamp(min=0.0)
    if name == "silu":
        return y / (1.0 + torch.exp(-y))
    if name == "gelu":
        return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-y))
    if name == "swiglu":
        gate, up = y.chunk(2, -1)
        return gate / (1.0 + torch.exp(-gate)) * up
    return y


def _linear_plain(s):
    case = s["case"]
    x, w = (_from_mx(*s["x"]), _from_mx(*s["weight"])) if case["format"] == "mx8" else (s["x"].float(), s["weight"].float())
    y = torch.matmul(x, w.t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    y = _activated(y, case["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return [y.to(_TYPES[case["out"]])]


# ------------------------------------------------------- the package's calls --

@functools.lru_cache(None)
def _package():
    path = os.path.join(os.getcwd(), "veystrix-core_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import veymoe.linear
    import veymoe.norm
    import veymoe.routing
    return veymoe


def _route_own(s):
    case = s["case"]
    return list(_package().routing.select_experts(
        s["logits"], case["top_k"], scoring=case["scoring"], bias=s["bias"], groups=case["groups"],
        top_groups=case["top_groups"], group_top=case["group_top"], renormalize=case["renormalize"], scale=case["scale"]))


def _block_own(s):
    case = s["case"]
    y, h = _package().norm.block_norm(
        s["x"], s["residual"], s["weight"], post_weight=s["post"], gate=s["gate"], sigmoid_gate=case["sigmoid"],
        scale=case["scale"], residual_scale=case["residual_scale"], eps=EPS, one_centered=case["centered"],
        quantize=case["quantize"])
    return [*(y if case["quantize"] else [y]), h]


def _linear_own(s):
    case, v = s["case"], _package()
    x, w = s["x"], s["weight"]
    if case["format"] == "mx8":
        x, w = v.norm.MxTensor(*x), v.norm.MxTensor(*w)
    return [v.linear.linear(x, w, s["bias"], activation=None if case["activation"] == "none" else case["activation"],
                            residual=s["residual"], dtype=_TYPES[case["out"]])]


def run(state):
    if own:
        return {"route": _route_own, "block": _block_own, "linear": _linear_own}[state["op"]](state)
    return {"route": _route_plain, "block": _block_plain, "linear": _linear_plain}[state["op"]](state)


# ------------------------------------------------------------------- work --

_BYTES = {"bf16": 2, "fp32": 4, "none": 0, "mx8": 1 + 1 / GROUP}


def work(case):
    rows = case["rows"]
    if case["op"] == "route":
        experts = case["experts"]
        return {"bytes": rows * (experts * _BYTES[case["dtype"]] + case["top_k"] * 8) + (4 * experts if case["bias"] else 0),
                "flops": 6 * rows * experts}
    if case["op"] == "block":
        values, size = rows * case["width"], _BYTES[case["dtype"]]
        gate = {"none": 0, "row": rows, "channel": case["width"], "value": values}[case["gate"]]
        out = _BYTES["mx8"] if case["quantize"] else size
        return {"bytes": values * (size + 2 * _BYTES[case["residual"]] + out) + gate * size
                + case["width"] * size * (2 if case["post"] else 1), "flops": 11 * values}
    k, n = case["k"], case["n"] * (2 if case["activation"] == "swiglu" else 1)
    return {"bytes": (rows + n) * k * _BYTES[case["format"]] + (2 * n if case["bias"] else 0)
            + rows * case["n"] * (_BYTES[case["out"]] + _BYTES[case["residual"]]), "flops": 2 * rows * k * n}


# ------------------------------------------------------------ in 64 bits --

def _mx_exact(y):
    """y in MX by the definition: per group of 32 the least 2^e >= 2^-127 with max|y| <= 448 * 2^e; y / 2^e to the
    nearest multiple of its binade's e4m3 step (eighths, 2^-9 at the least), ties to even."""
    g = y.unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    e = torch.ceil(torch.log2(top / E4M3_MAX))
    e = torch.where(top <= E4M3_MAX * torch.exp2(e - 1), e - 1, e)      # log2 next to a whole number
    e = torch.where(top > E4M3_MAX * torch.exp2(e), e + 1, e).clamp(min=-127)
    scale = torch.exp2(e)
    v = g / scale[..., None]
    step = torch.exp2(torch.frexp(v).exponent.double().clamp(min=-5) - 4)
    return (torch.round(v / step) * step).flatten(-2), scale


def _first_largest(c):
    """Index of each row's largest value, the lowest of several."""
    at = torch.arange(c.shape[-1], device=c.device).expand_as(c)
    return torch.where(c == c.amax(-1, keepdim=True), at, c.shape[-1]).amin(-1, keepdim=True)


def _route_exact(case, s):
    l = s["logits"].double()
    rows, experts = l.shape
    score = torch.softmax(l, -1) if case["scoring"] == "softmax" else torch.sigmoid(l)
    choice = l.clone() if s["bias"] is None else score + s["bias"].double()
    choice[torch.isneginf(l)] = -math.inf
    per = experts // case["groups"]
    if case["groups"] > 1:
        left = choice.clone()
        if s["bias"] is None and case["group_top"] == 2:
            left = torch.where(torch.isneginf(l), -math.inf, score)
        rank = torch.zeros((rows, case["groups"]), device=l.device, dtype=torch.float64)
        for g in range(case["groups"]):          # the group's best, one after the other
            part = left[:, g * per:(g + 1) * per].clone()
            for j in range(min(case["group_top"], per)):
                at = _first_largest(part)
                best = part.gather(1, at)[:, 0]
                rank[:, g] += best if j == 0 else torch.where(torch.isneginf(best), 0.0, best)
                part.scatter_(1, at, -math.inf)
        lost = torch.ones((rows, experts), device=l.device, dtype=torch.bool)
        for _ in range(case["top_groups"]):
            g = _first_largest(rank)
            rank.scatter_(1, g, -math.inf)
            lost &= torch.arange(experts, device=l.device) // per != g
        choice[lost] = -math.inf
    inds, w = [], []
    for _ in range(case["top_k"]):
        at = _first_largest(choice)
        none = torch.isneginf(choice.gather(1, at))
        inds.append(torch.where(none, -1, at))
        w.append(torch.where(none, 0.0, score.gather(1, at)))
        choice.scatter_(1, at, -math.inf)
    inds, w = torch.cat(inds, 1).to(torch.int32), torch.cat(w, 1)
    if case["renormalize"]:
        w = w / w.sum(-1, keepdim=True)
    return [inds, w * case["scale"]]


def _block_exact(case, s):
    def normed(v, w):
        return v / ((v * v).sum(-1, keepdim=True) / case["width"] + EPS).sqrt() * (w.double() + (not case["centered"]))

    b = s["x"].double()
    if case["post"]:
        b = normed(b, s["post"])
    if case["gate"] != "none":
        b = b * (torch.sigmoid(s["gate"].double()) if case["sigmoid"] else s["gate"].double())
    h = case["residual_scale"] * s["residual"].double() + case["scale"] * b
    y = normed(h, s["weight"])
    return [*(_mx_exact(y) if case["quantize"] else [y]), h]


def _linear_exact(case, s):
    def wide(t):
        if case["format"] != "mx8":
            return t.double()
        return t[0].double() * torch.exp2(t[1].view(torch.uint8).double() - 127.0).repeat_interleave(GROUP, -1)

    y = wide(s["x"]) @ wide(s["weight"]).T
    if case["bias"]:
        y += s["bias"].double()
    name = case["activation"]
    if name == "swiglu":
        y = torch.nn.functional.silu(y[:, :case["n"]]) * y[:, case["n"]:]
    elif name != "none":
        f = torch.nn.functional
        y = {"relu": torch.relu, "silu": f.silu, "gelu": f.gelu, "gelu_tanh": functools.partial(f.gelu, approximate="tanh"),
             "sigmoid": torch.sigmoid}[name](y)
    return [y + s["residual"].double() if s["residual"] is not None else y]


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _route_exact, "block": _block_exact, "linear": _linear_exact}[case["op"]](case, s)
