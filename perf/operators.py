"""Operators beside the MoE layer, as cases that can be timed and compared.

Three operators, each in its plain form (``own`` false: elementary torch operations in 32 bits, rounded once at the
end) and as calls of ``veymoe`` (``own`` true):

* ``norm``     root-mean-square norm of a row with the residual's addition in front of it (``rms_norm``); the output in
               the input's type, or in 8 bits with a power-of-two scale per group of 32 (MX: e4m3 values, e8m0 scales);
* ``experts``  products of token rows with the matrix of their expert (``grouped_matmul``): ragged groups, bf16 or MX
               operands, plain or with SwiGLU over a gate/up pair, output in bf16 or MX;
* ``lora``     low-rank adapters of many requests at once, added to the output of the projection that they share
               (``add_adapters``).

Widths: the small layer (hidden 1024, intermediate 256, 64 experts top-4), the full-size layer (2048 / 512, 512 experts
top-10) and the checkpoint's widths (2560 / 640, the same routing), and odd sizes around them.  Activations are N(0, 1),
weights N(0, 1/in), both in bf16; a skewed routing adds log Zipf(1.1) popularity to its logits, as decode batches meet it.
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
TILE = 64           # rows per block of the plain grouped product

# hidden, intermediate, experts, top_k
WIDTHS = {"small": (1024, 256, 64, 4), "full": (2048, 512, 512, 10), "wide": (2560, 640, 512, 10)}


def _norm(name, rows, width, dtype="bf16", residual=True, quantize=False, pad=0, centered=True):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual,
            "quantize": quantize, "pad": pad, "centered": centered}


def _experts(name, tokens, experts, slots, k, n, fmt="bf16", swiglu=False, quantize=False, per_slot=False, zipf=False,
             padded=0):
    return {"name": name, "op": "experts", "tokens": tokens, "experts": experts, "slots": slots, "k": k, "n": n,
            "format": fmt, "swiglu": swiglu, "quantize": quantize, "per_slot": per_slot, "zipf": zipf,
            "padded": padded}


def _lora(name, rows, k, n, rank, adapters, runs, without=0.0):
    return {"name": name, "op": "lora", "rows": rows, "k": k, "n": n, "rank": rank, "adapters": adapters,
            "runs": runs, "without": without}


def listed():
    return [
        # the norm in front of a decode step's branch, one token: latency
        _norm("norm_token", 1, 2560, quantize=True),
        # batched decode, bf16 out, gain stored around zero, rows inside a wider buffer
        _norm("norm_batch_37", 37, 2048, pad=64, centered=False),
        # a window of prefill chunks, 8 bits out for the experts' products
        _norm("norm_window_8192", 8192, 2560, quantize=True),
        # gate/up of one decode token: ten experts' weights streamed once
        _experts("experts_token", 1, 512, 10, 2048, 512, swiglu=True),
        # down of batched decode in 8 bits, skewed routing, every slot with a row of its own
        _experts("experts_batch_mx_32", 32, 512, 10, 640, 2560, "mx8", per_slot=True, zipf=True),
        # a short ragged prompt through small experts, padded at its end
        _experts("experts_prompt_333", 333, 64, 4, 1024, 256, swiglu=True, padded=13),
        # gate/up of a prefill chunk in 8 bits, the output ready for the down product
        _experts("experts_prefill_mx_2048", 2048, 512, 10, 2560, 640, "mx8", swiglu=True, quantize=True),
        # gate/up of a layer-major window of four chunks in bf16
        _experts("experts_window_8192", 8192, 512, 10, 2048, 512, swiglu=True),
        # one token of a request with an adapter
        _lora("lora_token", 1, 2560, 2560, 16, 32, False),
        # batched decode, every request with an adapter of its own or none
        _lora("lora_batch_48", 48, 2048, 1024, 32, 64, False, without=0.2),
        # prompts of several requests in one batch, odd sizes
        _lora("lora_prompts_1777", 1777, 2560, 1280, 64, 16, True, without=0.1),
        # a window of chunks
        _lora("lora_window_8192", 8192, 2560, 2560, 32, 32, True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_norm(rng):
    quantize = rng.random() < 0.5
    dtype = "fp32" if rng.random() < 0.3 else "bf16"
    if rng.random() < 0.6:
        width = rng.choice((1024, 2048, 2560, 4096, 8192))
    else:
        width = 32 * rng.randint(2, 200) if quantize else rng.randint(33, 6500)
    rows = _log(rng, 1, max(2, min(8192, 8192 * 2560 // (width * (2 if dtype == "fp32" else 1)))))
    c = _norm("", rows, width, dtype, rng.random() < 0.7, quantize, rng.choice((0, 0, 8, 40)), rng.random() < 0.6)
    return c


def _draw_experts(rng):
    hidden, inter, experts, slots = WIDTHS[rng.choice(("small", "full", "wide"))]
    fmt = rng.choice(("bf16", "mx8"))
    down = rng.random() < 0.4
    k, n = (inter, hidden) if down else (hidden, inter)
    if rng.random() < 0.3:     # odd sizes: other widths and expert counts
        unit = 32 if fmt == "mx8" else 8
        k = unit * rng.randint(64 // unit, 2560 // unit)
        n = rng.randint(33, 1100) if down else 32 * rng.randint(2, 20)
        experts = rng.randint(slots, 300)
    swiglu = not down and rng.random() < 0.8
    quantize = swiglu and fmt == "mx8" and rng.random() < 0.6
    rows = experts if rng.random() < 0.2 else 8192
    matrix = k * n * (2 if swiglu else 1)
    if fmt == "bf16":
        experts = min(experts, 512 * 2048 * 1024 // matrix)        # the weights and the products of the largest listed case
    most = 81920 * 2048 * 1024 // (slots * matrix)
    if experts * matrix > 512 * 2048 * 1024:                       # more weights than its, in 8 bits
        most //= 2
    tokens = _log(rng, 1, max(2, min(rows, most)))
    zipf = rng.random() < (0.6 if tokens <= 256 else 0.25)
    padded = rng.randint(0, max(0, tokens // 4)) if rng.random() < 0.3 else 0
    if zipf:
        tokens = min(tokens, 2048)
        padded = min(padded, tokens // 4)
    return _experts("", tokens, experts, slots, k, n, fmt, swiglu, quantize, down and rng.random() < 0.7, zipf, padded)


def _draw_lora(rng):
    k = rng.choice((1024, 2048, 2560, 2560, 8 * rng.randint(10, 320)))
    n = rng.choice((1024, 1280, 2048, 2560, rng.randint(65, 2560)))
    rank = rng.choice((8, 16, 16, 32, 32, 64, rng.randint(1, 64)))
    adapters = _log(rng, 1, 64)
    rows = _log(rng, 1, 8192)
    runs = rng.random() < (0.2 if rows <= 64 else 0.7)
    return _lora("", rows, k, n, rank, adapters, runs, rng.choice((0.0, 0.0, 0.1, 0.5)))


def draw(rng):
    c = rng.choices((_draw_norm, _draw_experts, _draw_lora), (3, 5, 4))[0](rng)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _normal(shape, gen, scale=1.0, dtype=torch.bfloat16):
    x = torch.empty(shape, device="cuda", dtype=dtype)
    return x.normal_(0.0, scale, generator=gen)


def _to_mx(v):
    """(e4m3 values, e8m0 scales) of fp32 rows whose width divides into groups: the scale is the least power of two
    that keeps the group's largest value within e4m3's range."""
    g = v.reshape(*v.shape[:-1], -1, GROUP)
    big = g.abs().amax(-1, keepdim=True)
    bits = (big.contiguous().view(torch.int32) + 0x1FFFFF) >> 23     # one exponent up where the mantissa is over 448's
    e = (bits - 8).clamp(min=0)                                      # biased by 127
    q = (g * torch.ldexp(torch.ones_like(big), 127 - e)).to(torch.float8_e4m3fn)
    return q.reshape(v.shape), e.squeeze(-1).to(torch.uint8).view(torch.float8_e8m0fnu)


def _from_mx(values, scales):
    e = scales.view(torch.uint8).to(torch.int32) - 127
    s = torch.ldexp(torch.ones(e.shape, device=e.device), e)
    g = values.float().reshape(*scales.shape, GROUP) * s[..., None]
    return g.reshape(values.shape)


def _mx_input(shape, gen, scale=1.0):
    """Random MX rows, quantised a slice at a time."""
    values = torch.empty(shape, device="cuda", dtype=torch.float8_e4m3fn)
    scales = torch.empty((*shape[:-1], shape[-1] // GROUP), device="cuda", dtype=torch.float8_e8m0fnu)
    step = max(1, (1 << 27) // max(1, math.prod(shape[1:])))
    for i in range(0, shape[0], step):
        part = values[i:i + step]
        q, s = _to_mx(_normal(part.shape, gen, scale).float())
        part.copy_(q)
        scales[i:i + step].view(torch.uint8).copy_(s.view(torch.uint8))
    return values, scales


def _routes(case, gen):
    """Distinct expert ids of every token, most probable first; padded tokens at the end have none (-1)."""
    tokens, experts = case["tokens"], case["experts"]
    logits = -torch.log(torch.empty((tokens, experts), device="cuda").exponential_(generator=gen))
    if case["zipf"]:
        popularity = -1.1 * torch.log(torch.arange(1, experts + 1, device="cuda", dtype=torch.float32))
        logits += popularity[torch.randperm(experts, device="cuda", generator=gen)]
    inds = logits.topk(case["slots"], dim=-1).indices.to(torch.int32)
    if case["padded"]:
        inds[tokens - case["padded"]:] = -1
    return inds


def _requests(case, gen):
    """Adapter of every row: one request per row, or runs of rows of one request; -1 where it has none."""
    rows = case["rows"]
    requests = max(1, min(rows, 2 * case["adapters"])) if case["runs"] else rows
    ids = torch.randint(0, case["adapters"], (requests,), device="cuda", generator=gen, dtype=torch.int32)
    ids[torch.rand(requests, device="cuda", generator=gen) < case["without"]] = -1
    if not case["runs"]:
        return ids
    ends = torch.randint(0, rows, (requests,), device="cuda", generator=gen).sort().values
    return ids[torch.searchsorted(ends, torch.arange(rows, device="cuda")).clamp(max=requests - 1)].contiguous()


def prepare(case, seed):
    gen = _gen(seed)
    s = {"op": case["op"], "case": dict(case)}
    if case["op"] == "norm":
        dtype = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
        shape = (case["rows"], case["width"] + case["pad"])
        s["x"] = _normal(shape, gen, dtype=dtype)[:, :case["width"]]
        s["residual"] = _normal(shape, gen, 2.0, dtype)[:, :case["width"]] if case["residual"] else None
        s["weight"] = (1.0 if case["centered"] else 0.0) + 0.2 * torch.randn(case["width"], device="cuda", generator=gen)
        s["weight"] = s["weight"].to(dtype)
    elif case["op"] == "experts":
        k, n = case["k"], case["n"] * (2 if case["swiglu"] else 1)
        rows = (case["tokens"], case["slots"], k) if case["per_slot"] else (case["tokens"], k)
        make = _mx_input if case["format"] == "mx8" else _normal
        s["inds"] = _routes(case, gen)
        s["x"] = make(rows, gen)
        s["weight"] = make((case["experts"], n, k), gen, k ** -0.5)
    else:
        s["ids"] = _requests(case, gen)
        s["x"] = _normal((case["rows"], case["k"]), gen)
        s["a"] = _normal((case["adapters"], case["rank"], case["k"]), gen, case["k"] ** -0.5)
        s["b"] = _normal((case["adapters"], case["n"], case["rank"]), gen, case["rank"] ** -0.5)
        s["scales"] = torch.empty(case["adapters"], device="cuda").uniform_(0.5, 2.0, generator=gen)
        s["base"] = _normal((case["rows"], case["n"]), gen)
    return s


# ------------------------------------------------------------ plain forms --

def _norm_plain(s):
    case = s["case"]
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    gain = s["weight"].float() if case["centered"] else 1.0 + s["weight"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * gain
    out = list(_to_mx(y)) if case["quantize"] else [y.to(s["x"].dtype)]
    if s["residual"] is not None:
        out.append(h.to(s["x"].dtype))
    return out


def _products_by_row(x, weight, ids):
    """x [R, K] with the matrix of each row's expert, gathered per row: few rows."""
    return torch.matmul(weight(ids.clamp(min=0)), x[:, :, None])[:, :, 0]


def _products_by_tile(x, weight, ids, experts):
    """x [R, K] sorted by expert into tiles of TILE rows, one expert to a tile, and one batch of products over them."""
    rows, width = x.shape
    key = torch.where((ids < 0) | (ids >= experts), experts, ids)
    order = torch.argsort(key, stable=True)
    key = key[order]
    starts = torch.searchsorted(key, torch.arange(experts + 2, device=x.device, dtype=key.dtype))
    last = torch.cumsum((starts[1:] - starts[:-1] + TILE - 1) // TILE, 0)      # tiles up to and with each expert
    place = torch.arange(rows, device=x.device) - starts[key]
    tile = torch.where(key > 0, last[(key - 1).clamp(min=0)], 0) + place // TILE
    count = -(-rows // TILE) + min(experts + 1, rows)
    tiles = torch.zeros((count, TILE, width), device=x.device)
    tiles[tile, place % TILE] = x[order]
    of = torch.searchsorted(last, torch.arange(count, device=x.device), right=True).clamp(max=experts - 1)
    y = torch.matmul(tiles, weight(of).transpose(1, 2))[tile, place % TILE]
    return torch.empty_like(y).index_copy_(0, order, y)


def _experts_plain(s):
    case = s["case"]
    inds, slots = s["inds"], case["slots"]
    if case["format"] == "mx8":
        x = _from_mx(*s["x"])
        weight = lambda of: _from_mx(s["weight"][0].view(torch.uint8)[of].view(torch.float8_e4m3fn),  # noqa: E731
                                     s["weight"][1].view(torch.uint8)[of].view(torch.float8_e8m0fnu))
    else:
        x = s["x"].float()
        weight = lambda of: s["weight"][of].float()  # noqa: E731
    x = x.reshape(-1, case["k"]) if case["per_slot"] else x.repeat_interleave(slots, 0)
    ids = inds.reshape(-1).long()
    y = _products_by_row(x, weight, ids) if ids.numel() <= 256 else _products_by_tile(x, weight, ids, case["experts"])
    if case["swiglu"]:
        gate, up = y[:, :case["n"]], y[:, case["n"]:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    y = torch.where((ids >= 0)[:, None], y, 0.0).reshape(*inds.shape, case["n"])
    return list(_to_mx(y)) if case["quantize"] else [y.bfloat16()]


def _lora_plain(s):
    case = s["case"]
    ids, x, a, b = s["ids"].long(), s["x"].float(), s["a"], s["b"]
    if ids.numel() <= 64:        # the adapters' matrices gathered per row
        at = ids.clamp(min=0)
        low = torch.matmul(a[at].float(), x[:, :, None])
        low = low * torch.where(ids >= 0, s["scales"][at], 0.0)[:, None, None]
        add = torch.matmul(b[at].float(), low)[:, :, 0]
    else:                        # every adapter's product, the row's own kept
        low = torch.matmul(x, a.float().reshape(-1, case["k"]).t()).reshape(-1, case["adapters"], case["rank"])
        mine = torch.arange(case["adapters"], device=ids.device) == ids[:, None]
        low = torch.where(mine[:, :, None], low * s["scales"][:, None], 0.0).reshape(ids.numel(), -1)
        add = torch.matmul(low, b.float().transpose(1, 2).reshape(-1, case["n"]))
    return [(s["base"].float() + add).bfloat16()]


# ------------------------------------------------------- the package's calls --

@functools.lru_cache(None)
def _package():
    path = os.path.join(os.getcwd(), "veystrix-core_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import veymoe.adapters
    import veymoe.norm
    import veymoe.products
    return veymoe


def _norm_own(s):
    case, v = s["case"], _package()
    got = v.norm.rms_norm(s["x"], s["weight"], eps=EPS, residual=s["residual"], one_centered=case["centered"],
                          quantize=case["quantize"])
    y, h = got if s["residual"] is not None else (got, None)
    return [*(y if case["quantize"] else [y]), *([] if h is None else [h])]


def _experts_own(s):
    case, v = s["case"], _package()
    x, weight = s["x"], s["weight"]
    if case["format"] == "mx8":
        x, weight = v.norm.MxTensor(*x), v.norm.MxTensor(*weight)
    y = v.products.grouped_matmul(x, weight, s["inds"], activation="swiglu" if case["swiglu"] else None,
                                  quantize=case["quantize"])
    return list(y) if case["quantize"] else [y]


def _lora_own(s):
    return [_package().adapters.add_adapters(s["base"], s["x"], s["a"], s["b"], s["ids"], scales=s["scales"])]


def run(state):
    if own:
        return {"norm": _norm_own, "experts": _experts_own, "lora": _lora_own}[state["op"]](state)
    return {"norm": _norm_plain, "experts": _experts_plain, "lora": _lora_plain}[state["op"]](state)


# ------------------------------------------------------------------- work --

def _experts_met(case):
    """Expected number of distinct experts that the tokens' routes name."""
    tokens, experts, slots = case["tokens"] - case["padded"], case["experts"], case["slots"]
    if not case["zipf"]:
        return experts * (1.0 - (1.0 - slots / experts) ** tokens)
    mass = [(i + 1) ** -1.1 for i in range(experts)]
    low, high = 0.0, 1e9       # a token names expert i with 1 - exp(-c mass_i), slots of them in all
    for _ in range(100):
        c = (low + high) / 2
        low, high = (c, high) if sum(1.0 - math.exp(-c * m) for m in mass) < slots else (low, c)
    return sum(1.0 - math.exp(-c * m * tokens) for m in mass)


def work(case):
    if case["op"] == "norm":
        values = case["rows"] * case["width"]
        size = 4 if case["dtype"] == "fp32" else 2
        out = 1 + 1 / GROUP if case["quantize"] else size
        return {"bytes": values * (size * (3 if case["residual"] else 1) + out) + case["width"] * size,
                "flops": 5 * values}
    if case["op"] == "experts":
        size = 1 + 1 / GROUP if case["format"] == "mx8" else 2
        routed = (case["tokens"] - case["padded"]) * case["slots"]
        n = case["n"] * (2 if case["swiglu"] else 1)
        rows = routed if case["per_slot"] else case["tokens"] - case["padded"]
        out = case["tokens"] * case["slots"] * case["n"] * (1 + 1 / GROUP if case["quantize"] else 2)
        return {"bytes": _experts_met(case) * n * case["k"] * size + rows * case["k"] * size + out
                + case["tokens"] * case["slots"] * 4, "flops": 2 * routed * n * case["k"]}
    rows, k, n, rank = case["rows"], case["k"], case["n"], case["rank"]
    share = 1.0 - case["without"]
    requests = max(1, min(rows, 2 * case["adapters"])) if case["runs"] else rows
    met = case["adapters"] * (1.0 - (1.0 - share / case["adapters"]) ** requests)
    return {"bytes": met * rank * (k + n) * 2 + rows * (share * k + 2 * n) * 2 + rows * 4,
            "flops": 2 * rows * share * rank * (k + n)}


# ------------------------------------------------------------ in 64 bits --

def _mx_exact(y):
    """y in MX by the definition: per group of 32 the least 2^e >= 2^-127 with max|y| <= 448 * 2^e; y / 2^e to the
    nearest multiple of its binade's e4m3 step (eighths, 2^-9 at the least), ties to even."""
    g = y.unflatten(-1, (-1, GROUP))
    e = torch.ceil(torch.log2(g.abs().amax(-1) / E4M3_MAX))
    top = g.abs().amax(-1)
    e = torch.where(top <= E4M3_MAX * torch.exp2(e - 1), e - 1, e)      # log2 next to a whole number
    e = torch.where(top > E4M3_MAX * torch.exp2(e), e + 1, e).clamp(min=-127)
    scale = torch.exp2(e)
    v = g / scale[..., None]
    step = torch.exp2(torch.frexp(v).exponent.double().clamp(min=-5) - 4)
    return (torch.round(v / step) * step).flatten(-2), scale


def _norm_exact(case, s):
    h = s["x"].double()
    if case["residual"]:
        h += s["residual"].double()
    w = s["weight"].double() + (0.0 if case["centered"] else 1.0)
    y = w * h / ((h * h).sum(-1, keepdim=True) / case["width"] + EPS).sqrt()
    return [*(_mx_exact(y) if case["quantize"] else [y]), *([h] if case["residual"] else [])]


def _experts_exact(case, s):
    mx = case["format"] == "mx8"

    def wide(values, scales):
        exponent = scales.view(torch.uint8).double() - 127.0
        return values.double() * torch.exp2(exponent).repeat_interleave(GROUP, -1)

    x = wide(*s["x"]) if mx else s["x"].double()
    y = torch.zeros((*s["inds"].shape, case["n"]), device="cuda", dtype=torch.float64)
    for e in torch.unique(s["inds"]).tolist():
        if e < 0:
            continue
        token, slot = torch.nonzero(s["inds"] == e, as_tuple=True)
        w = wide(s["weight"][0][e], s["weight"][1][e]) if mx else s["weight"][e].double()
        p = (x[token, slot] if case["per_slot"] else x[token]) @ w.T
        if case["swiglu"]:
            p = p[:, :case["n"]] * torch.sigmoid(p[:, :case["n"]]) * p[:, case["n"]:]
        y[token, slot] = p
    return list(_mx_exact(y)) if case["quantize"] else [y]


def _lora_exact(case, s):
    y = s["base"].double()
    for i in range(case["adapters"]):
        rows = torch.nonzero(s["ids"] == i)[:, 0]
        low = s["x"][rows].double() @ s["a"][i].double().T
        y[rows] += s["scales"][i].double() * (low @ s["b"][i].double().T)
    return [y]


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _norm_exact, "experts": _experts_exact, "lora": _lora_exact}[case["op"]](case, s)
