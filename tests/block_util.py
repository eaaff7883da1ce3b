"""Helpers of the tests of the routing, the block's norms and the dense products (not collected by pytest): the definitions
in 64 bits on the CPU, and the error that fp32 arithmetic may leave before the last rounding."""
import math

import torch

from op_util import F32, mx_value

INF = math.inf


def select_exact(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=1, group_top=1, renormalize=True, scale=1.0):
    """(inds, weights) row by row from the definition; weights in 64 bits."""
    lead, experts = logits.shape[:-1], logits.shape[-1]
    rows = logits.detach().cpu().double().reshape(-1, experts).tolist()
    b = None if bias is None else bias.detach().cpu().double().tolist()
    per = experts // groups
    before = lambda c, i: (0 if math.isnan(c) else 1, 0.0 if math.isnan(c) else -c, i)  # noqa: E731
    all_inds, all_weights = [], []
    for l in rows:
        live = [i for i in range(experts) if l[i] != -INF]
        if scoring == "softmax":
            top = max((l[i] for i in live if not math.isnan(l[i])), default=0.0)
            e = [math.exp(v - top) if math.isfinite(v - top) else (0.0 if v - top == -INF else math.nan) for v in l]
            total = math.fsum(e[i] for i in live) if all(math.isfinite(e[i]) for i in live) else math.nan
            score = [e[i] / total if i in set(live) else 0.0 for i in range(experts)]
        else:
            score = [math.nan if math.isnan(v) else 1.0 / (1.0 + math.exp(-v)) if v > -700.0 else 0.0 for v in l]
        choice = {i: (l[i] if b is None else score[i] + b[i]) for i in live}
        choice = {i: c for i, c in choice.items() if c != -INF}
        if groups > 1:
            ranks = []
            for g in range(groups):
                mine = [score[i] if b is None and group_top == 2 else c for i, c in choice.items() if i // per == g]
                best = sorted(mine, key=lambda c: before(c, 0))[:group_top]
                ranks.append(sum(best) if best else -INF)
            kept = sorted(range(groups), key=lambda g: before(ranks[g], g))[:top_groups]
            choice = {i: c for i, c in choice.items() if i // per in kept}
        inds = sorted(choice, key=lambda i: before(choice[i], i))[:top_k]
        w = [score[i] for i in inds]
        if renormalize:
            total = sum(w)
            w = [0.0 if total == 0.0 else v / total for v in w]
        none = top_k - len(inds)
        all_inds.append(inds + [-1] * none)
        all_weights.append([v * scale for v in w] + [0.0] * none)
    return (torch.tensor(all_inds, dtype=torch.int32).reshape(*lead, top_k),
            torch.tensor(all_weights, dtype=torch.float64).reshape(*lead, top_k))


def block_exact(x, residual, weight=None, post_weight=None, gate=None, sigmoid_gate=False, scale=1.0, residual_scale=1.0,
                eps=1e-6, one_centered=True):
    """(y, h, bound of y's fp32 error, of h's) in 64 bits."""
    x, r = x.detach().cpu().double(), residual.detach().cpu().double()
    at = 0.0 if one_centered else 1.0
    b = x
    steps = 0
    if post_weight is not None:   # factor, its two products, the gain's sum: half a step each
        b = b / torch.sqrt(b.square().mean(-1, keepdim=True) + eps) * (post_weight.detach().cpu().double() + at)
        steps += 4
    if gate is not None:          # its product; exp (2), a sum and a quotient of up to two each where it is a sigmoid
        g = gate.detach().cpu().double()
        b = b * (torch.sigmoid(g) if sigmoid_gate else g)
        steps += 7 if sigmoid_gate else 1
    part = scale * b
    h = residual_scale * r + part
    # the scales' own roundings, their products, the sum
    h_err = F32 * (part.abs() * (steps + 3) + (residual_scale * r).abs() * 2 + h.abs())
    if weight is None:
        return None, h, None, h_err
    w = weight.detach().cpu().double() + at
    factor = 1.0 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    y = h * factor * w
    # h's errors move the factor by at most their norm over h's
    off = h_err.square().sum(-1, keepdim=True).sqrt() / h.square().sum(-1, keepdim=True).sqrt().clamp(min=1e-300)
    return y, h, y.abs() * (F32 * 4 + off) + h_err * (factor * w).abs(), h_err


def _activation(v, name):
    """(value, |derivative| bound, relative error in half steps of fp32) of an activation."""
    if name == "relu":
        return v.clamp(min=0.0), 1.0, torch.zeros_like(v)
    if name == "silu":
        return v * torch.sigmoid(v), 1.1, 16 + 2 * v.abs()
    if name == "gelu":            # erfc to 4 steps, its argument's rounding times 2 z^2 = v^2, two products
        return 0.5 * v * torch.erfc(v * -math.sqrt(0.5)), 1.13, 12 + 4 * v.square()
    if name == "gelu_tanh":       # the argument's five half steps and the sigmoid's own
        s = math.sqrt(8.0 / math.pi) * (v + 0.044715 * v ** 3)
        return v * torch.sigmoid(s), 1.13, 20 + 7 * s.abs()
    if name == "sigmoid":
        return torch.sigmoid(v), 0.25, 16 + 2 * v.abs()
    return v, 1.0, torch.zeros_like(v)


def linear_exact(x, weight, bias=None, activation=None, residual=None):
    """(value, bound of the fp32 error) in 64 bits; x and weight tensors or MxTensors."""
    wide = lambda t: mx_value(t) if isinstance(t, tuple) else t.detach().cpu().double()  # noqa: E731
    x, w = wide(x), wide(weight)
    k = x.shape[-1]
    v = x @ w.T
    err = (x.abs() @ w.abs().T) * (2 * F32 * (k + 1))   # products and sums, at most a step each
    if bias is not None:
        b = bias.detach().cpu().double()
        v = v + b
        err = err + v.abs() * F32
    if activation == "swiglu":
        n = v.shape[-1] // 2
        g, u, eg, eu = v[..., :n], v[..., n:], err[..., :n], err[..., n:]
        silu = g * torch.sigmoid(g)
        y = silu * u
        err = 1.1 * eg * (u.abs() + eu) + silu.abs() * eu + y.abs() * F32 * 2 * (8 + g.abs())
    else:
        y, slope, steps = _activation(v, activation)
        err = slope * err + y.abs() * F32 * steps + 2.0 ** -120
    if residual is not None:
        y = y + residual.detach().cpu().double()
        err = err + y.abs() * F32
    return y, err
