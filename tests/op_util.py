"""Helpers of the tests of the norm, the grouped products and the adapters (not collected by pytest): the definitions
in 64 bits on the CPU, and the error that fp32 arithmetic and one rounding may leave."""
import torch

F32 = 2.0 ** -24                 # half a step of fp32, relative
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
E4M3 = 2.0 ** -4
E4M3_LEAST = 2.0 ** -10          # half of e4m3's least step


def mx_exact(y):
    """(values, scales) of [.., width] in 64 bits, by the definition of an MX group."""
    g = y.double().unflatten(-1, (-1, 32))
    top = g.abs().amax(-1)
    e = torch.full_like(top, -127.0)
    live = torch.isfinite(top) & (top > 0)
    m, x = torch.frexp(torch.where(live, top, 1.0))          # top = m 2^x, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(live, torch.where(m <= 0.875, x - 9, x - 8).double(), e).clamp(min=-127)
    scale = torch.exp2(e)
    v = g / scale[..., None]
    step = torch.exp2(torch.frexp(v).exponent.double().clamp(min=-5) - 4)
    q = torch.round(v / step) * step
    bad = ~torch.isfinite(g).all(-1)
    return (torch.where(bad[..., None], float("nan"), q).flatten(-2), torch.where(bad, float("nan"), scale))


def mx_value(t):
    """What an MxTensor stands for, in 64 bits on the CPU."""
    scale = torch.exp2(t.scales.view(torch.uint8).cpu().double() - 127.0)
    scale[t.scales.view(torch.uint8).cpu() == 255] = float("nan")
    return t.values.cpu().float().double() * scale.repeat_interleave(32, -1)


def assert_within(got, want, bound, message=""):
    """|got - want| <= bound elementwise, in 64 bits; NaN where and only where want has NaN."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, (message, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), message
    fine = torch.isfinite(want)
    off = torch.where(fine, (got - want).abs() - bound, torch.zeros_like(want))
    assert not (off > 0).any(), (message, float(off.max()), float(((got - want).abs() / bound.clamp(min=1e-300))[fine].max()))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), message


def assert_mx_within(t, want, fp32_error, message=""):
    """An MxTensor against exact values known to +-fp32_error: half a step of e4m3 of the value, or of the least step
    under the group's scale; the scale is at most twice the exact one's (the error may carry the group's largest value
    over a power of two), and no smaller than it has to be."""
    got = mx_value(t)
    _, scale = mx_exact(want)
    scale = scale.repeat_interleave(32, -1)
    bound = fp32_error + torch.maximum(E4M3 * (want.double().abs() + fp32_error), 2 * E4M3_LEAST * scale)
    assert_within(got, want, bound, message)
    mine = torch.exp2(t.scales.view(torch.uint8).cpu().double() - 127.0).repeat_interleave(32, -1)
    ratio = mine / scale
    assert ((ratio == 1) | (ratio == 2) | (ratio == 0.5)).all(), message
    assert (ratio != 1).double().mean() <= 0.01, message


def norm_exact(x, weight, residual=None, eps=1e-6, one_centered=True):
    """(normed, h, error bound of normed in fp32) in 64 bits."""
    h = x.cpu().double()
    if residual is not None:
        h = h + residual.cpu().double()
    w = weight.cpu().double() + (0.0 if one_centered else 1.0)
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * w
    # h, 1 + w: half a step each; the mean of squares of n terms: at most n + 2 half steps of itself (all terms are
    # positive), half of that in the root; root, quotient and two products: four more
    n = x.shape[-1]
    return y, h, y.abs() * F32 * (2 + (n + 2) / 2 + 1 + 4)


def product_exact(x, weight, inds, swiglu):
    """(result, error bound in fp32) of rows [*inds.shape, k] and weight [e, n, k] given in 64 bits."""
    ids = inds.cpu().reshape(-1).long()
    k = weight.shape[-1]
    rows = x.reshape(-1, k)
    n = weight.shape[1]
    p, mag = torch.zeros(len(ids), n, dtype=torch.float64), torch.zeros(len(ids), n, dtype=torch.float64)
    for e in torch.unique(ids).tolist():
        if 0 <= e < weight.shape[0]:
            at = ids == e
            p[at] = rows[at] @ weight[e].T
            mag[at] = rows[at].abs() @ weight[e].abs().T
    # k products and sums, each at most one step (two half steps: the matrix units need not round to nearest)
    err = mag * (2 * F32 * (k + 1))
    if swiglu:
        h = n // 2
        g, u, eg, eu = p[:, :h], p[:, h:], err[:, :h], err[:, h:]
        silu = g * torch.sigmoid(g)
        y = silu * u
        # |silu'| <= 1.1; exp2 with its argument's rounding (|g| half steps), the sum, reciprocal and products: 8 + |g|
        err = 1.1 * eg * (u.abs() + eu) + silu.abs() * eu + y.abs() * F32 * 2 * (8 + g.abs())
        p = y
    return p.reshape(*inds.shape, -1), err.reshape(*inds.shape, -1)


def adapters_exact(base, x, a, b, ids, scales=None):
    """(result, error bound before the last rounding) in 64 bits."""
    base, x, a, b = (t.cpu().double() for t in (base, x, a, b))
    ids = ids.cpu().long()
    y, err = base.clone(), torch.zeros_like(base)
    k, rank = a.shape[2], a.shape[1]
    for i in torch.unique(ids).tolist():
        if not 0 <= i < a.shape[0]:
            continue
        at = ids == i
        s = 1.0 if scales is None else float(scales[i].double())
        v = x[at] @ a[i].T
        v_err = (x[at].abs() @ a[i].abs().T) * (2 * F32 * (k + 1))
        y[at] += s * (v @ b[i].T)
        # the rank sums' own error and 2^-16 of them (a bf16 value and its bf16 rest), then rank products and sums
        err[at] = abs(s) * ((v_err + v.abs() * 2.0 ** -16) @ b[i].abs().T
                            + (v.abs() @ b[i].abs().T) * (2 * F32 * (2 * rank + 3)))
    return y, err + y.abs() * 2 * F32
