"""The block's norms, the router's logits, the routing, routed and shared experts together, as a block of a model uses them,
against the block in 64 bits; the same in a graph; calls on other streams, at once, and at sizes past 32 bits of offset."""
import pytest
import torch

from block_util import block_exact, select_exact
from op_util import mx_value
from veymoe.executor import weighted_combine
from veymoe.linear import linear
from veymoe.norm import MxTensor, block_norm, mx_quantize
from veymoe.products import grouped_matmul
from veymoe.routing import select_experts

pytestmark = pytest.mark.gpu

HIDDEN, INTER, EXPERTS, SLOTS, GROUPS = 512, 256, 24, 4, 6
ROUTE = dict(scoring="sigmoid", groups=GROUPS, top_groups=3, group_top=2, scale=1.5)


def _block(branch, residual, w, mx):
    """The previous block's branch joins the residual stream; this block's routed and shared experts follow."""
    rows, hidden = block_norm(branch, residual, w["pre"], post_weight=w["post"], gate=w["gate"], sigmoid_gate=True, scale=0.5)
    x = block_norm(branch, residual, w["pre"], post_weight=w["post"], gate=w["gate"], sigmoid_gate=True, scale=0.5,
                   quantize=True)[0] if mx else rows
    logits = linear(rows, w["router"], w["router_bias"], dtype=torch.float32)
    inds, weights = select_experts(logits, SLOTS, bias=w["balance"], **ROUTE)
    act = grouped_matmul(x, w["gate_up"], inds, activation="swiglu")
    routed = weighted_combine(grouped_matmul(act, w["down"], inds), inds, weights)
    shared = linear(x, w["shared_gate_up"], activation="swiglu")
    return linear(shared, w["shared_down"], residual=routed), hidden, logits, inds, weights


def _exact(branch, residual, w, inds, weights):
    """The block in 64 bits over the given routes."""
    wide = lambda t: mx_value(t) if isinstance(t, MxTensor) else t.cpu().double()  # noqa: E731
    n, h, _, _ = block_exact(branch, residual, w["pre"], post_weight=w["post"], gate=w["gate"], sigmoid_gate=True, scale=0.5)
    logits = n @ wide(w["router"]).T + wide(w["router_bias"])
    y = torch.zeros_like(n)
    gate_up, down = wide(w["gate_up"]), wide(w["down"])
    for j in range(SLOTS):
        e = inds[:, j].cpu().long()
        g = torch.matmul(gate_up[e], n[:, :, None])[:, :, 0]
        a = g[:, :INTER] * torch.sigmoid(g[:, :INTER]) * g[:, INTER:]
        y += torch.matmul(down[e], a[:, :, None])[:, :, 0] * weights[:, j:j + 1].cpu().double()
    g = n @ wide(w["shared_gate_up"]).T
    return y + (g[:, :INTER] * torch.sigmoid(g[:, :INTER]) * g[:, INTER:]) @ wide(w["shared_down"]).T, h, logits


def _weights(device, gen, mx):
    make = lambda *shape: (torch.randn(shape, generator=gen) * shape[-1] ** -0.5).bfloat16().to(device)  # noqa: E731
    w = {"pre": (1 + 0.1 * torch.randn(HIDDEN, generator=gen)).bfloat16().to(device),
         "post": (1 + 0.1 * torch.randn(HIDDEN, generator=gen)).bfloat16().to(device),
         "gate": torch.randn(HIDDEN, generator=gen).bfloat16().to(device), "router": make(EXPERTS, HIDDEN),
         "router_bias": torch.randn(EXPERTS, generator=gen).to(device),
         "balance": (0.05 * torch.randn(EXPERTS, generator=gen)).to(device),
         "gate_up": make(EXPERTS, 2 * INTER, HIDDEN), "down": make(EXPERTS, HIDDEN, INTER),
         "shared_gate_up": make(2 * INTER, HIDDEN), "shared_down": make(HIDDEN, INTER)}
    if mx:
        w["gate_up"], w["shared_gate_up"] = mx_quantize(w["gate_up"]), mx_quantize(w["shared_gate_up"])
    return w


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("tokens", [1, 7, 60, 700])
def test_block(device, tokens, mx):
    """Relative error of the whole output (2-norm).  Roundings on the way are at most half a step of their values, of random
    sign over hundreds of terms, so their norms add up like a root of squares: the normed rows, routed activations, down
    rows, combine, shared activations and the output in bf16 2^-8 each: under 4 * 2^-8.  MX rows carry 2^-4 at most, 2^-5.5
    in the mean of a uniform error, over both gate/up products: under 0.06.  Logits: k products of bf16 rows."""
    gen = torch.Generator().manual_seed(tokens)
    w = _weights(device, gen, mx)
    x = torch.randn((tokens, HIDDEN), generator=gen).bfloat16().to(device)
    r = (2 * torch.randn((tokens, HIDDEN), generator=gen)).to(device)
    got, hidden, logits, inds, weights = _block(x, r, w, mx)
    want, h, exact_logits = _exact(x, r, w, inds, weights)
    off = float((got.cpu().double() - want).norm() / want.norm())
    assert off <= (0.06 if mx else 4 * 2.0 ** -8), off
    assert float((hidden.cpu().double() - h).abs().max()) <= 2.0 ** -20 * float(h.abs().max())
    # the normed rows' bf16 rounding under a product of 512 terms of N(0, 1/512)
    assert float((logits.cpu().double() - exact_logits).norm() / exact_logits.norm()) <= 2.0 ** -8
    i, s = select_exact(logits, SLOTS, bias=w["balance"], **ROUTE)
    assert torch.equal(inds.cpu(), i) and float((weights.cpu().double() - s).abs().max()) <= 2.0 ** -22

    # the block as one graph, replayed on new rows beside eager calls
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            kept = _block(x, r, w, mx)
    torch.cuda.current_stream().wait_stream(side)
    for n in range(3):
        x.copy_(torch.randn(x.shape, generator=gen).bfloat16())
        graph.replay()
        eager = _block(x, r, w, mx)
        torch.cuda.synchronize()
        for a, b in zip(kept, eager):
            assert torch.equal(a, b), n


def _calls(device, seed):
    """Calls of every form, each with its result on the default stream."""
    gen = torch.Generator().manual_seed(seed)
    make = lambda *shape: (torch.randn(shape, generator=gen) * shape[-1] ** -0.5).bfloat16().to(device)  # noqa: E731
    out = []
    for rows, k, n, act in ((2, 512, 300, None), (20, 512, 300, "gelu"), (300, 1000, 640, "silu"), (2300, 512, 700, "swiglu"),
                            (4096, 640, 1280, "relu"), (2048, 512, 2560, None)):
        x, m = make(rows, k), make(n * (2 if act == "swiglu" else 1), k)
        out.append(lambda x=x, m=m, act=act: linear(x, m, activation=act))
        if k % 32 == 0:
            qx, qm = mx_quantize(x), mx_quantize(m)
            out.append(lambda x=qx, m=qm, act=act: linear(x, m, activation=act))
    for rows, width in ((3, 2560), (1500, 1024), (1200, 5000)):
        x, r, w = make(rows, width), make(rows, width), make(width)
        out.append(lambda x=x, r=r, w=w: block_norm(x, r, w, post_weight=w, gate=w, sigmoid_gate=True))
    for rows, experts in ((5, 512), (3000, 160)):
        logits, bias = torch.randn((rows, experts), generator=gen).to(device), torch.randn(experts, generator=gen).to(device)
        out.append(lambda x=logits, b=bias: select_experts(x, 6, scoring="sigmoid", bias=b, groups=8, top_groups=4, group_top=2))
    return out


def _same(a, b):
    if isinstance(a, torch.Tensor):
        return torch.equal(a, b)
    return all(_same(x, y) for x, y in zip(a, b))


def test_calls_on_two_streams_at_once(device):
    calls = [_calls(device, seed) for seed in (1, 2)]
    want = [[c() for c in side] for side in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[], []]
    for n in range(len(calls[0])):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(calls[i][n]())
    torch.cuda.synchronize()
    for i in range(2):
        for n, (a, b) in enumerate(zip(got[i], want[i])):
            assert _same(a, b), (i, n)


def test_every_form_in_a_graph(device):
    calls = _calls(device, 3)
    want = [c() for c in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            kept = [c() for c in calls]
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        graph.replay()
        again = [c() for c in calls]
        torch.cuda.synchronize()
        for n in range(len(calls)):
            assert _same(kept[n], want[n]) and _same(again[n], want[n]), n


def test_offsets_past_32_bits(device):
    """Rows whose first and last lie more than 4 GiB apart, in operands and outputs."""
    gen = torch.Generator().manual_seed(4)
    stride = (1 << 25) + 64                      # 80 rows: 5.4 GB of bf16
    big = torch.empty((80, stride), dtype=torch.bfloat16, device=device)
    x = torch.randn((80, 256), generator=gen).bfloat16().to(device)
    w = torch.randn((96, 256), generator=gen).bfloat16().to(device)
    far = big[:, :256]
    far.copy_(x)
    assert torch.equal(linear(far, w), linear(x, w))
    assert torch.equal(linear(far[:3], w), linear(x[:3], w))
    assert torch.equal(linear(w[:, :256], far), linear(w, x))
    out = big[:, 512:608]
    linear(x, w, out=out)
    assert torch.equal(out, linear(x, w))
    r = torch.randn((80, 256), generator=gen).bfloat16().to(device)
    want = block_norm(x, r, w[0])
    got = block_norm(far, r, w[0], residual_out=big[:, 1024:1280], out=big[:, 2048:2304])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for a, b in zip(select_experts(far, 5), select_experts(x, 5)):
        assert torch.equal(a, b)
    del big, far, out
    torch.cuda.empty_cache()


def test_large_tiles_of_ragged_sizes(device):
    """Calls that fill the chip with large tiles, at edges of rows, outputs and inputs, against products of 32 bits, whose
    own error is as large: k products and sums of a step each on either side."""
    gen = torch.Generator(device=device).manual_seed(5)
    for rows, k, n, act in ((8192, 40, 2570, None), (7937, 1000, 2559, "silu"), (8191, 72, 1285, "swiglu"), (6001, 2080, 2051, None)):
        make = lambda *shape: torch.randn(shape, generator=gen, device=device).bfloat16()  # noqa: E731
        m = n * (2 if act == "swiglu" else 1)
        x, w, b, r = make(rows, k), make(m, k) * k ** -0.5, make(m), make(rows, n)
        got = linear(x, w, b, activation=act, residual=r, dtype=torch.float32)
        v = x.float() @ w.float().t()
        size = x.float().abs() @ w.float().abs().t()
        err = size * 2 * 2.0 ** -23 * (k + 2) + 1e-6
        v += b.float()
        if act == "swiglu":
            want = torch.nn.functional.silu(v[:, :n]) * v[:, n:] + r.float()
            err = 1.2 * err[:, :n] * (v[:, n:].abs() + 1) + (v[:, :n].abs() + 1) * err[:, n:]
        else:
            want = (torch.nn.functional.silu(v) if act else v) + r.float()
            err = 1.2 * err
        off = (got - want).abs() - err - (want.abs() + v.abs().amax()) * 2.0 ** -19
        assert not (off > 0).any(), (rows, k, n, float(off.max()))
