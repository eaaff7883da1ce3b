"""The norm, the router, the grouped products, the combine and the adapters together, as a MoE block with unquantised or
MX experts uses them, against the block in 64 bits."""
import pytest
import torch

from op_util import mx_value
from veymoe.adapters import add_adapters
from veymoe.executor import weighted_combine
from veymoe.norm import mx_quantize, rms_norm
from veymoe.products import grouped_matmul
from veymoe.router import router_topk

pytestmark = pytest.mark.gpu

HIDDEN, INTER, EXPERTS, SLOTS, RANK = 512, 256, 24, 4, 16


def _block(x, residual, w, ids, mx):
    """One block: the normed sum, routed SwiGLU experts, their combine, and adapters beside a shared projection."""
    normed, hidden = rms_norm(x, w["norm"], residual=residual)
    rows = rms_norm(x, w["norm"], residual=residual, quantize=True)[0] if mx else normed
    inds, scores = router_topk(normed, w["router"], SLOTS)
    act = grouped_matmul(rows, w["gate_up"], inds, activation="swiglu", quantize=mx)
    down = grouped_matmul(act, w["down"], inds)
    y = weighted_combine(down, inds, scores)
    # the shared projection is a grouped product of one group
    none = torch.zeros((x.shape[0], 1), dtype=torch.int32, device=x.device)
    shared = grouped_matmul(normed, w["shared"], none).view(x.shape[0], HIDDEN)
    shared = add_adapters(shared, normed, w["a"], w["b"], ids, scales=w["scales"])
    return y + shared, hidden, inds, scores


def _exact(x, residual, w, ids, inds, scores, wide):
    """The block in 64 bits over the given routes; wide(t): a weight in 64 bits."""
    h = x.cpu().double() + residual.cpu().double()
    n = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * w["norm"].cpu().double()
    gate_up, down = wide(w["gate_up"]), wide(w["down"])
    y = torch.zeros_like(n)
    for j in range(SLOTS):
        g = torch.einsum("tk,tnk->tn", n, gate_up[inds[:, j].cpu().long()])
        a = g[:, :INTER] * torch.sigmoid(g[:, :INTER]) * g[:, INTER:]
        y += torch.einsum("tk,tnk->tn", a, down[inds[:, j].cpu().long()]) * scores[:, j:j + 1].cpu().double()
    y += n @ w["shared"][0].cpu().double().T
    for i in range(w["a"].shape[0]):
        at = ids.cpu() == i
        low = n[at] @ w["a"][i].cpu().double().T
        y[at] += w["scales"][i].cpu().double() * (low @ w["b"][i].cpu().double().T)
    return y, h


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
@pytest.mark.parametrize("tokens", [1, 7, 60, 700])
def test_block(device, tokens, mx):
    """Relative error of the whole output (2-norm).  Every rounding on the way is at most half a step of its value:
    normed, activation, down and shared rows, products with scores, their sum and the last addition in bf16 2^-8 each,
    of random sign over hundreds of terms, so their norms add up like a root of squares: under 4 * 2^-8.  MX rows and
    activations carry 2^-4 at most each, 2^-5.5 in the mean of a uniform error, twice: under 0.06."""
    gen = torch.Generator().manual_seed(tokens)
    make = lambda *shape: (torch.randn(shape, generator=gen) * shape[-1] ** -0.5).bfloat16().to(device)  # noqa: E731
    w = {"norm": (1 + 0.1 * torch.randn(HIDDEN, generator=gen)).bfloat16().to(device),
         "router": make(EXPERTS, HIDDEN), "gate_up": make(EXPERTS, 2 * INTER, HIDDEN), "down": make(EXPERTS, HIDDEN, INTER),
         "shared": make(1, HIDDEN, HIDDEN), "a": make(3, RANK, HIDDEN), "b": make(3, HIDDEN, RANK),
         "scales": torch.tensor([0.5, 1.0, 2.0], device=device)}
    if mx:
        w["gate_up"], w["down"] = mx_quantize(w["gate_up"]), mx_quantize(w["down"])
    x, r = (torch.randn((tokens, HIDDEN), generator=gen).bfloat16().to(device) for _ in range(2))
    ids = torch.randint(-1, 3, (tokens,), generator=gen, dtype=torch.int32).to(device)
    got, hidden, inds, scores = _block(x, r, w, ids, mx)
    want, h = _exact(x, r, w, ids, inds, scores, mx_value if mx else lambda t: t.cpu().double())
    off = float((got.cpu().double() - want).norm() / want.norm())
    assert off <= (0.06 if mx else 4 * 2.0 ** -8), off
    assert float((hidden.cpu().double() - h).abs().max()) <= 2.0 ** -8 * float(h.abs().max())

    # the whole block as one graph, replayed on new rows beside eager calls
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            kept = _block(x, r, w, ids, mx)
    torch.cuda.current_stream().wait_stream(side)
    for n in range(3):
        x.copy_(torch.randn(x.shape, generator=gen).bfloat16())
        graph.replay()
        eager = _block(x, r, w, ids, mx)
        torch.cuda.synchronize()
        for a, b in zip(kept, eager):
            assert torch.equal(a, b), n
