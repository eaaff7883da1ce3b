"""Calls behind a sort, whose scratch is the caller's: in graphs, on another stream, and on two streams at once.

The sizes are asserted to take a workspace, so a change of the dispatch rules cannot take these tests off the sort."""
import pytest
import torch

from test_gpu_ops_run import EXPERTS, HIDDEN, INTER, RANK, SLOTS, _block
from veymoe import _lib
from veymoe.adapters import add_adapters
from veymoe.norm import mx_quantize
from veymoe.products import grouped_matmul

pytestmark = pytest.mark.gpu

# tokens, slots, experts: sorts of one launch, of one launch over several blocks, and of two launches
PRODUCTS = [(60, 4, 200), (1500, 4, 200), (1200, 4, 20), (4300, 4, 20)]
# rows, adapters
ADAPTERS = [(2100, 9), (9000, 40), (16500, 300)]


def _product(gen, tokens, slots, experts, mx, device):
    """call(ids), the ids and a maker of new ids of a product that sorts."""
    assert _lib.lib().vm_grouped_matmul_workspace(tokens * slots, experts) > 0
    x = torch.randn((tokens, 96), generator=gen).bfloat16().to(device)
    w = (torch.randn((experts, 128, 96), generator=gen) * 96 ** -0.5).bfloat16().to(device)
    if mx:
        x, w = mx_quantize(x), mx_quantize(w)

    def call(ids):
        y = grouped_matmul(x, w, ids, activation="swiglu", quantize=mx)
        return [y.values.view(torch.uint8), y.scales.view(torch.uint8)] if mx else [y]

    return call, lambda: torch.randint(-1, experts, (tokens, slots), generator=gen, dtype=torch.int32)


def _adapter(gen, rows, adapters, device):
    assert _lib.lib().vm_add_adapters_workspace(rows, 8, adapters) > 0
    base, x = (torch.randn((rows, w), generator=gen).bfloat16().to(device) for w in (72, 64))
    a = torch.randn((adapters, 8, 64), generator=gen).bfloat16().to(device)
    b = torch.randn((adapters, 72, 8), generator=gen).bfloat16().to(device)
    return (lambda ids: [add_adapters(base, x, a, b, ids)],
            lambda: torch.randint(-1, adapters, (rows,), generator=gen, dtype=torch.int32))


def _calls(device):
    for size in PRODUCTS:
        for mx in (False, True):
            yield f"products {size} {mx}", _product(torch.Generator().manual_seed(sum(size)), *size, mx, device)
    for size in ADAPTERS:
        yield f"adapters {size}", _adapter(torch.Generator().manual_seed(sum(size)), *size, device)


def _same(a, b, message):
    assert len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b)), message


def test_sorted_calls_in_graphs(device):
    """Two captured calls on a side stream, replayed in turn over new ids, with eager calls and other allocations between:
    every replay equals the eager call."""
    for name, (call, new_ids) in _calls(device):
        ids = [new_ids().to(device) for _ in range(2)]
        call(ids[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        graphs, kept = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
        with torch.cuda.stream(side):
            for g, i in zip(graphs, ids):
                with torch.cuda.graph(g, stream=side):
                    kept.append(call(i))
        torch.cuda.current_stream().wait_stream(side)
        for n in range(4):
            for i in ids:
                i.copy_(new_ids())
            graphs[n % 2].replay()
            graphs[1 - n % 2].replay()
            other = torch.full((1 << 22,), n, dtype=torch.uint8, device=device)   # over freed scratch, if any was
            for k, i in zip(kept, ids):
                eager = call(i)
                torch.cuda.synchronize()
                _same(k, eager, (name, n))
            del other


def test_sorted_calls_on_two_streams_at_once(device):
    """Calls on two streams, each over its own ids, beside one another and beside a third on the current stream."""
    for name, (call, new_ids) in _calls(device):
        ids = [new_ids().to(device) for _ in range(3)]
        want = [call(i) for i in ids]
        streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.current_stream()]
        torch.cuda.synchronize()
        got = [[], [], []]
        for _ in range(6):
            for j, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[j].append(call(ids[j]))
        torch.cuda.synchronize()
        for j, runs in enumerate(got):
            for y in runs:
                _same(y, want[j], (name, j))


def test_sorted_calls_repeat_themselves(device):
    """The order of a group's rows differs from sort to sort and changes no bit."""
    for name, (call, new_ids) in _calls(device):
        ids = new_ids().to(device)
        first = call(ids)
        for n in range(8):
            _same(call(ids), first, (name, n))


@pytest.mark.parametrize("mx", [False, True], ids=["bf16", "mx"])
def test_block_of_sorted_calls(device, mx):
    """The operators together at a size whose products and adapters sort: in a graph, and against the same tokens in calls
    that do not sort, where the routes agree (each is within 4 * 2^-8 of the exact block, 0.06 in MX, relative in the 2-norm)."""
    tokens = 2100
    lib = _lib.lib()
    assert lib.vm_grouped_matmul_workspace(tokens * SLOTS, EXPERTS) > 0
    assert lib.vm_add_adapters_workspace(tokens, RANK, 3) > 0
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
    got = _block(x, r, w, ids, mx)
    parts = [_block(x[i:i + 60], r[i:i + 60], w, ids[i:i + 60], mx) for i in range(0, tokens, 60)]
    same = (got[2] == torch.cat([p[2] for p in parts])).all(-1)      # the norm's forms may differ by a bit, and a near tie
    assert same.float().mean() > 0.9
    got, part = got[0].double()[same], torch.cat([p[0] for p in parts]).double()[same]
    off = float((got - part).norm() / part.norm())
    assert off <= 2 * (0.06 if mx else 4 * 2.0 ** -8), off

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            kept = _block(x, r, w, ids, mx)
    torch.cuda.current_stream().wait_stream(side)
    for n in range(3):
        x.copy_(torch.randn(x.shape, generator=gen).bfloat16())
        ids.copy_(torch.randint(-1, 3, (tokens,), generator=gen, dtype=torch.int32))
        graph.replay()
        eager = _block(x, r, w, ids, mx)
        torch.cuda.synchronize()
        for a, b in zip(kept, eager):
            assert torch.equal(a, b), n
