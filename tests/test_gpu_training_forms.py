"""gated_linear and expert_linear as training programs run them: captured with their backward pass, with what is kept moved to the host, computed
again under a checkpoint, and asked twice for the same gradients.  Every form against the eager step, to the bit."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from unit_amd.experts import expert_linear, gated_linear

pytestmark = pytest.mark.gpu
KEEPS = [("gated", "pre"), ("gated", "mxfp8"), ("gated", "rows"), ("plain", None), ("plain", "mxfp8")]


def operands(dev, seed, rows=120, experts=3, n=72, k=136):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g).bfloat16().to(dev)
    cut = 10 + 7 * seed % 60
    return r(rows, k), r(experts, 2 * n, k), r(rows, 2 * n), torch.tensor([cut, 0, rows - cut - 4], device=dev)


def step(kind, keep, x, w, dy, sizes, trained):
    """the result and the gradients of the operands that train"""
    a, b = (t.detach().requires_grad_(n in trained) for n, t in (("x", x), ("w", w)))
    if kind == "gated":
        y, dy = gated_linear(a, b, sizes, "silu", keep), dy[:, :dy.shape[1] // 2]
    else:
        y = expert_linear(a, b, sizes, keep)
    return y.detach(), *torch.autograd.grad(y, [t for t in (a, b) if t.requires_grad], dy)


@pytest.mark.parametrize("trained", ["xw", "x", "w"])
@pytest.mark.parametrize("kind,keep", KEEPS)
def test_captured_step(dev, kind, keep, trained):
    """Replays on new inputs, each against an eager step, with eager steps and synchronisation between; one eager graph lives all the while."""
    args = operands(dev, 1)
    alive = gated_linear(args[0].clone().requires_grad_(), args[1].clone().requires_grad_(), args[3].clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(kind, keep, *args, trained)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(kind, keep, *args, trained)
    for seed in (1, 2, 3, 4):
        for a, b in zip(args, operands(dev, seed)):
            a.copy_(b)
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(held, step(kind, keep, *args, trained)):
                assert torch.equal(a, b)
    alive.float().sum().backward()


@pytest.mark.parametrize("trained", ["xw", "x", "w"])
@pytest.mark.parametrize("kind,keep", KEEPS)
def test_kept_on_the_host_and_computed_again(dev, kind, keep, trained):
    args = operands(dev, 5)
    want = step(kind, keep, *args, trained)
    with torch.autograd.graph.save_on_cpu():
        got = step(kind, keep, *args, trained)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    x, w, dy, sizes = args
    a, b = (t.clone().requires_grad_(n in trained) for n, t in (("x", x), ("w", w)))
    call = (lambda p, q: gated_linear(p, q, sizes, "silu", keep)) if kind == "gated" else (lambda p, q: expert_linear(p, q, sizes, keep))
    y = checkpoint(call, a, b, use_reentrant=False)
    y.backward(dy[:, :y.shape[1]])
    for g, v in zip([t.grad for t in (a, b) if t.requires_grad], want[1:]):
        assert torch.equal(g, v)


@pytest.mark.parametrize("kind,keep", KEEPS)
def test_gradients_asked_for_twice(dev, kind, keep):
    x, w, dy, sizes = operands(dev, 6)
    x.requires_grad_(), w.requires_grad_()
    y = gated_linear(x, w, sizes, "silu", keep) if kind == "gated" else expert_linear(x, w, sizes, keep)
    dy = dy[:, :y.shape[1]]
    first = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    for a, b in zip(torch.autograd.grad(y, (x, w), dy), first):
        assert torch.equal(a, b)


@pytest.mark.parametrize("keep", ["pre", "mxfp8"])
def test_frozen_weight_and_rows_written_over(dev, keep):
    """The rows are not read again, so they may be: a buffer that the next layer's result overwrites, say."""
    x, w, dy, sizes = operands(dev, 7)
    want = step("gated", keep, x, w, dy, sizes, "x")[1]
    leaf = x.clone().requires_grad_()
    rows = leaf * 1.0
    y = gated_linear(rows, w, sizes, "silu", keep)
    rows.detach().zero_()
    y.backward(dy[:, :y.shape[1]])
    assert torch.equal(leaf.grad, want)
