"""The layer of gated experts, and the gated operators as a program runs them together: autograd, graphs, streams, long tensors.

Tolerances of the layer, as relative 2-norms.  16-bit values are rounded where the layer rounds them (h, the down product, the shares' sum;
backwards the gate's gradients and the two products'), each by at most 2^-8 (bfloat16) or 2^-11 (float16) of its value: 8 roundings of
the result's norm.  A checkpoint in 8 bits is off by at most 2^-4 of its value; one of the rows, one of each pre-activation and one of h
reach a gradient, none with a factor above 1.13 (the largest slope of an activation, over the norm): 4 * 2^-4."""
import threading

import pytest
import torch

import unit_amd as U
from unit_amd.experts import ExpertLayer, expert_linear, gated_linear

pytestmark = pytest.mark.gpu
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(tokens, experts, model, hidden, dtype, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    x, logits = r(tokens, model).to(dtype).to(dev), r(tokens, experts).to(dev)
    return x, logits, (r(experts, 2 * hidden, model) / model ** 0.5).to(dtype).to(dev), (r(experts, model, hidden) / hidden ** 0.5).to(dtype).to(dev)


def act(z, gate):
    return torch.nn.functional.silu(z) if gate == "silu" else torch.nn.functional.gelu(z, approximate="tanh")


def plain(x, logits, up, down, top_k, gate):
    best, expert = logits.to(x.dtype).topk(top_k, -1)
    share = torch.softmax(best, -1)
    y = torch.zeros_like(x)
    for j in range(top_k):
        for e in range(up.shape[0]):
            m = expert[:, j] == e
            g, u = (x[m] @ up[e].T).chunk(2, -1)
            y = y.index_put((m.nonzero().flatten(),), share[m, j, None] * ((act(g, gate) * u) @ down[e].T), accumulate=True)
    return y


def far(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gate", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("tokens,experts,top_k,model,hidden", [(1, 8, 2, 64, 128), (7, 5, 1, 72, 40), (130, 9, 3, 256, 136), (600, 4, 2, 128, 512)])
def test_layer(dev, dtype, gate, tokens, experts, top_k, model, hidden):
    x, logits, up, down = make(tokens, experts, model, hidden, dtype, dev)
    got = ExpertLayer(up, down, top_k, gate)(x, logits)
    assert got.dtype == dtype and got.shape == x.shape
    assert far(got, plain(x.double(), logits.double(), up.double(), down.double(), top_k, gate)) <= 8 * ROUND[dtype]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gate", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("keep", ["pre", "rows", "mxfp8"])
def test_training_step(dev, dtype, gate, keep):
    x, logits, up, down = make(150, 6, 128, 192, dtype, dev)
    seed = torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).to(dev)
    ours = [t.clone().requires_grad_() for t in (x, up, down)]
    y = ExpertLayer(ours[1], ours[2], 2, gate, keep)(ours[0], logits)
    (y.float() * seed).sum().backward()
    exact = [t.double().requires_grad_() for t in (x, up, down)]
    want = plain(exact[0], logits.double(), exact[1], exact[2], 2, gate)
    (want * seed.double()).sum().backward()
    assert far(y.detach(), want.detach()) <= 8 * ROUND[dtype]  # the forward pass loses nothing to what is kept
    for a, b in zip(ours, exact):
        assert a.grad.dtype == dtype and a.grad.shape == b.grad.shape
        assert far(a.grad, b.grad) <= 8 * ROUND[dtype] + (4 * 2.0 ** -4 if keep == "mxfp8" else 0)


def test_what_is_kept(dev):
    """Bytes held between forward and backward, beside the result: rows and pre-activations of 16 bits, of 8 bits, or the rows alone."""
    rows, k, n = 4096, 512, 1024
    g = torch.Generator(device=dev).manual_seed(4)
    x0, w = (torch.randn(s, device=dev, generator=g).bfloat16().requires_grad_() for s in ((rows, k), (2 * n, k)))
    held = {}
    for keep in ("pre", "mxfp8", "rows"):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        h = gated_linear(x0 * 1.0, w, keep=keep)  # its rows are an activation that nothing else holds
        held[keep] = torch.cuda.memory_allocated() - before - h.numel() * 2
        h.float().sum().backward()
        x0.grad = w.grad = None
        del h
    assert held == {"pre": rows * (2 * k + 4 * n), "mxfp8": rows * (k + 2 * n) * 33 // 32, "rows": rows * 2 * k}


def test_quantized_layer(dev):
    """Against the same layer on the values that weights and rows stand for; h is rounded to x's type, then quantised again."""
    x, logits, up, down = make(90, 6, 160, 224, torch.bfloat16, dev)
    layer = ExpertLayer(up, down, 2, "silu").quantized()
    assert layer.gate == "silu"
    values = lambda t: U.dequantize_mxfp4(U.quantize_mxfp4(t)).double()
    best, expert = logits.topk(2, -1)
    share = torch.softmax(best, -1).double()
    wu, wd = U.dequantize_mxfp4(layer.up).double(), U.dequantize_mxfp4(layer.down).double()
    want = torch.zeros((90, 160), dtype=torch.float64, device=dev)
    for j in range(2):
        for e in range(6):
            m = expert[:, j] == e
            g, u = (values(x[m]) @ wu[e].T).chunk(2, -1) if bool(m.any()) else (None, None)
            if g is not None:
                want[m] += share[m, j, None] * (values((act(g, "silu") * u).bfloat16()) @ wd[e].T).bfloat16().double()
    # h may be rounded to the other of two neighbours than in 64 bits, and a quantised value moves by a step then: one of several hundred
    assert far(layer(x, logits), want) <= 8 * ROUND[torch.bfloat16]


def test_no_tokens(dev):
    for keep in ("pre", "rows", "mxfp8"):
        x, logits, up, down = (t.requires_grad_() for t in make(0, 5, 64, 40, torch.bfloat16, dev))
        y = ExpertLayer(up, down, 2, "silu", keep)(x, logits)
        assert y.shape == (0, 64)
        y.float().sum().backward()
        assert x.grad.shape == (0, 64) and not bool(up.grad.any()) and not bool(down.grad.any())
        with torch.no_grad():
            assert ExpertLayer(up, down, 2, "silu").quantized()(x, logits).shape == (0, 64)


@pytest.mark.parametrize("keep", ["pre", "rows", "mxfp8"])
def test_frozen_operands_and_gradients_that_begin_anywhere(dev, keep):
    x, _, up, _ = make(40, 3, 64, 48, torch.float16, dev)
    sizes = torch.tensor([10, 0, 25], device=dev)
    seed = torch.randn((40, 48), generator=torch.Generator().manual_seed(5)).half().to(dev)

    def run(*trained):
        a, b = (t.clone().requires_grad_(t is x and "x" in trained or t is up and "w" in trained) for t in (x, up))
        h = gated_linear(a, b, sizes, "gelu_tanh", keep)
        torch.cat((torch.zeros(1, device=dev, dtype=h.dtype), h.flatten())).backward(torch.cat((seed.new_zeros(1), seed.flatten())))
        return a.grad, b.grad

    dx, dw = run("x", "w")
    alone_x, none = run("x")
    assert none is None
    none, alone_w = run("w")
    assert none is None
    for a, b in ((dx, alone_x), (dw, alone_w)):  # the same sums in another order of tiles
        assert far(a, b) <= 2 * ROUND[torch.float16]


def test_second_derivatives_are_refused(dev):
    x, _, up, _ = (t.requires_grad_() for t in make(40, 3, 64, 48, torch.float16, dev))
    sizes = torch.tensor([10, 0, 25], device=dev)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(gated_linear(x, up, sizes).float().square().sum(), x, create_graph=True)


def test_gated_linear_is_the_operator(dev):
    x, _, up, _ = make(40, 3, 64, 48, torch.float16, dev)
    sizes = torch.tensor([10, 0, 25], device=dev)
    want = U.gated_dense(x, up, sizes, "gelu_tanh", "float16")
    assert torch.equal(gated_linear(x, up, sizes, "gelu_tanh"), want)
    for keep in ("pre", "rows", "mxfp8"):
        assert torch.equal(gated_linear(x.clone().requires_grad_(), up, sizes, "gelu_tanh", keep).detach(), want)


def test_rows_in_8_bits_for_a_plain_product(dev):
    """The weight's gradient is that of the rows that the checkpoint stands for, the rows' gradient is untouched."""
    x, _, up, _ = make(60, 3, 96, 40, torch.bfloat16, dev)
    sizes = torch.tensor([20, 0, 35], dtype=torch.int32, device=dev)
    seed = torch.randn((60, 80), generator=torch.Generator().manual_seed(6)).bfloat16().to(dev)
    got = [t.clone().requires_grad_() for t in (x, up)]
    expert_linear(*got, sizes, keep="mxfp8").backward(seed)
    x8 = U.dequantize_mxfp8(U.quantize_mxfp8(x), "bfloat16")
    dx, dw = U.grouped_dense_grad(x8, up, seed, sizes, "bfloat16", "bfloat16")
    assert torch.equal(got[0].grad, dx) and torch.equal(got[1].grad, dw)
    for a, b in zip(U.grouped_dense_grad(U.quantize_mxfp8(x), up, seed, sizes, "bfloat16", "bfloat16"), (dx, dw)):
        assert torch.equal(a, b)
    with pytest.raises(ValueError, match="keep"):
        expert_linear(x, up, sizes, keep="pre")


def everything(x, w, wq, dy, sizes):
    h, pre = U.gated_dense(x, w, sizes, "silu", "bfloat16", keep="pre")
    h8, pre8 = U.gated_dense(x, w, sizes, "gelu_tanh", "float32", keep="mxfp8")
    x8 = U.quantize_mxfp8(x)
    out = [h, pre, h8, U.dequantize_mxfp8(pre8), U.dequantize_mxfp8(x8, "bfloat16"), U.gated_dense_mxfp4(x, wq, sizes)]
    for data, kept in ((x, pre), (x8, pre8), (x8, None)):
        out += U.gated_dense_grad(data, w, dy, sizes, "silu", kept, "bfloat16", "float32")
    return out


def case(rows, sizes, n, k, dev, seed=7):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    lead = () if sizes is None else (len(sizes),)
    x, w, dy = r(rows, k).bfloat16().to(dev), (r(*lead, 2 * n, k) / k ** 0.5).bfloat16().to(dev), r(rows, n).bfloat16().to(dev)
    return x, w, U.quantize_mxfp4(w), dy, None if sizes is None else torch.tensor(sizes, device=dev)


@pytest.mark.parametrize("rows,sizes,n,k", [(5, None, 72, 136), (300, [100, 0, 190], 136, 72), (4000, None, 64, 64)])
def test_streams_and_replays(dev, rows, sizes, n, k):
    """On another stream than the operands', and captured: every replay on new inputs against the eager results, with eager work between."""
    args = case(rows, sizes, n, k, dev)
    want = everything(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = everything(*args)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = everything(*args)
    for seed in (7, 8, 9, 10):
        new = case(rows, sizes, n, k, dev, seed)
        for a, b in zip(args, new):
            (a.buf if isinstance(a, U.Mxfp4Tensor) else a).copy_(b.buf if isinstance(b, U.Mxfp4Tensor) else b) if a is not None else None
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(held, everything(*args)):
                assert torch.equal(a, b)


def test_two_graphs_do_not_share_workspaces(dev):
    """Gradients captured twice, replayed on two streams at a time."""
    one, two = case(600, None, 136, 72, dev, 1), case(600, None, 136, 72, dev, 2)
    run = lambda a: U.gated_dense_grad(U.quantize_mxfp8(a[0]), a[1], a[3], None, "silu", None, "bfloat16", "float32")
    want = run(one), run(two)
    graphs, held = [], []
    for a in (one, two):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(run(a))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for h, w in zip(held, want):
            assert all(torch.equal(a, b) for a, b in zip(h, w))


def test_calls_from_two_threads(dev):
    args = [case(200, [50, 0, 140], 72, 136, dev, s) for s in (1, 2)]
    want = [everything(*a) for a in args]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    got = everything(*args[i])
                    s.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append(i)
                s.synchronize()
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_operands_that_are_not_contiguous(dev):
    x, w, _, dy, s = case(90, [40, 0, 45], 72, 136, dev)
    _, pre = U.gated_dense(x, w, s, keep="pre")
    want = U.gated_dense(x, w, s), *U.gated_dense_grad(x, w, dy, s, pre=pre)
    wide = lambda t: torch.cat((t, t), -1)[..., :t.shape[-1]]
    got = U.gated_dense(wide(x), w.transpose(1, 2).contiguous().transpose(1, 2), torch.stack((s, s), 1)[:, 0]), *U.gated_dense_grad(
        x.t().contiguous().t(), wide(w), wide(dy), s, pre=wide(pre))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_sizes_that_promise_more_rows_than_there_are(dev):
    x, w, wq, dy, _ = case(50, [1, 1, 1], 40, 72, dev)
    for given, counted in (([20, -5, 1000], [20, 0, 30]), ([60, 60, 60], [50, 0, 0]), ([0, 0, 0], [0, 0, 0]), ([1 << 40, 3, 4], [50, 0, 0])):
        a = everything(x, w, wq, dy, torch.tensor(given, dtype=torch.int64, device=dev))
        b = everything(x, w, wq, dy, torch.tensor(counted, dtype=torch.int32, device=dev))
        for t, u in zip(a, b):
            assert torch.equal(t, u)


def test_rows_beyond_2_31_bytes(dev):
    """Rows, results, pre-activations and gate gradients whose offsets pass 32 bits: the last rows against a call of their own."""
    rows, n, k = 540_000, 2056, 2056
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device=dev)
    g = torch.Generator(device=dev).manual_seed(8)
    tail = 700
    x[-tail:] = torch.randn((tail, k), generator=g, device=dev).bfloat16()
    w = (torch.randn((2 * n, k), generator=g, device=dev) / k ** 0.5).bfloat16()
    dy = torch.zeros((rows, n), dtype=torch.bfloat16, device=dev)
    dy[-tail:] = torch.randn((tail, n), generator=g, device=dev).bfloat16()
    for keep in ("pre", "mxfp8"):
        h, pre = U.gated_dense(x, w, None, "silu", "bfloat16", keep=keep)
        few, few_pre = U.gated_dense(x[-tail:].contiguous(), w, None, "silu", "bfloat16", keep=keep)
        assert far(h[-tail:], few) <= 2 * ROUND[torch.bfloat16] and not bool(h[:-tail].any())
        dx, dw = U.gated_dense_grad(x, w, dy, None, "silu", pre, "bfloat16", "float32")
        few_dx, few_dw = U.gated_dense_grad(x[-tail:].contiguous(), w, dy[-tail:].contiguous(), None, "silu", few_pre, "bfloat16", "float32")
        assert far(dx[-tail:], few_dx) <= 4 * ROUND[torch.bfloat16] and far(dw, few_dw) <= 4 * ROUND[torch.bfloat16] and not bool(dx[:-tail].any())
        del h, pre, dx, dw
    x8 = U.quantize_mxfp8(x)
    assert torch.equal(U.dequantize_mxfp8(x8, "bfloat16")[-tail:], U.dequantize_mxfp8(U.quantize_mxfp8(x[-tail:].contiguous()), "bfloat16"))


def test_refusals(dev):
    x, logits, up, down = make(4, 3, 64, 48, torch.float16, dev)
    for args, text in (((up, up, 1, "silu"), "expected"), ((up[:, :48].contiguous(), down, 1, "silu"), "2 \\* hidden"), ((up, down, 1), "expected"),
                       ((up, down, 1, "relu"), "activation"), ((up, down, 1, "silu", "all"), "keep"), ((up[:, :48].contiguous(), down, 1, None, "mxfp8"), "gate"),
                       ((up, down, 4, "silu"), "top_k")):
        with pytest.raises(ValueError, match=text):
            ExpertLayer(*args)
    with pytest.raises(ValueError, match="x: requires a gradient"):
        ExpertLayer(up, down, 1, "silu").quantized()(x.clone().requires_grad_(), logits)
    with pytest.raises(ValueError, match="keep"):
        gated_linear(x, up[0], keep="all")
    with pytest.raises(ValueError, match="activation"):
        gated_linear(x, up[0], activation="tanh")
