"""What the gated layer does around its products, on the CPU: the operators are replaced by plain products that, like the kernels, leave no
trace for autograd."""
import pytest
import torch

from unit_amd import experts as X
from unit_amd.grouped import Mxfp4Tensor, Mxfp8Tensor


def _groups(sizes, rows):
    at = 0
    for g, n in enumerate([rows] if sizes is None else sizes.tolist()):
        yield (None if sizes is None else g), slice(at, at + n)
        at += n


def _pre(x, w, sizes):
    pre = x.new_zeros((x.shape[0], w.shape[-2]))
    for g, r in _groups(sizes, len(x)):
        pre[r] = x[r] @ (w if g is None else w[g]).T
    return pre.unflatten(-1, (2, -1))


@pytest.fixture
def products(monkeypatch):
    """the gated operators and the checkpoints as plain ones; what ran"""
    ran = []

    class Kept:  # stands for an Mxfp8Tensor
        def __init__(self, buf, shape):
            self.buf, self.shape = buf, shape

    def gated_dense(x, w, sizes, activation, out, keep=None):
        ran.append(("forward", keep))
        pre = _pre(x.detach(), w.detach(), sizes)
        h = torch.nn.functional.silu(pre[:, 0]) * pre[:, 1]
        return h if keep is None else (h, pre if keep == "pre" else Kept(pre, tuple(pre.shape)))

    def grad(x, w, dy, sizes, activation, pre, out, wout, wanted=(True, True)):
        ran.append(("backward", type(x).__name__, None if pre is None else type(pre).__name__, tuple(wanted)))
        x = x.buf if isinstance(x, Kept) else x
        pre = _pre(x.detach(), w.detach(), sizes) if pre is None else pre.buf if isinstance(pre, Kept) else pre
        with torch.enable_grad():
            p = pre.detach().requires_grad_()
            dpre, = torch.autograd.grad(torch.nn.functional.silu(p[:, 0]) * p[:, 1], p, dy)
        dpre, dx, dw = dpre.flatten(1), torch.zeros_like(x), torch.zeros_like(w)
        for g, r in _groups(sizes, len(x)):
            dx[r] = dpre[r] @ (w if g is None else w[g])
            (dw if g is None else dw[g]).copy_(dpre[r].T @ x[r])
        return dx if wanted[0] else None, dw if wanted[1] else None

    monkeypatch.setattr(X, "Mxfp8Tensor", Kept)
    monkeypatch.setattr(X, "quantize_mxfp8", lambda x: Kept(x.detach().clone(), tuple(x.shape)))
    monkeypatch.setattr(X, "gated_dense", gated_dense)
    monkeypatch.setattr(X, "gated_dense_grad", grad)
    monkeypatch.setattr(X, "_gated_grad", grad)
    return ran


def operands(sizes, n=8, k=16):
    g = torch.Generator().manual_seed(1)
    lead = () if sizes is None else (3,)
    return torch.randn((7, k), generator=g), torch.randn(lead + (2 * n, k), generator=g), None if sizes is None else torch.tensor(sizes)


@pytest.mark.parametrize("sizes", [None, [2, 0, 5]], ids=["dense", "experts"])
@pytest.mark.parametrize("keep", ["pre", "mxfp8", "rows"])
def test_gradients_and_what_is_kept(products, keep, sizes):
    x, w, s = operands(sizes)
    x.requires_grad_(), w.requires_grad_()
    y = X.gated_linear(x, w, s, "silu", keep)
    y.square().sum().backward()
    rows, pre = {"pre": ("Tensor", "Tensor"), "mxfp8": ("Kept", "Kept"), "rows": ("Tensor", None)}[keep]
    assert products == [("forward", None if keep == "rows" else keep), ("backward", rows, pre, (True, True))]
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    p = _pre(a, b, s) if s is None else torch.cat([a[r] @ b[g].T for g, r in _groups(s, 7)]).unflatten(-1, (2, -1))
    (torch.nn.functional.silu(p[:, 0]) * p[:, 1]).square().sum().backward()
    # float32 sums of some tens of products, in another order
    assert torch.allclose(x.grad, a.grad, rtol=1e-4, atol=1e-4) and torch.allclose(w.grad, b.grad, rtol=1e-4, atol=1e-4)


def test_nothing_is_kept_without_a_gradient(products):
    x, w, _ = operands(None)
    X.gated_linear(x, w)
    with torch.no_grad():
        X.gated_linear(x.requires_grad_(), w)
    assert products == [("forward", None)] * 2


@pytest.mark.parametrize("trained", ["x", "w"])
def test_frozen_operands(products, trained):
    x, w, _ = operands(None)
    (x if trained == "x" else w).requires_grad_()
    X.gated_linear(x, w).square().sum().backward()
    assert products[-1][-1] == (trained == "x", trained == "w")
    assert (x.grad is None) == (trained == "w") and (w.grad is None) == (trained == "x")


def test_second_derivatives_are_refused(products):
    x, w, _ = operands(None)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="gated_linear: .*create_graph"):
        torch.autograd.grad(X.gated_linear(x, w).square().sum(), x, create_graph=True)


def test_gradients_that_begin_anywhere_reach_the_products_aligned(products, monkeypatch):
    x, w, _ = operands(None)
    x.requires_grad_(), w.requires_grad_()
    seen, plain = [], X.gated_dense_grad
    monkeypatch.setattr(X, "gated_dense_grad", lambda x, w, dy, *rest: (seen.append((dy.data_ptr() % 16, dy.is_contiguous())), plain(x, w, dy, *rest))[1])
    torch.cat((torch.ones(1), X.gated_linear(x, w).flatten())).square().sum().backward()
    assert seen == [(0, True)]


def test_arguments_are_refused_by_name():
    x, w, _ = operands(None)
    for call, text in ((lambda: X.gated_linear(x, w, keep="16"), "keep: expected"), (lambda: X.gated_linear(x, w, activation="tanh"), "activation: expected"),
                       (lambda: X.expert_linear(x, w, None, keep="pre"), "keep: expected"),
                       (lambda: X.ExpertLayer(torch.zeros(3, 24, 16), torch.zeros(3, 16, 24), 1, "silu"), r"expected \(E, 2 \* hidden, model\)"),
                       (lambda: X.ExpertLayer(torch.zeros(3, 48, 16), torch.zeros(3, 16, 24), 1), r"expected \(E, hidden, model\)"),
                       (lambda: X.ExpertLayer(torch.zeros(3, 48, 16), torch.zeros(3, 16, 24), 1, "relu"), "activation: expected"),
                       (lambda: X.ExpertLayer(torch.zeros(3, 24, 16), torch.zeros(3, 16, 24), 1, None, "rows"), "layer with a gate")):
        with pytest.raises(ValueError, match=text):
            call()
    with pytest.raises(TypeError, match="x: expected dtype"):
        X.gated_linear(x.double(), w.double())


def test_what_is_no_tensor_is_refused():
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(32, 64, dtype=torch.bfloat16)
    codes = torch.zeros(20000, dtype=torch.uint8)
    x4, w4, x8 = Mxfp4Tensor(codes, (4, 64)), Mxfp4Tensor(codes, (32, 64)), Mxfp8Tensor(codes, (4, 64))
    for grad in (True, False):
        with torch.set_grad_enabled(grad):
            for bad in (x4, x8, [1.0]):
                with pytest.raises(TypeError, match="x: expected a torch.Tensor"):
                    X.gated_linear(bad, w)
                with pytest.raises(TypeError, match="x: expected a torch.Tensor"):
                    X.expert_linear(bad, w[None], torch.tensor([4]))
            for bad in (w4, None):
                with pytest.raises(TypeError, match="weight: expected a torch.Tensor"):
                    X.gated_linear(x, bad)
                with pytest.raises(TypeError, match="weight: expected a torch.Tensor"):
                    X.expert_linear(x, bad, torch.tensor([4]))
