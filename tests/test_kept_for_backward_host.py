"""What expert_linear and gated_linear do and hold for a backward pass that will not ask for it, on the CPU: the operators are replaced by plain
products that, like the kernels, leave no trace for autograd."""
import pytest
import torch

from unit_amd import experts as X


class Kept:  # stands for an Mxfp8Tensor
    def __init__(self, buf, shape):
        self.buf, self.shape = buf, shape


def values(x):
    return x.buf if isinstance(x, Kept) else x


@pytest.fixture
def ran(monkeypatch):
    """the operators as plain products of one expert; the names of those that ran"""
    ran = []

    def gated_dense(x, w, sizes, activation, out, keep=None):
        ran.append(("gated", keep))
        pre = (x.detach() @ w.detach().T).unflatten(-1, (2, -1))
        h = torch.nn.functional.silu(pre[:, 0]) * pre[:, 1]
        return h if keep is None else (h, pre if keep == "pre" else Kept(pre, tuple(pre.shape)))

    def gated_grad(x, w, dy, sizes, activation, pre, out, wout, wanted=(True, True)):
        ran.append(("gated_grad", tuple(wanted)))
        read = wanted[1] or pre is None
        assert tuple(x.shape) == (dy.shape[0], w.shape[-1])
        p = ((values(x) @ w.T).unflatten(-1, (2, -1)) if pre is None else values(pre)).detach().requires_grad_()
        with torch.enable_grad():
            dpre, = torch.autograd.grad(torch.nn.functional.silu(p[:, 0]) * p[:, 1], p, dy)
        dpre = dpre.flatten(1)
        return dpre @ w if wanted[0] else None, dpre.T @ values(x) if wanted[1] and read else None

    def grouped_dense(x, w, sizes, out):
        ran.append("grouped")
        return x.detach() @ w.detach()[0].T

    def grouped_grad(x, w, dy, sizes, out, wout, wanted=(True, True)):
        ran.append(("grouped_grad", tuple(wanted)))
        assert tuple(x.shape) == (dy.shape[0], w.shape[-1])
        return dy @ w[0] if wanted[0] else None, (dy.T @ values(x))[None] if wanted[1] else None

    def quantize(x):
        ran.append("quantize")
        return Kept(x.detach().clone(), tuple(x.shape))

    for name, f in (("Mxfp8Tensor", Kept), ("quantize_mxfp8", quantize), ("gated_dense", gated_dense), ("gated_dense_grad", gated_grad), ("_gated_grad", gated_grad),
                    ("grouped_dense", grouped_dense), ("grouped_dense_grad", grouped_grad), ("_grouped_grad", grouped_grad)):
        monkeypatch.setattr(X, name, f)
    return ran


def operands(*lead, n=12, k=16):
    g = torch.Generator().manual_seed(1)
    return torch.randn((7, k), generator=g), torch.randn(lead + (n, k), generator=g)


def test_rows_are_not_quantised_where_nothing_asks_for_a_gradient(ran):
    x, w = operands(1)
    sizes = torch.tensor([7])
    X.expert_linear(x, w, sizes, keep="mxfp8")
    with torch.no_grad():
        y = X.expert_linear(x.requires_grad_(), w.requires_grad_(), sizes, keep="mxfp8")
    assert ran == ["grouped"] * 2 and y.grad_fn is None


def test_evaluating_a_layer_quantises_nothing(ran):
    up, down = torch.randn(1, 12, 16).requires_grad_(), torch.randn(1, 16, 6).requires_grad_()
    layer = X.ExpertLayer(up, down, 1, "silu", "mxfp8")
    layer._hidden = lambda x, sizes, product: torch.randn(x.shape[0], 6)
    with torch.no_grad():
        layer(torch.randn(5, 16), torch.zeros(5, 1))
    assert ran == ["grouped"]


def held(y):
    """elements that the function holds beside the weight and the sizes"""
    return [None if t is None else t.numel() for t in y.grad_fn.saved_tensors]


@pytest.mark.parametrize("keep", ["pre", "mxfp8", "rows"])
@pytest.mark.parametrize("trained", ["x", "w", "both"])
def test_gated_linear_holds_rows_that_are_read_again(ran, keep, trained):
    x, w = operands()
    x.requires_grad_(trained != "w"), w.requires_grad_(trained != "x")
    y = X.gated_linear(x, w, None, "silu", keep)
    rows = 7 * 16 if trained != "x" or keep == "rows" else None
    assert held(y) == [rows, 12 * 16, None, None if keep == "rows" else 7 * 12]
    assert ran.count("quantize") == (1 if keep == "mxfp8" and rows else 0)
    y.square().sum().backward()
    a, b = (t.detach().clone().requires_grad_() for t in (x, w))
    p = (a @ b.T).unflatten(-1, (2, -1))
    (torch.nn.functional.silu(p[:, 0]) * p[:, 1]).square().sum().backward()
    assert (x.grad is None) == (trained == "w") and (w.grad is None) == (trained == "x")
    for ours, want in ((x.grad, a.grad), (w.grad, b.grad)):  # float32 sums of some tens of products, in another order
        assert ours is None or torch.allclose(ours, want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("keep", [None, "mxfp8"])
@pytest.mark.parametrize("trained", ["x", "w", "both"])
def test_expert_linear_holds_rows_that_are_read_again(ran, keep, trained):
    x, w = operands(1)
    x.requires_grad_(trained != "w"), w.requires_grad_(trained != "x")
    y = X.expert_linear(x, w, torch.tensor([7]), keep)
    assert held(y)[:2] == [None if trained == "x" else 7 * 16, 12 * 16]
    assert ran.count("quantize") == (1 if keep == "mxfp8" and trained != "x" else 0)
    y.square().sum().backward()
    a, b = (t.detach().clone().requires_grad_() for t in (x, w))
    (a @ b[0].T).square().sum().backward()
    assert (x.grad is None) == (trained == "w") and (w.grad is None) == (trained == "x")
    for ours, want in ((x.grad, a.grad), (w.grad, b.grad)):
        assert ours is None or torch.allclose(ours, want, rtol=1e-4, atol=1e-4)
