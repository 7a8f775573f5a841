"""What the expert layer does around its products, on the CPU: the operators are replaced by plain products that, like the kernels,
leave no trace for autograd."""
import pytest
import torch

from unit_amd import experts as X


def _groups(sizes):
    at = 0
    for g, n in enumerate(sizes.tolist()):
        yield g, slice(at, at + n)
        at += n


@pytest.fixture
def products(monkeypatch):
    """grouped_dense and grouped_dense_grad as plain products; the names of those that ran"""
    ran = []

    def forward(x, w, sizes, out_dtype):
        ran.append("forward")
        x, w = x.detach(), w.detach()
        y = x.new_zeros((x.shape[0], w.shape[1]))
        for g, r in _groups(sizes):
            y[r] = x[r] @ w[g].T
        return y

    def backward(x, w, dy, sizes, out_dtype, weight_out_dtype):
        ran.append("both")
        x, w, dy = x.detach(), w.detach(), dy.detach()
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        for g, r in _groups(sizes):
            dx[r], dw[g] = dy[r] @ w[g], dy[r].T @ x[r]
        return dx, dw

    monkeypatch.setattr(X, "grouped_dense", forward)
    monkeypatch.setattr(X, "grouped_dense_grad", backward)
    return ran


def operands(rows=7, experts=3, n=8, k=16, seed=1):
    g = torch.Generator().manual_seed(seed)
    sizes = torch.tensor([2, 0, rows - 2][:experts])
    return torch.randn((rows, k), generator=g), torch.randn((experts, n, k), generator=g), sizes


@pytest.mark.parametrize("loss", [lambda y: y.sum(), lambda y: y.square().sum()], ids=["linear", "square"])
def test_a_gradient_that_is_to_be_differentiated_again_is_refused(products, loss):
    x, w, sizes = operands()
    x.requires_grad_(), w.requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(loss(X.expert_linear(x, w, sizes)), x, create_graph=True)
    loss(X.expert_linear(x, w, sizes)).backward()  # the first derivative is there
    assert x.grad.shape == x.shape and w.grad.shape == w.shape


@pytest.fixture
def quantized(monkeypatch):
    """a layer with MXFP4 weights whose product is a constant"""
    monkeypatch.setattr(X, "grouped_dense_mxfp4", lambda x, w, sizes, out: torch.full((x.shape[0], w.shape[1]), 0.5, dtype=x.dtype))
    weight = lambda *shape: X.Mxfp4Tensor(torch.empty(0, dtype=torch.uint8), shape)
    return X.ExpertLayer(weight(3, 24, 16), weight(3, 16, 24), 2)


def test_mxfp4_layer_refuses_rows_that_want_a_gradient(quantized):
    x, logits = torch.randn(5, 16, requires_grad=True), torch.randn(5, 3, requires_grad=True)
    with pytest.raises(ValueError, match="x: .*gradient"):
        quantized(x, logits)
    with torch.no_grad():
        assert quantized(x, logits).shape == (5, 16)
    quantized(x.detach(), logits).square().sum().backward()  # the router's gradient is whole
    assert logits.grad is not None


def test_no_tokens(products, quantized):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(s, generator=g).requires_grad_()
    up, down, x, logits = r(3, 24, 16), r(3, 16, 24), r(0, 16), r(0, 3)
    y = X.ExpertLayer(up, down, 2)(x, logits)
    assert y.shape == (0, 16)
    y.sum().backward()
    assert x.grad.shape == (0, 16) and logits.grad.shape == (0, 3) and not up.grad.any() and not down.grad.any()
    assert quantized(x.detach(), logits.detach()).shape == (0, 16)


def test_gradients_that_begin_anywhere_reach_the_products_aligned(products, monkeypatch):
    """Joined with other values the result gets its gradient as a part of theirs, at any element."""
    x, w, sizes = operands()
    x.requires_grad_(), w.requires_grad_()
    seen, plain = [], X.grouped_dense_grad
    monkeypatch.setattr(X, "grouped_dense_grad", lambda x, w, dy, *rest: (seen.append((dy.data_ptr() % 16, dy.is_contiguous())), plain(x, w, dy, *rest))[1])
    y = X.expert_linear(x, w, sizes)
    head = torch.ones(1, requires_grad=True)
    torch.cat((head, y.flatten())).square().sum().backward()
    assert seen == [(0, True)]
    got = x.grad, w.grad
    x.grad = w.grad = None
    X.expert_linear(x, w, sizes).square().sum().backward()
    assert torch.equal(got[0], x.grad) and torch.equal(got[1], w.grad)


@pytest.mark.parametrize("trained", ["x", "w"])
def test_frozen_operands_have_no_gradient_computed(products, monkeypatch, trained):
    x, w, sizes = operands()
    x.requires_grad_(), w.requires_grad_()
    X.expert_linear(x, w, sizes).square().sum().backward()
    assert products == ["forward", "both"]
    want = {"x": x.grad, "w": w.grad}[trained]
    (w if trained == "x" else x).requires_grad_(False)
    x.grad = w.grad = None

    def one(data, weight, grad, group_sizes, out_dtype, weight_out_dtype, wanted):
        products.append(wanted)
        both = plain(data, weight, grad, group_sizes, out_dtype, weight_out_dtype)
        return both[0] if wanted[0] else None, both[1] if wanted[1] else None

    plain = X.grouped_dense_grad
    monkeypatch.setattr(X, "_grouped_grad", one)
    monkeypatch.setattr(X, "grouped_dense_grad", lambda *args: pytest.fail("both gradients were computed"))
    X.expert_linear(x, w, sizes).square().sum().backward()
    assert (trained == "x", trained == "w") in products
    assert torch.equal({"x": x.grad, "w": w.grad}[trained], want)


def test_arguments_are_refused_by_name(quantized):
    x, w, sizes = operands()
    with pytest.raises(TypeError, match="x: expected dtype .*float64"):
        X.expert_linear(x.double(), w.double(), sizes)
    with pytest.raises(TypeError, match="x: expected dtype .*int32"):
        quantized(torch.zeros((5, 16), dtype=torch.int32), torch.zeros((5, 3)))
    for up, down in ((torch.zeros(24, 16), torch.zeros(16, 24)), (torch.zeros(3, 24, 16), torch.zeros(3, 16))):
        with pytest.raises(ValueError, match=r"expected \(E, hidden, model\)"):
            X.ExpertLayer(up, down, 1)
    with pytest.raises(ValueError, match="x: expected two axes"):
        quantized(torch.zeros((5, 2, 16)), torch.zeros((5, 3)))
