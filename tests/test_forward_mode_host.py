"""Forward-mode derivatives, on the CPU: the layer's products have none, and an operand with a tangent is refused, not taken as a constant.
The operators are replaced by plain products that, like the kernels, leave no trace for autograd."""
import pytest
import torch
from torch.autograd import forward_ad

from unit_amd import experts as X


@pytest.fixture(autouse=True)
def products(monkeypatch):
    def gated_dense(x, w, sizes, activation, out, keep=None):
        pre = (x.detach() @ (w.detach() if sizes is None else w.detach()[0]).T).unflatten(-1, (2, -1))
        h = torch.nn.functional.silu(pre[:, 0]) * pre[:, 1]
        return h if keep is None else (h, pre)

    monkeypatch.setattr(X, "gated_dense", gated_dense)
    monkeypatch.setattr(X, "grouped_dense", lambda x, w, sizes, out: x.detach() @ w.detach()[0].T)


def operands():
    g = torch.Generator().manual_seed(1)
    return torch.randn((5, 16), generator=g), torch.randn((12, 16), generator=g)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("dual", ["x", "w", "both"])
def test_gated_linear_refuses_tangents(dual, grad):
    x, w = operands()
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x, w = (forward_ad.make_dual(t, torch.ones_like(t)) if dual in (n, "both") else t for n, t in (("x", x), ("w", w)))
        with pytest.raises(NotImplementedError, match="jvp"):
            X.gated_linear(x, w)


@pytest.mark.parametrize("keep", ["pre", "rows"])
def test_and_so_do_operands_that_train(keep):
    x, w = operands()
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            X.gated_linear(forward_ad.make_dual(x, torch.ones_like(x)), w.requires_grad_(), keep=keep)


def test_function_transforms_are_refused():
    x, w = operands()
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: X.gated_linear(t, w), (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("gate", [None, "silu"])
def test_layer_of_frozen_weights_refuses_tangents(gate):
    x, _ = operands()
    up, down = torch.randn(1, 12 if gate else 6, 16), torch.randn(1, 16, 6)
    layer = X.ExpertLayer(up, down, 1, gate)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            layer(forward_ad.make_dual(x, torch.ones_like(x)), torch.zeros(5, 1))
        assert layer(x, torch.zeros(5, 1)).shape == x.shape  # a level alone changes nothing


def test_a_level_without_tangents_keeps_nothing():
    x, w = operands()
    with forward_ad.dual_level():
        assert X.gated_linear(x, w).grad_fn is None


@pytest.mark.parametrize("gate", [None, "silu"])
def test_layer_of_mxfp4_weights_refuses_tangents_of_its_rows(monkeypatch, gate):
    product = lambda x, w, *rest: torch.full((x.shape[0], 6 if w.shape[1] == 12 else w.shape[1]), 0.5, dtype=x.dtype)
    monkeypatch.setattr(X, "grouped_dense_mxfp4", product)
    monkeypatch.setattr(X, "gated_dense_mxfp4", product)
    weight = lambda *shape: X.Mxfp4Tensor(torch.empty(0, dtype=torch.uint8), shape)
    layer = X.ExpertLayer(weight(3, 12 if gate else 6, 16), weight(3, 16, 6), 2, gate)
    x, logits = torch.randn(5, 16), torch.randn(5, 3)
    with forward_ad.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="x: carries a forward-mode tangent"):
                layer(forward_ad.make_dual(x, torch.ones_like(x)), logits)
        y = layer(x, forward_ad.make_dual(logits, torch.ones_like(logits)))  # the router's derivative is whole
        assert forward_ad.unpack_dual(y).tangent is not None
