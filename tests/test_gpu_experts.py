"""The layer of experts against plain products in 64 bits, its gradients through autograd, and its MXFP4 form against the same layer
on the values that its operands stand for.

Tolerances.  16-bit results are rounded where the layer rounds them (two products, the shares' sum), each by at most 2^-8 (bfloat16)
or 2^-11 (float16) of its value; silu and the products carry a relative error on as a whole of no more than a few of them: 8
roundings of the result's norm."""
import pytest
import torch

import unit_amd as U
from unit_amd.experts import ExpertLayer, expert_linear, route

pytestmark = pytest.mark.gpu
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def make(tokens, experts, model, hidden, dtype, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    x, logits = r(tokens, model).to(dtype).to(dev), r(tokens, experts).to(dev)
    up, down = (r(experts, hidden, model) / model ** 0.5).to(dtype).to(dev), (r(experts, model, hidden) / hidden ** 0.5).to(dtype).to(dev)
    return x, logits, up, down


def plain(x, logits, up, down, top_k):
    """every token through every one of its experts, one product at a time, in x's type"""
    best, expert = logits.to(x.dtype).topk(top_k, -1)
    share = torch.softmax(best, -1)
    y = torch.zeros_like(x)
    for j in range(top_k):
        for e in range(up.shape[0]):
            m = expert[:, j] == e
            y = y.index_put((m.nonzero().flatten(),), share[m, j, None] * (torch.nn.functional.silu(x[m] @ up[e].T) @ down[e].T), accumulate=True)
    return y


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts,top_k,model,hidden", [(1, 8, 2, 64, 128), (7, 5, 1, 72, 40), (130, 9, 3, 256, 136), (600, 4, 2, 128, 512)])
def test_layer(dev, dtype, tokens, experts, top_k, model, hidden):
    x, logits, up, down = make(tokens, experts, model, hidden, dtype, dev)
    got = ExpertLayer(up, down, top_k)(x, logits)
    want = plain(x.double(), logits.double(), up.double(), down.double(), top_k)
    assert got.dtype == dtype and got.shape == x.shape
    assert float((got.double() - want).norm() / want.norm()) <= 8 * ROUND[dtype]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_training_step(dev, dtype):
    x, logits, up, down = make(150, 6, 128, 192, dtype, dev)
    seed = torch.randn(x.shape, generator=torch.Generator().manual_seed(3)).to(dev)
    ours = [t.clone().requires_grad_() for t in (x, up, down)]
    (ExpertLayer(ours[1], ours[2], 2)(ours[0], logits).float() * seed).sum().backward()
    exact = [t.double().requires_grad_() for t in (x, up, down)]
    (plain(exact[0], logits.double(), exact[1], exact[2], 2) * seed.double()).sum().backward()
    for a, b in zip(ours, exact):
        assert a.grad.dtype == dtype
        assert float((a.grad.double() - b.grad).norm() / b.grad.norm()) <= 8 * ROUND[dtype]


def test_quantized_layer(dev):
    x, logits, up, down = make(90, 6, 160, 224, torch.bfloat16, dev)
    layer = ExpertLayer(up, down, 2).quantized()
    order, token, sizes, share = route(logits, 2)
    assert int(sizes.sum()) == 180
    values = lambda t: U.dequantize_mxfp4(U.quantize_mxfp4(t)).double()
    wu, wd = U.dequantize_mxfp4(layer.up).double(), U.dequantize_mxfp4(layer.down).double()
    expert = torch.repeat_interleave(torch.arange(6, device=dev), sizes)
    h = torch.bmm(wu[expert], values(x[token]).unsqueeze(-1)).squeeze(-1).bfloat16()
    h = torch.nn.functional.silu(h)
    y = torch.bmm(wd[expert], values(h).unsqueeze(-1)).squeeze(-1).bfloat16().double()
    want = torch.zeros((90, 160), dtype=torch.float64, device=dev).index_add_(0, token, y * share.flatten()[order].double().unsqueeze(-1))
    got = layer(x, logits)
    # the first product may round a value to the other of two neighbours than the 64-bit sum does, and a quantised one moves by a step
    # then: one of several hundred, seldom
    assert float((got.double() - want).norm() / want.norm()) <= 8 * ROUND[torch.bfloat16]


def test_expert_linear_is_the_operator(dev):
    x, _, up, _ = make(40, 3, 64, 48, torch.float16, dev)
    sizes = torch.tensor([10, 0, 25], device=dev)
    assert torch.equal(expert_linear(x, up, sizes), U.grouped_dense(x, up, sizes, "float16"))


def test_refusals(dev):
    x, logits, up, down = make(4, 3, 64, 48, torch.float16, dev)
    with pytest.raises(ValueError, match="expected"):
        ExpertLayer(up, up, 1)
    with pytest.raises(TypeError, match="MXFP4"):
        ExpertLayer(U.quantize_mxfp4(up), down, 1)
    with pytest.raises(ValueError, match="top_k"):
        ExpertLayer(up, down, 4)
    with pytest.raises(ValueError, match="logits"):
        ExpertLayer(up, down, 1)(x, logits[:, :2])
