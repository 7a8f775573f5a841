"""The expert layer on the GPU at its edges: no tokens, gradients that begin on any element, frozen operands."""
import pytest
import torch

import unit_amd as U
from unit_amd.experts import ExpertLayer, expert_linear

pytestmark = pytest.mark.gpu


def make(tokens, experts, model, hidden, dtype, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    x, logits = r(tokens, model).to(dtype).to(dev), r(tokens, experts).to(dev)
    return x, logits, (r(experts, hidden, model) / model ** 0.5).to(dtype).to(dev), (r(experts, model, hidden) / hidden ** 0.5).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_no_tokens(dev, dtype):
    x, logits, up, down = (t.requires_grad_() for t in make(0, 5, 64, 40, dtype, dev))
    y = ExpertLayer(up, down, 2)(x, logits)
    assert y.shape == (0, 64) and y.dtype == dtype
    y.float().sum().backward()
    assert x.grad.shape == (0, 64) and not bool(up.grad.any()) and not bool(down.grad.any())
    with torch.no_grad():
        assert ExpertLayer(up, down, 2).quantized()(x, logits).shape == (0, 64)


def test_gradients_that_begin_anywhere(dev):
    x, _, up, _ = (t.requires_grad_() for t in make(40, 3, 64, 48, torch.bfloat16, dev))
    sizes = torch.tensor([10, 0, 30], device=dev)
    expert_linear(x, up, sizes).float().square().sum().backward()
    want = x.grad, up.grad
    x.grad = up.grad = None
    head = torch.ones(1, device=dev, dtype=torch.bfloat16, requires_grad=True)
    y = expert_linear(x, up, sizes)
    parts = torch.cat((head, y.flatten()))
    parts.backward(torch.cat((head.detach(), (2 * y.detach().float()).to(y.dtype).flatten())))
    assert torch.equal(x.grad, want[0]) and torch.equal(up.grad, want[1])


def test_frozen_operands(dev):
    """The same gradient with the other operand frozen, from its kernel alone and without the other's memory."""
    x, _, up, _ = (t.requires_grad_() for t in make(40, 64, 256, 512, torch.float16, dev))
    sizes = torch.zeros(64, dtype=torch.int64, device=dev)
    sizes[3], sizes[50] = 10, 30
    expert_linear(x, up, sizes).float().sum().backward()
    want = x.grad, up.grad
    for trained, frozen, i, kernel in ((x, up, 0, "groupeddx"), (up, x, 1, "groupeddw")):
        frozen.requires_grad_(False)
        x.grad = up.grad = None
        y = expert_linear(x, up, sizes).float().sum()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        ran = []
        hook = trained.register_hook(lambda g: ran.append(U.last_variant()))  # on autograd's thread, like the calls
        y.backward()
        torch.cuda.synchronize()
        hook.remove()
        assert len(ran) == 1 and kernel in ran[0]
        assert torch.equal(trained.grad, want[i]) and frozen.grad is None
        if i == 0:  # 16 MiB of weight gradients are not allocated
            assert torch.cuda.max_memory_allocated() - before < 4 << 20
        frozen.requires_grad_()
