"""The expert layer on the GPU where it has little to do: no tokens."""
import pytest
import torch

from unit_amd.experts import ExpertLayer

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
