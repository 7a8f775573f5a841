"""A feed-forward layer of experts on the grouped products: tokens are routed to their `top_k` experts, sorted by expert, taken through
an up and a down product, and put together again.  16-bit weights, trainable through torch.autograd (`expert_linear`), or MXFP4
weights for serving.  No counterpart in the reference.

  python -m unit_amd.experts [TOKENS EXPERTS TOP_K MODEL HIDDEN]     times both, forward and training step
"""
import sys
import time

import torch

from .grouped import Mxfp4Tensor, _grouped_grad, grouped_dense, grouped_dense_grad, grouped_dense_mxfp4, quantize_mxfp4

__all__ = ["ExpertLayer", "expert_linear", "route"]

_NAME = {torch.float32: "float32", torch.float16: "float16", torch.bfloat16: "bfloat16"}


def _name(x):
    try:
        return _NAME[x.dtype]
    except KeyError:
        raise TypeError(f"x: expected dtype {' or '.join(str(d) for d in _NAME)}, got {x.dtype}") from None


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, group_sizes):
        ctx.save_for_backward(x, weight, group_sizes)
        return grouped_dense(x, weight, group_sizes, _name(x))

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled():  # the products below leave no trace: a derivative of these gradients would lack its part
            raise RuntimeError("expert_linear: its gradients have no derivative of their own (create_graph=True)")
        x, weight, group_sizes = ctx.saved_tensors
        grad = grad.contiguous()
        if grad.data_ptr() % 16:  # a part of a larger gradient (torch.cat's, say): the kernels read 16 bytes at a time
            grad = grad.clone()
        wanted = ctx.needs_input_grad[:2]  # a frozen operand's gradient is not computed
        args = x, weight, grad, group_sizes, _NAME[x.dtype], _NAME[weight.dtype]
        return *(grouped_dense_grad(*args) if all(wanted) else _grouped_grad(*args, wanted)), None


def expert_linear(x, weight, group_sizes):
    """grouped_dense in x's type, differentiable in x and weight, once: a backward pass with create_graph=True is refused."""
    return _ExpertLinear.apply(x, weight, group_sizes)


def route(logits, top_k):
    """logits (tokens, experts) -> (order, token, group_sizes, share): the token-expert pairs sorted by expert, the token of each sorted
    pair, how many pairs each expert has (on the GPU: nothing waits for them), and each token's shares of its experts."""
    best, expert = logits.float().topk(top_k, dim=-1)
    flat = expert.flatten()
    order = torch.argsort(flat, stable=True)
    sizes = torch.zeros((logits.shape[-1],), dtype=torch.int64, device=logits.device)
    sizes.scatter_add_(0, flat, torch.ones_like(flat))
    return order, order // top_k, sizes, torch.softmax(best, -1)


class ExpertLayer:
    """y[t] = sum over t's experts e of share * down[e] . silu(up[e] . x[t]).

    up (E, hidden, model) and down (E, model, hidden): float16 or bfloat16 tensors of x's type, or Mxfp4Tensors, for which
    x has no gradient (an x that asks for one is refused) and the logits have theirs."""

    def __init__(self, up, down, top_k):
        if not len(up.shape) == len(down.shape) == 3 or up.shape[0] != down.shape[0] or up.shape[1] != down.shape[2] or up.shape[2] != down.shape[1]:
            raise ValueError(f"up {tuple(up.shape)}, down {tuple(down.shape)}: expected (E, hidden, model) and (E, model, hidden)")
        if isinstance(up, Mxfp4Tensor) != isinstance(down, Mxfp4Tensor):
            raise TypeError("up, down: both or neither in MXFP4")
        if not 0 < top_k <= up.shape[0]:
            raise ValueError(f"top_k: {top_k} of {up.shape[0]} experts")
        self.up, self.down, self.top_k = up, down, top_k

    def quantized(self):
        """The same layer with MXFP4 weights."""
        return ExpertLayer(quantize_mxfp4(self.up.detach()), quantize_mxfp4(self.down.detach()), self.top_k)

    def __call__(self, x, logits):
        name = _name(x)
        if x.dim() != 2:
            raise ValueError(f"x: expected two axes, got shape {tuple(x.shape)}")
        if tuple(logits.shape) != (x.shape[0], self.up.shape[0]):
            raise ValueError(f"logits: expected ({x.shape[0]}, {self.up.shape[0]}), got {tuple(logits.shape)}")
        if isinstance(self.up, Mxfp4Tensor) and x.requires_grad and torch.is_grad_enabled():
            raise ValueError("x: requires a gradient, which a layer with MXFP4 weights has none of; detach it or use torch.no_grad()")
        order, token, sizes, share = route(logits, self.top_k)
        if isinstance(self.up, Mxfp4Tensor):
            product = lambda a, w: grouped_dense_mxfp4(a, w, sizes, name)  # noqa: E731
        else:
            product = lambda a, w: expert_linear(a, w, sizes)  # noqa: E731
        y = product(torch.nn.functional.silu(product(x[token], self.up)), self.down)
        back = torch.empty_like(order).scatter_(0, order, torch.arange(len(order), device=order.device))
        # every token's pairs side by side again: added in one order, whatever runs beside it
        y = y[back].view(x.shape[0], self.top_k, self.down.shape[1])
        return (y.float() * share.unsqueeze(-1)).sum(1).to(x.dtype)


def _time(f, reps=20):
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(reps):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / reps * 1e6


def main(argv):
    tokens, experts, top_k, model, hidden = (int(a) for a in argv) if argv else (2048, 16, 2, 1024, 2048)
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    up, down = ((rand(experts, a, b) / b ** 0.5).bfloat16().requires_grad_() for a, b in ((hidden, model), (model, hidden)))
    x, logits = rand(tokens, model).bfloat16().requires_grad_(), rand(tokens, experts)
    layer = ExpertLayer(up, down, top_k)
    served = layer.quantized()

    def step():
        layer(x, logits).float().square().mean().backward()
        x.grad = up.grad = down.grad = None

    with torch.no_grad():
        y, q = layer(x, logits).float(), served(x, logits).float()
        print(f"{tokens} tokens, {top_k} of {experts} experts, {model} -> {hidden} -> {model}")
        print(f"bf16 forward          {_time(lambda: layer(x, logits)):9.1f} us")
        print(f"MXFP4 forward         {_time(lambda: served(x, logits)):9.1f} us   relative difference {float((q - y).norm() / y.norm()):.3f}")
    print(f"bf16 forward and back {_time(step):9.1f} us")


if __name__ == "__main__":
    main(sys.argv[1:])
