"""A feed-forward layer of experts on the grouped products: tokens are routed to their `top_k` experts, sorted by expert, taken through
an up and a down product, or a gated one and a down product, and put together again.  16-bit weights, trainable through torch.autograd
(`expert_linear`, `gated_linear`), activations kept in 16 bits, in MXFP8 or not at all, or MXFP4 weights for serving.  No counterpart in
the reference.

  python -m unit_amd.experts [TOKENS EXPERTS TOP_K MODEL HIDDEN [silu|gelu_tanh]]     times both, forward and training step; gated
"""
import sys
import time

import torch
from torch.autograd import forward_ad

from .gated import _activation, _gated_grad, gated_dense, gated_dense_grad, gated_dense_mxfp4
from .grouped import Mxfp4Tensor, Mxfp8Tensor, _grouped_grad, grouped_dense, grouped_dense_grad, grouped_dense_mxfp4, quantize_mxfp4, quantize_mxfp8

__all__ = ["ExpertLayer", "expert_linear", "gated_linear", "route"]

_NAME = {torch.float32: "float32", torch.float16: "float16", torch.bfloat16: "bfloat16"}


def _name(x):
    try:
        return _NAME[x.dtype]
    except (KeyError, AttributeError):
        _tensor(x, "x")
        raise TypeError(f"x: expected dtype {' or '.join(str(d) for d in _NAME)}, got {x.dtype}") from None


def _tensor(t, name, kinds=torch.Tensor, expected="a torch.Tensor"):
    if not isinstance(t, kinds):
        raise TypeError(f"{name}: expected {expected}, got {type(t).__name__}")


def _derived(x, weight):
    """whether a derivative may be asked for: in the backward pass, or in forward mode, whose tangents an autograd function refuses and a
    bare product would drop"""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return True
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside of any level nothing has a tangent: asking each operand takes a microsecond
        return False
    return any(forward_ad.unpack_dual(t).tangent is not None for t in (x, weight))


def _aligned(grad):
    grad = grad.contiguous()
    if grad.data_ptr() % 16:  # a part of a larger gradient (torch.cat's, say): the kernels read 16 bytes at a time
        grad = grad.clone()
    return grad


def _once(name):
    if torch.is_grad_enabled():  # the products below leave no trace: a derivative of these gradients would lack its part
        raise RuntimeError(f"{name}: its gradients have no derivative of their own (create_graph=True)")


def _keep(ctx, *kept):
    """what the backward pass needs: tensors as autograd keeps them, of an Mxfp8Tensor its buffer and shape"""
    ctx.shapes = [t.shape if isinstance(t, Mxfp8Tensor) else None for t in kept]
    ctx.save_for_backward(*(t.buf if isinstance(t, Mxfp8Tensor) else t for t in kept))


def _kept(ctx):
    return [t if shape is None else Mxfp8Tensor(t, shape) for t, shape in zip(ctx.saved_tensors, ctx.shapes)]


def _rows_kept(ctx, x, keep):
    """the rows as the backward pass reads them: for the weight's gradient, or to compute pre-activations again; None where it does neither"""
    if not ctx.needs_input_grad[1] and keep != "rows":
        return None
    return quantize_mxfp8(x) if keep == "mxfp8" else x


def _unread(weight, grad):
    """in the place of rows that were not kept: of their shape, an element's memory"""
    return weight.new_empty(()).expand(grad.shape[0], weight.shape[-1])


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, group_sizes, keep):
        ctx.name = _name(x)
        _keep(ctx, _rows_kept(ctx, x, keep), weight, group_sizes)
        return grouped_dense(x, weight, group_sizes, _name(x))

    @staticmethod
    def backward(ctx, grad):
        _once("expert_linear")
        x, weight, group_sizes = _kept(ctx)
        wanted = ctx.needs_input_grad[:2]  # a frozen operand's gradient is not computed
        x = _unread(weight, grad) if x is None else x
        args = x, weight, _aligned(grad), group_sizes, ctx.name, _NAME[weight.dtype]
        return *(grouped_dense_grad(*args) if all(wanted) else _grouped_grad(*args, wanted)), None, None


def expert_linear(x, weight, group_sizes, keep=None):
    """grouped_dense in x's type, differentiable in x and weight, once: a backward pass with create_graph=True is refused.
    x is held for it where the weight asks for a gradient; keep "mxfp8": in 8 bits."""
    if keep not in (None, "mxfp8"):
        raise ValueError(f"keep: expected None or 'mxfp8', got {keep!r}")
    _tensor(x, "x")
    _tensor(weight, "weight")
    if not _derived(x, weight):
        return grouped_dense(x, weight, group_sizes, _name(x))
    return _ExpertLinear.apply(x, weight, group_sizes, keep)


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, group_sizes, activation, keep):
        ctx.name, ctx.activation = _name(x), activation
        if keep == "rows":
            h, pre = gated_dense(x, weight, group_sizes, activation, _name(x)), None
        else:
            h, pre = gated_dense(x, weight, group_sizes, activation, _name(x), keep=keep)
        _keep(ctx, _rows_kept(ctx, x, keep), weight, group_sizes, pre)
        return h

    @staticmethod
    def backward(ctx, grad):
        _once("gated_linear")
        x, weight, group_sizes, pre = _kept(ctx)
        wanted = ctx.needs_input_grad[:2]
        x = _unread(weight, grad) if x is None else x
        args = x, weight, _aligned(grad), group_sizes, ctx.activation, pre, ctx.name, _NAME[weight.dtype]
        return *(gated_dense_grad(*args) if all(wanted) else _gated_grad(*args, wanted)), None, None, None


def gated_linear(x, weight, group_sizes=None, activation="silu", keep="pre"):
    """gated_dense in x's type, differentiable in x and weight, once, by the backward pass alone (forward mode is refused).  keep: what it
    holds until then beside the weight, bytes per row of 16-bit operands: "pre" x and the pre-activations (2 K + 4 N), "mxfp8" both in
    8 bits (K + 2 N and a thirty-second), "rows" x alone (2 K): the pre-activations are computed again.  With a frozen weight x is held
    for "rows" alone."""
    if keep not in ("pre", "mxfp8", "rows"):
        raise ValueError(f"keep: expected 'pre', 'mxfp8' or 'rows', got {keep!r}")
    _activation(activation)
    _tensor(x, "x")
    _tensor(weight, "weight")
    if not _derived(x, weight):
        return gated_dense(x, weight, group_sizes, activation, _name(x))
    return _GatedLinear.apply(x, weight, group_sizes, activation, keep)


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
    """y[t] = sum over t's experts e of share * down[e] . silu(up[e] . x[t]), or, with gate "silu" or "gelu_tanh", of
    share * down[e] . (gate(g[e] . x[t]) * (u[e] . x[t])), g[e] the first half of up[e]'s rows and u[e] the second.

    up (E, hidden, model), gated (E, 2 * hidden, model), and down (E, model, hidden): float16 or bfloat16 tensors of x's type, or
    Mxfp4Tensors, for which x has no gradient (an x that asks for one is refused) and the logits have theirs.
    keep, of a gated layer: what it holds for the backward pass, as in gated_linear; with "mxfp8" down's rows are in 8 bits too."""

    def __init__(self, up, down, top_k, gate=None, keep="pre"):
        if gate is not None:
            _activation(gate)
        if keep not in ("pre", "mxfp8", "rows"):
            raise ValueError(f"keep: expected 'pre', 'mxfp8' or 'rows', got {keep!r}")
        if gate is None and keep != "pre":
            raise ValueError(f"keep: {keep!r} is of a layer with a gate")
        for name, t in (("up", up), ("down", down)):
            _tensor(t, name, (torch.Tensor, Mxfp4Tensor), "a torch.Tensor or an Mxfp4Tensor")
        times, width = (1, "hidden") if gate is None else (2, "2 * hidden")
        if not len(up.shape) == len(down.shape) == 3 or up.shape[0] != down.shape[0] or up.shape[1] != times * down.shape[2] or up.shape[2] != down.shape[1]:
            raise ValueError(f"up {tuple(up.shape)}, down {tuple(down.shape)}: expected (E, {width}, model) and (E, model, hidden)")
        if isinstance(up, Mxfp4Tensor) != isinstance(down, Mxfp4Tensor):
            raise TypeError("up, down: both or neither in MXFP4")
        if not 0 < top_k <= up.shape[0]:
            raise ValueError(f"top_k: {top_k} of {up.shape[0]} experts")
        self.up, self.down, self.top_k, self.gate, self.keep = up, down, top_k, gate, keep

    def quantized(self):
        """The same layer with MXFP4 weights."""
        if isinstance(self.up, Mxfp4Tensor):
            raise TypeError("quantized: the layer's weights are in MXFP4 already")
        return ExpertLayer(quantize_mxfp4(self.up.detach()), quantize_mxfp4(self.down.detach()), self.top_k, self.gate, self.keep)

    def _hidden(self, x, sizes, product):
        if self.gate is None:
            return torch.nn.functional.silu(product(x, self.up))
        if isinstance(self.up, Mxfp4Tensor):
            return gated_dense_mxfp4(x, self.up, sizes, self.gate, _name(x))
        return gated_linear(x, self.up, sizes, self.gate, self.keep)

    def __call__(self, x, logits):
        name = _name(x)
        if x.dim() != 2:
            raise ValueError(f"x: expected two axes, got shape {tuple(x.shape)}")
        _tensor(logits, "logits")
        if tuple(logits.shape) != (x.shape[0], self.up.shape[0]):
            raise ValueError(f"logits: expected ({x.shape[0]}, {self.up.shape[0]}), got {tuple(logits.shape)}")
        if isinstance(self.up, Mxfp4Tensor):
            if x.requires_grad and torch.is_grad_enabled():
                raise ValueError("x: requires a gradient, which a layer with MXFP4 weights has none of; detach it or use torch.no_grad()")
            if _derived(x, x):
                raise ValueError("x: carries a forward-mode tangent, which a layer with MXFP4 weights has no derivative for")
        order, token, sizes, share = route(logits, self.top_k)
        if isinstance(self.up, Mxfp4Tensor):
            product = lambda a, w: grouped_dense_mxfp4(a, w, sizes, name)  # noqa: E731
        else:
            kept = "mxfp8" if self.gate is not None and self.keep == "mxfp8" else None
            product = lambda a, w: expert_linear(a, w, sizes, kept)  # noqa: E731
        y = product(self._hidden(x[token], sizes, product), self.down)
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
    gate = argv[5] if len(argv) > 5 else None
    tokens, experts, top_k, model, hidden = (int(a) for a in argv[:5]) if argv else (2048, 16, 2, 1024, 2048)
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    wide = hidden if gate is None else 2 * hidden
    up, down = ((rand(experts, a, b) / b ** 0.5).bfloat16().requires_grad_() for a, b in ((wide, model), (model, hidden)))
    x, logits = rand(tokens, model).bfloat16().requires_grad_(), rand(tokens, experts)
    layer = ExpertLayer(up, down, top_k, gate)
    served = layer.quantized()

    def step(layer):
        layer(x, logits).float().square().mean().backward()
        x.grad = up.grad = down.grad = None

    with torch.no_grad():
        y, q = layer(x, logits).float(), served(x, logits).float()
        print(f"{tokens} tokens, {top_k} of {experts} experts, {model} -> {hidden} -> {model}" + ("" if gate is None else f", gated by {gate}"))
        print(f"bf16 forward          {_time(lambda: layer(x, logits)):9.1f} us")
        print(f"MXFP4 forward         {_time(lambda: served(x, logits)):9.1f} us   relative difference {float((q - y).norm() / y.norm()):.3f}")
    for keep in ("pre",) if gate is None else ("pre", "mxfp8", "rows"):
        kept = ExpertLayer(up, down, top_k, gate, keep)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = kept(x, logits)
        held = torch.cuda.memory_allocated() - before
        del loss
        print(f"bf16 forward and back {_time(lambda: step(kept)):9.1f} us" + ("" if gate is None else f"   keep {keep!r}: {held / 2 ** 20:.1f} MiB until the backward pass"))


if __name__ == "__main__":
    main(sys.argv[1:])
