"""Gradients of products of which one operand is frozen: the same as where both train, and what they hold and take on the way."""
import pytest
import torch

import unit_amd as U
from unit_amd.experts import expert_linear, gated_linear

pytestmark = pytest.mark.gpu


def operands(rows, experts, n, k, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)
    lead = (experts,) if experts else ()
    return r(rows, k).bfloat16().to(dev), (r(*lead, n, k) / k ** 0.5).bfloat16().to(dev)


def asked(which="current"):
    """bytes asked of the allocator and not given back; its blocks may be larger, by what it has at hand"""
    return torch.cuda.memory_stats()[f"requested_bytes.all.{which}"]


def held_by(call):
    """bytes that `call` leaves allocated beside its result, which it returns"""
    torch.cuda.synchronize()
    before = asked()
    y = call()
    return y, asked() - before - y.numel() * y.element_size()


def test_rows_that_a_frozen_weight_leaves_unread_are_not_held(dev):
    rows, k, n = 4096, 512, 1024
    x, w = operands(rows, 0, 2 * n, k, dev)
    x.requires_grad_()
    for keep, want in (("pre", rows * 4 * n), ("mxfp8", rows * 2 * n * 33 // 32), ("rows", rows * 2 * k)):
        y, held = held_by(lambda: gated_linear(x * 1.0, w, keep=keep))
        assert held == want
        y.float().sum().backward()
        del y
    w, sizes = w[None], torch.tensor([rows], device=dev)
    for keep in (None, "mxfp8"):
        y, held = held_by(lambda: expert_linear(x * 1.0, w, sizes, keep))
        assert held == 0
        y.float().sum().backward()
        del y


@pytest.mark.parametrize("keep", ["pre", "mxfp8", "rows"])
@pytest.mark.parametrize("rows,experts,n,k", [(40, 3, 96, 64), (300, 0, 272, 136), (9, 2, 16, 72), (0, 2, 16, 72)])
def test_gradient_of_the_rows_alone(dev, keep, rows, experts, n, k):
    """dx with a frozen weight against dx of gated_dense_grad: the same sums in another order of tiles, rounded once (2^-8)."""
    x, w = operands(rows, experts, n, k, dev)
    sizes = torch.tensor([rows // 2] + [rows - rows // 2 - rows // 7] + [0] * (experts - 2), device=dev) if experts else None
    seed = torch.randn((rows, n // 2), generator=torch.Generator().manual_seed(5)).bfloat16().to(dev)
    kept = None if keep == "rows" else U.gated_dense(x, w, sizes, "silu", "bfloat16", keep=keep)[1]
    want = U.gated_dense_grad(x, w, seed, sizes, "silu", kept, "bfloat16", "bfloat16")[0]
    a = x.clone().requires_grad_()
    gated_linear(a, w, sizes, "silu", keep).backward(seed)
    assert a.grad.shape == want.shape and float((a.grad.double() - want.double()).norm()) <= 2 * 2.0 ** -8 * float(want.double().norm())


@pytest.mark.parametrize("keep", [None, "mxfp8"])
def test_gradient_of_a_plain_product_s_rows_alone(dev, keep):
    x, w = operands(60, 3, 40, 96, dev)
    sizes = torch.tensor([20, 0, 35], dtype=torch.int32, device=dev)
    seed = torch.randn((60, 40), generator=torch.Generator().manual_seed(6)).bfloat16().to(dev)
    a = x.clone().requires_grad_()
    expert_linear(a, w, sizes, keep).backward(seed)
    assert torch.equal(a.grad, U.grouped_dense_grad(x, w, seed, sizes, "bfloat16", "bfloat16")[0])


def test_evaluation_takes_no_checkpoint(dev):
    """Under no_grad, and with nothing that trains, the product alone."""
    x, w = operands(60, 3, 40, 96, dev)
    sizes = torch.tensor([20, 0, 35], dtype=torch.int32, device=dev)
    want = U.grouped_dense(x, w, sizes, "bfloat16")
    expert_linear(x, w, sizes, keep="mxfp8")
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = asked()
    got = expert_linear(x, w, sizes, keep="mxfp8")
    assert asked("peak") - before == got.numel() * 2  # the result alone
    assert torch.equal(got, want) and got.grad_fn is None
    with torch.no_grad():
        assert torch.equal(expert_linear(x.clone().requires_grad_(), w, sizes, keep="mxfp8"), want)


def peak_of(call):
    """bytes that `call` has allocated at a time, its results among them"""
    call()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = asked()
    out = call()
    return asked("peak") - before, out


@pytest.mark.parametrize("keep", ["pre", "mxfp8", "rows"])
def test_a_single_gradient_takes_its_own_workspace(dev, keep):
    """The gate's gradients; for dw, or where pre-activations are computed again, the rows restored from MXFP8.  No sums of dw's splits."""
    from unit_amd.gated import _gated_grad
    rows, n, k = 10000, 256, 256  # whose dw alone is shared out to many workgroups beside dx
    x, w = operands(rows, 0, 2 * n, k, dev)
    seed = torch.randn((rows, n), generator=torch.Generator().manual_seed(5)).bfloat16().to(dev)
    pre = None if keep == "rows" else U.gated_dense(x, w, None, "silu", "bfloat16", keep=keep)[1]
    data = U.quantize_mxfp8(x) if keep != "pre" else x
    want = U.gated_dense_grad(data, w, seed, None, "silu", pre, "bfloat16", "bfloat16")
    restored = -(-rows * k * 2 // 256) * 256 if keep != "pre" else 0
    for wanted, result, x16 in (((True, False), rows * k * 2, restored if pre is None else 0), ((False, True), 2 * n * k * 2, restored)):
        peak, both = peak_of(lambda: _gated_grad(data, w, seed, None, "silu", pre, "bfloat16", "bfloat16", wanted))
        assert peak == rows * n * 4 + x16 + result, (wanted, peak)
        i = wanted.index(True)
        assert both[1 - i] is None and float((both[i].double() - want[i].double()).norm() / want[i].double().norm()) <= 2 * 2.0 ** -8
