"""Gated products and checkpoints near their limits: a weight of almost 2^31 bytes, whose gradient in float32 is twice as long, and rows whose
pieces of eight elements pass 2^30, where the kernels go by slices of them."""
import pytest
import torch

import unit_amd as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("n,k", [(16376, 32768), (120, (1 << 22) - 64)])
def test_weight_of_2_31_bytes(dev, n, k, rows):
    """Integer operands, most of them zero: every sum is exact; silu(0) = 0, and silu(z) of the few integers is off by a few 2^-22.  The
    gradients' products are of gate gradients rounded to 16 bits (2^-8), K of them at most sixteen."""
    g = torch.Generator(device=dev).manual_seed(rows)
    w = torch.zeros((2 * n, k), dtype=torch.bfloat16, device=dev)
    at = torch.cat((torch.randint(0, k, (14,), generator=g, device=dev), torch.tensor([0, k - 1], device=dev)))  # the columns that are not zero
    w[:, at] = torch.randint(-1, 2, (2 * n, len(at)), generator=g, device=dev).bfloat16()
    x = torch.randint(-2, 3, (rows, k), generator=g, device=dev, dtype=torch.int8).bfloat16()
    h, pre = U.gated_dense(x, w, keep="pre")
    cols = torch.unique(at)
    want = (x[:, cols].double() @ w[:, cols].double().T).unflatten(-1, (2, n))
    assert torch.equal(pre.double(), want)
    assert float((h.double() - torch.nn.functional.silu(want[:, 0]) * want[:, 1]).abs().max()) <= 2.0 ** -22 * 64 * 64 * 40
    dy = torch.randint(-1, 2, (rows, n), generator=g, device=dev, dtype=torch.int8).bfloat16()
    z = want.clone().requires_grad_()
    dpre, = torch.autograd.grad(torch.nn.functional.silu(z[:, 0]) * z[:, 1], z, dy.double())
    dpre = dpre.flatten(1)
    for kept in (pre, None):
        dx, dw = U.gated_dense_grad(x, w, dy, pre=kept)
        assert dw.shape == w.shape
        exact = dpre @ w[:, cols].double()
        assert float((dx[:, cols].double() - exact).norm() / exact.norm()) <= 2.0 ** -8
        zero = torch.ones(k, dtype=torch.bool, device=dev)
        zero[cols] = False
        assert not bool(dx[:, zero].any())
        for c in range(0, k, k // 4):
            part = dpre.T.float() @ x[:, c:c + 2048].float()
            assert float((dw[:, c:c + 2048] - part).norm() / part.norm()) <= 2.0 ** -8
        part = dpre.T.float() @ x[:, -2048:].float()
        assert float((dw[:, -2048:] - part).norm() / part.norm()) <= 2.0 ** -8
        del dx, dw


def test_rows_by_slices(dev):
    """2^20 rows and some of 8192: 2^30 pieces and more of checkpoints and of gate gradients.  The last rows against a call of their own; all
    others are zero and stay it."""
    rows, n, k, tail = (1 << 20) + 700, 8192, 8, 500
    g = torch.Generator(device=dev).manual_seed(1)
    x = torch.zeros((rows, k), dtype=torch.bfloat16, device=dev)
    x[-tail:] = torch.randn((tail, k), generator=g, device=dev).bfloat16()
    w = torch.randn((2 * n, k), generator=g, device=dev).bfloat16()
    few, few_pre = U.gated_dense(x[-tail:].contiguous(), w, None, "silu", "bfloat16", keep="pre")
    h, pre8 = U.gated_dense(x, w, None, "silu", "bfloat16", keep="mxfp8")
    # one product's worth of roundings: K = 8 terms, whatever tile they are summed in
    assert float((h[-tail:].double() - few.double()).norm() / few.double().norm()) <= 2.0 ** -7 and not bool(h[:-tail].any())
    few8 = U.quantize_mxfp8(few)
    q = U.quantize_mxfp8(h)
    back = U.dequantize_mxfp8(q, "bfloat16")
    assert torch.equal(back[-tail:], U.dequantize_mxfp8(U.quantize_mxfp8(h[-tail:].contiguous()), "bfloat16")) and not bool(back[:-tail].any())
    assert few8.shape == few.shape
    del q, back
    dx, dw = U.gated_dense_grad(x, w, h, None, "silu", pre8, "bfloat16", "float32")
    few_dx, few_dw = U.gated_dense_grad(x[-tail:].contiguous(), w, few, None, "silu", few_pre, "bfloat16", "float32")
    for a, b in ((dx[-tail:], few_dx), (dw, few_dw)):  # pre-activations in 8 bits against 16: a sixteenth each of two factors
        assert float((a.double() - b.double()).norm() / b.double().norm()) <= 2 * 2.0 ** -4
    assert not bool(dx[:-tail].any())
