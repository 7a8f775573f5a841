"""Weight gradients of 16 bits on both sides of the line from which they are written past the caches, whole lines and not.

The same call in float32 sums in the same order, so 16 bits are its result rounded once, to the bit; and float32 is held against 64-bit
products of the gate's gradients rounded to 16 bits: two roundings' worth, 2 * 2^-8 (2^-11 in fp16), of a group's norm."""
import pytest
import torch

import unit_amd as U

pytestmark = pytest.mark.gpu
STEP = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}

CASES = [  # rows, experts (0: one weight), N, K, kept;  dw in MiB, MiB moved
    (300, 20, 512, 1024, None),     # 40: past them
    (300, 19, 512, 1024, None),     # 38
    (300, 21, 512, 1016, None),     # 42, rows of dw that are no whole lines
    (100, 0, 4096, 2560, None),     # 40, one weight
    (100, 0, 4096, 2552, None),
    (3000, 32, 1024, 1024, "pre"),  # 128, 297: past them
    (700, 32, 1024, 960, "pre"),    # 120, 249
    (3000, 32, 1024, 1024, "mxfp8"),
    (3000, 32, 1024, 1000, "pre"),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("rows,experts,n,k,keep", CASES)
def test_large_weight_gradients(dev, rows, experts, n, k, keep, dtype):
    g = torch.Generator(device=dev).manual_seed(rows + k)
    rand = lambda *s: torch.randn(s, generator=g, device=dev)
    t = getattr(torch, dtype)
    lead = (experts,) if experts else ()
    x, w, dy = rand(rows, k).to(t), (rand(*lead, 2 * n, k) / k ** 0.5).to(t), (rand(rows, n) / 32).to(t)
    sizes = torch.zeros(experts, dtype=torch.int64) if experts else None
    if experts:  # the first and the last have none, some rows belong to nobody
        sizes[1:-1] = (rows - 5) // (experts - 2)
        sizes = sizes.to(dev)
    pre = U.gated_dense(x, w, sizes, "silu", dtype, keep=keep)[1] if keep else None
    args = x, w, dy, sizes, "silu", pre
    dx, dw = U.gated_dense_grad(*args, dtype, "float32")
    dx16, dw16 = U.gated_dense_grad(*args, dtype, dtype)
    assert dw16.dtype == t and torch.equal(dw16, dw.to(t)) and torch.equal(dx16, dx)
    for _ in range(2):  # what was written past the caches is what the next call writes over
        again = U.gated_dense_grad(*args, dtype, dtype)[1]
        assert torch.equal(again, dw16)
    del again, dw16
    groups = [(0, slice(0, rows))] if not experts else [(e, slice(int(sizes[:e].sum()), int(sizes[:e + 1].sum()))) for e in (0, 1, experts // 2, experts - 1)]
    kept = None if keep is None else (pre if keep == "pre" else U.dequantize_mxfp8(pre, "float32")).double()
    for e, r in groups:
        we, got = (w, dw) if not experts else (w[e], dw[e])
        z = ((x[r].double() @ we.double().T).unflatten(-1, (2, n)) if kept is None else kept[r]).requires_grad_()
        dpre, = torch.autograd.grad(torch.nn.functional.silu(z[:, 0]) * z[:, 1], z, dy[r].double())
        want = dpre.flatten(1).to(t).double().T @ x[r].double()
        assert float((got.double() - want).norm()) <= 2 * STEP[dtype] * float(want.norm())
