"""The large tiles of the grouped and MXFP4 products, in every type that they are built for: as the rule picks them (each test says which
kernel that is), and the 192-row and 256-row ones pinned on small and odd sizes.  Tolerances as in test_gpu_grouped.py."""
import pytest
import torch

import unit_amd as U
from test_gpu_grouped import CASES, backward, forward, near, operands
from unit_amd.grouped import _grouped_grad

pytestmark = pytest.mark.gpu

TYPES = [("float16", "float32"), ("float16", "float16"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")]
SHORT = {"float16": "f16", "bfloat16": "bf16"}
ONE_ROUND = [2100, 0, 1500, 1200, 900]   # 224 tiles of 192 x 256 at most for 1544 columns
SEVERAL = [2900, 1, 2400, 0, 2600]       # 301


def data(sizes, spare, n, k, dtype, dev):
    """as test_gpu_grouped.operands, made on the GPU"""
    g, rows, t = torch.Generator(device=dev).manual_seed(n + k), sum(sizes) + spare, getattr(torch, dtype)
    r = lambda *s: torch.randn(s, generator=g, device=dev)
    return r(rows, k).to(t), (r(len(sizes), n, k) * k ** -0.5).to(t), (r(rows, n) * 2.0 ** -5).to(t), torch.tensor(sizes, device=dev)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("sizes,k,rows", [(ONE_ROUND, 520, 192), (SEVERAL, 1032, 256)])
def test_forward(dev, sizes, k, rows, dtype, out):
    x, w, _, s = data(sizes, 5, 1544, k, dtype, dev)
    got = U.grouped_dense(x, w, s, out)
    assert U.last_variant() == f"{SHORT[dtype]}grouped_x{rows}_y256_k128_r2"
    x, w = x.double(), w.double()
    near(got, forward(x, w, sizes), forward(x.abs(), w.abs(), sizes), k, out)


@pytest.mark.parametrize("dtype,out", TYPES)
@pytest.mark.parametrize("sizes,n,rows", [(ONE_ROUND, 520, 192), (SEVERAL, 1032, 256)])
def test_data_gradient(dev, sizes, n, rows, dtype, out):
    x, w, dy, s = data(sizes, 5, n, 1544, dtype, dev)
    got, none = _grouped_grad(x, w, dy, s, out, out, (True, False))
    assert none is None and U.last_variant() == f"{SHORT[dtype]}groupeddx_x{rows}_y256_k128_r2"
    want, size = (backward(*(f(t.double()) for t in (x, w, dy)), sizes)[0] for f in (lambda t: t, torch.abs))
    near(got, want, size, n, out)


@pytest.mark.parametrize("dtype,out", TYPES)
def test_weight_gradient(dev, dtype, out):
    x, w, dy, s = data(SEVERAL, 5, 1544, 1032, dtype, dev)
    none, got = _grouped_grad(x, w, dy, s, out, out, (False, True))
    assert none is None and U.last_variant() == f"{SHORT[dtype]}groupeddw_x256_y256_k128_r2"
    want, size = (backward(*(f(t.double()) for t in (x, w, dy)), SEVERAL)[1] for f in (lambda t: t, torch.abs))
    near(got, want, size, max(SEVERAL), out)


@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
def test_mxfp4(dev, out):
    for sizes, n, k in (([3100], 2900, 1100), ([1500, 0, 1700, 1801], 2500, 1064)):
        x, w, _, s = data(sizes, 0, n, k, "bfloat16", dev)
        wq = U.quantize_mxfp4(w[0] if len(sizes) == 1 else w)
        got = U.dense_mxfp4(x, wq, out) if len(sizes) == 1 else U.grouped_dense_mxfp4(x, wq, s, out)
        assert U.last_variant() == "mxdense_x256_y256_k128_r2"
        xd, wd = U.dequantize_mxfp4(U.quantize_mxfp4(x)).double(), U.dequantize_mxfp4(wq).double().view(len(sizes), n, k)
        near(got, forward(xd, wd, sizes), forward(xd.abs(), wd.abs(), sizes), k, out)


@pytest.mark.parametrize("tile", [4, 5])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_pinned_on_any_sizes(dev, case, tile, monkeypatch):
    monkeypatch.setenv("UNIT_AMD_GROUPED_TILE", str(tile))
    sizes, spare, n, k = CASES[case]
    for dtype, out in TYPES:
        x, w, dy, s = operands(sizes, spare, n, k, dtype, dev)
        xd, wd, dyd = x.double(), w.double(), dy.double()
        got = U.grouped_dense(x, w, s, out)
        assert f"_x{192 if tile == 5 else 256}_" in U.last_variant()
        near(got, forward(xd, wd, sizes), forward(xd.abs(), wd.abs(), sizes), k, out)
        got, want, size = U.grouped_dense_grad(x, w, dy, s, out, out), backward(xd, wd, dyd, sizes), backward(xd.abs(), wd.abs(), dyd.abs(), sizes)
        near(got[0], want[0], size[0], n, out)
        near(got[1], want[1], size[1], max(sizes), out)
    q, wq = U.quantize_mxfp4(x), U.quantize_mxfp4(w)
    xd, wd = U.dequantize_mxfp4(q).double(), U.dequantize_mxfp4(wq).double()
    for out in ("float16", "bfloat16"):
        near(U.grouped_dense_mxfp4(q, wq, s, out), forward(xd, wd, sizes), forward(xd.abs(), wd.abs(), sizes), k, out)
