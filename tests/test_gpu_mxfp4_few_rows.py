"""MXFP4 products of up to 16 rows in floats, the kernel that quantises them in its lanes: values that are not finite stay in their row
or column, also in a last block that the reduction does not fill."""
import pytest
import torch

import unit_amd as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 200, 704), (5, 33, 8), (16, 130, 4096), (3, 64, 1048)])
def test_dense_keeps_nonfinite_values_in_place(dev, m, n, k, dtype):
    g = torch.Generator().manual_seed(m)
    x, w = torch.randn((m, k), generator=g).to(dtype).to(dev), torch.randn((n, k), generator=g).to(dtype).to(dev)
    clean = U.dense_mxfp4(x, U.quantize_mxfp4(w))
    assert U.last_variant().startswith("mxdense_split") and bool(torch.isfinite(clean).all())
    for bad in (float("inf"), float("-inf"), float("nan")):
        xb, wb = x.clone(), w.clone()
        xb[m // 2, k - 1], wb[n - 1, 0] = bad, bad
        got = U.dense_mxfp4(xb, U.quantize_mxfp4(wb))
        lost = torch.zeros((m, n), dtype=torch.bool, device=dev)
        lost[m // 2], lost[:, n - 1] = True, True
        assert torch.equal(got.isnan(), lost) and torch.equal(got[~lost], clean[~lost])


@pytest.mark.parametrize("sizes", [[1, 0, 3], [0, 2, 9], [4, 4, 0]])
def test_experts_keep_nonfinite_values_in_place(dev, sizes):
    g, n, k = torch.Generator().manual_seed(7), 72, 520
    rows = sum(sizes) + 2
    x, w = torch.randn((rows, k), generator=g).bfloat16().to(dev), torch.randn((3, n, k), generator=g).bfloat16().to(dev)
    s = torch.tensor(sizes, device=dev)
    clean = U.grouped_dense_mxfp4(x, U.quantize_mxfp4(w), s)
    assert U.last_variant().startswith("mxdense_split") and bool((clean[-2:] == 0).all())
    x[-2:], x[0, k - 1], w[1, 3, 5] = float("nan"), float("inf"), float("nan")  # rows of no expert, the first row, a column of the second expert
    got = U.grouped_dense_mxfp4(x, U.quantize_mxfp4(w), s)
    lost = torch.zeros((rows, n), dtype=torch.bool, device=dev)
    lost[0] = True
    lost[sizes[0]:sizes[0] + sizes[1], 3] = True
    assert torch.equal(got.isnan(), lost) and torch.equal(got[~lost], clean[~lost])
