"""Grouped products near the limit of a group's weight, 2^31 - 1 bytes: the fp32 gradient of such a weight is twice as long.  Integer
operands, so sums are exact."""
import pytest
import torch

import unit_amd as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("n,k", [(16392, 32776), (248, 1 << 22)])
def test_weight_gradient_beyond_2_31_bytes(dev, n, k, rows):
    """Columns past 2^29 elements of one weight, and rows of 2^24 bytes, where a tile's offsets come up to 2^32."""
    g = torch.Generator(device=dev).manual_seed(rows)
    ints = lambda *shape: torch.randint(-2, 3, shape, generator=g, device=dev, dtype=torch.int8).to(torch.bfloat16)
    x, dy, sizes = ints(rows + 1, k), ints(rows + 1, n), torch.tensor([rows], device=dev)
    w = torch.zeros((1, n, k), dtype=torch.bfloat16, device=dev)
    for out in ("float32", "bfloat16"):
        _, dw = U.grouped_dense_grad(x, w, dy, sizes, "bfloat16", out)
        assert dw.shape == (1, n, k)
        for c in range(0, k, 4096):
            want = dy[:rows].float().t() @ x[:rows, c:c + 4096].float()
            assert torch.equal(dw[0, :, c:c + 4096].float(), want.to(dw.dtype).float()), (out, c)
        del dw
