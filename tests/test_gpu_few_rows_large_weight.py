"""A few rows on MXFP4 weights of 2^29 rows in all, whose planes of scales are 2^31 bytes long: the experts that they go to against the same
product with those experts' weights alone.  Such weights have no Mxfp4Tensor, which ends at 2^35 elements with its padding; the C ABI takes
them."""
import ctypes

import pytest
import torch

import unit_amd as U
from unit_amd import _lib
from unit_amd._lib import check

pytestmark = pytest.mark.gpu
GROUPS, N, K = 1 << 17, 4096, 64  # two blocks a row, one in each plane of scales
ROWS = GROUPS * N
BF16, F32 = 2, 0


@pytest.fixture(scope="module")
def weights(dev):
    """the address of codes and scales of all rows, zeros but for the last 2 N rows; those rows' weight by itself, and its values"""
    need = ROWS * 136 + 1024
    if torch.cuda.mem_get_info()[0] < need + (8 << 30):
        pytest.skip("not enough free memory")
    values = torch.randint(-3, 4, (2 * N, K), generator=torch.Generator().manual_seed(1)).float().to(dev)
    last = U.quantize_mxfp4(values)
    buf = torch.zeros(need, dtype=torch.uint8, device=dev)
    buf[(ROWS - 2 * N) * 128:ROWS * 128] = last.buf[:2 * N * 128]
    buf[ROWS * 128:ROWS * 136].view(2, ROWS, 4)[:, -2 * N:] = last.buf[2 * N * 128:2 * N * 136].view(2, 2 * N, 4)
    yield buf, last, values
    del buf
    torch.cuda.empty_cache()


def operands(rows, dev):
    x = torch.randint(-2, 3, (rows, K), generator=torch.Generator().manual_seed(2)).bfloat16().to(dev)
    need = ctypes.c_size_t()
    check(_lib.load().unit_mxfp4_workspace_bytes(rows, K, ctypes.byref(need)))
    return x, torch.empty(need.value, dtype=torch.uint8, device=dev), torch.full((rows, N), -1.0, device=dev)


@pytest.mark.parametrize("rows", [1, 5])
def test_grouped(dev, weights, rows):
    buf, _, values = weights
    x, ws, out = operands(rows, dev)
    sizes = torch.zeros(GROUPS, dtype=torch.int32, device=dev)
    sizes[-2], sizes[-1] = rows // 2, rows - rows // 2
    check(_lib.load().unit_grouped_dense_mxfp4(x.data_ptr(), None, BF16, buf.data_ptr(), buf.data_ptr() + ROWS * 128, sizes.data_ptr(), 4, out.data_ptr(), F32,
                                               rows, GROUPS, N, K, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    want = torch.cat((x[:rows // 2].double() @ values[:N].double().T, x[rows // 2:].double() @ values[N:].double().T))
    assert torch.equal(out.double(), want)  # small integers: elements, products and sums are exact


@pytest.mark.parametrize("rows", [1, 5])
def test_gated(dev, weights, rows):
    buf, last, _ = weights
    x, ws, out = operands(rows, dev)
    sizes = torch.zeros(GROUPS // 2, dtype=torch.int32, device=dev)
    sizes[-1] = rows
    check(_lib.load().unit_gated_dense_mxfp4(x.data_ptr(), None, BF16, buf.data_ptr(), buf.data_ptr() + ROWS * 128, sizes.data_ptr(), 4, out.data_ptr(), F32, 0,
                                             rows, GROUPS // 2, N, K, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    want = U.gated_dense_mxfp4(x, last)
    assert bool(want.any()) and torch.equal(out, want)  # the sums are exact, and what is made of them is the same
