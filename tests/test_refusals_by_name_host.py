"""Operands that are not the tensors an operator takes are refused by their argument's name, before anything looks for a GPU."""
import pytest
import torch

import unit_amd as U
from unit_amd import experts as X

CODES = torch.zeros(20000, dtype=torch.uint8)


@pytest.mark.parametrize("shape", [(4, 64), (2, 2, 64)])
def test_grouped_dense_refuses_rows_in_8_bits(shape):
    """grouped_dense_grad takes them; the forward product does not."""
    w, sizes = torch.zeros((3, 32, 64), dtype=torch.bfloat16), torch.tensor([4, 0, 0])
    with pytest.raises(TypeError, match="data: expected a torch.Tensor, got Mxfp8Tensor"):
        U.grouped_dense(U.Mxfp8Tensor(CODES, shape), w, sizes)
    with pytest.raises(TypeError, match="data: expected a torch.Tensor"):
        U.grouped_dense(U.Mxfp4Tensor(CODES, shape), w, sizes)
