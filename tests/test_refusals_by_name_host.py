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


def test_layer_refuses_operands_that_are_no_tensors():
    layer = X.ExpertLayer(torch.zeros(3, 48, 16), torch.zeros(3, 16, 24), 1, "silu")
    quantized = X.ExpertLayer(U.Mxfp4Tensor(CODES, (3, 24, 16)), U.Mxfp4Tensor(CODES, (3, 16, 24)), 1)
    for bad in (U.Mxfp4Tensor(CODES, (5, 16)), U.Mxfp8Tensor(CODES, (5, 16)), [[0.0] * 16], None):
        for one in (layer, quantized):
            with pytest.raises(TypeError, match="x: expected a torch.Tensor, got"):
                one(bad, torch.zeros(5, 3))
            with pytest.raises(TypeError, match="logits: expected a torch.Tensor, got"):
                one(torch.zeros(5, 16), bad)
    for bad in (U.Mxfp8Tensor(CODES, (3, 48, 16)), [1.0], None):
        with pytest.raises(TypeError, match="up: expected a torch.Tensor or an Mxfp4Tensor, got"):
            X.ExpertLayer(bad, torch.zeros(3, 16, 24), 1, "silu")
        with pytest.raises(TypeError, match="down: expected a torch.Tensor or an Mxfp4Tensor, got"):
            X.ExpertLayer(torch.zeros(3, 48, 16), bad, 1, "silu")
    with pytest.raises(TypeError, match="quantized: .*already"):
        quantized.quantized()
