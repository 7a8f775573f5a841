"""The 192-row tile of the grouped products is there to make one round of tiles on the 256 CUs: where it is taken, it does, however the
rows fall on the groups."""
import pytest
import torch

import unit_amd as U
from unit_amd.grouped import _grouped_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes,reduction,columns", [
    ([4835], 3848, 2400),                                # one group: 26 x 10 tiles of 192 rows
    ([420, 400, 193, 390, 250, 300, 385, 385], 3440, 3424),  # 19 row tiles or more, 14 of columns
    ([390] * 16, 1032, 1536),                            # balanced: every group six rows into its third tile, 288 in all
    ([500] * 16, 2048, 1024),                            # 192 tiles
    ([5184], 1024, 2304),                                # 243
])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_one_round(dev, sizes, reduction, columns, dtype):
    rows, e, t, s = sum(sizes), len(sizes), getattr(torch, dtype), torch.tensor(sizes, device=dev)
    x, w, wide = (torch.zeros(*shape, dtype=t, device=dev) for shape in ((rows, reduction), (e, columns, reduction), (rows, columns)))
    tiles = lambda high: sum(-(-n // high) for n in sizes) * -(-columns // 256)
    assert not bool(U.grouped_dense(x, w, s, dtype).any())
    ran = [U.last_variant()]
    assert not bool(_grouped_grad(wide, w.transpose(1, 2).contiguous(), x, s, dtype, dtype, (True, False))[0].any())
    ran.append(U.last_variant())
    for variant in ran:
        assert "_x256_" in variant or ("_x192_" in variant and tiles(192) <= 256), (variant, tiles(192))
        if tiles(192) <= 243:
            assert "_x192_" in variant, variant
