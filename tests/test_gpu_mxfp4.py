"""MXFP4 on the GPU: quantisation and its inverse bit for bit against a table-driven definition in 64 bits, products against
64-bit sums of the stored values.

Tolerance of a product: K terms summed in float32 in any order are off by at most K * 2^-23 times the sum of their magnitudes (2^-24
a rounding, doubled for adders that truncate), and the result is rounded once: 2^-24, 2^-11 or 2^-8 of it (float16: 2^-25 below its
normal range)."""
import pytest
import torch

import unit_amd as U

pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def encode(x):
    """(..., K) -> (codes 0..15 (..., K), scales (..., blocks)) by the definition, on the CPU in 64 bits."""
    x = x.cpu().double()
    k = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -k % 32)).unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    _, e = torch.frexp(top)
    s = torch.where(top > 0, (e.long() - 1 - 2 + 127).clamp(0, 254), 0)
    s = torch.where(torch.isfinite(top), s, 255)
    a = (b / torch.pow(2.0, torch.where(s == 255, 127, s).double() - 127).unsqueeze(-1)).abs()
    d = (a.unsqueeze(-1) - VALUES).abs()
    tied = d == d.amin(-1, keepdim=True)  # the nearest one or two
    even = tied & (torch.arange(8) % 2 == 0)
    pick = torch.where(even.any(-1), even.int().argmax(-1), tied.int().argmax(-1))
    codes = pick + 8 * torch.signbit(b).long()
    return codes.flatten(-2)[..., :k], s


def decode(codes, scales):
    v = VALUES[codes % 8] * torch.where(codes < 8, 1.0, -1.0)
    p = torch.where(scales == 255, torch.nan, torch.pow(2.0, scales.double() - 127))
    return v * p.repeat_interleave(32, -1)[..., :codes.shape[-1]]


def stored(codes, scales):
    """codes, scales -> a checkpoint's bytes"""
    c = torch.nn.functional.pad(codes, (0, -codes.shape[-1] % 32)).unflatten(-1, (-1, 2))
    return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8), scales.to(torch.uint8)


def data(shape, dtype, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.pow(2.0, torch.randint(-6, 7, (*shape[:-1], 1), generator=g).float())
    return x.to(TYPES[dtype]).to(dev)


def same(got, want):
    assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=1e300), torch.nan_to_num(want, nan=1e300))


def near(got, x, w, out):
    """got against x . w^T, both float64 on the CPU"""
    want, size = x @ w.T, x.abs() @ w.abs().T
    bound = x.shape[1] * 2.0 ** -23 * size + ROUND[out] * want.abs() + (2.0 ** -25 if out == "float16" else 0.0)
    err = (got.cpu().double() - want).abs()
    assert got.dtype == TYPES[out] and tuple(got.shape) == tuple(want.shape)
    assert bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 255), (4, 256), (7, 257), (2, 3, 520), (33, 1333), (300, 2048), (1, 16384)])
def test_quantise_matches_the_definition(dev, dtype, shape):
    x = data(shape, dtype, 1 + shape[-1], dev)
    q = U.quantize_mxfp4(x)
    assert q.shape == shape
    want = decode(*encode(x))
    same(U.dequantize_mxfp4(q), want)
    same(U.dequantize_mxfp4(q, "bfloat16"), want)  # an element and a power of two fit a bfloat16
    same(U.dequantize_mxfp4(q, "float16"), want.to(torch.float16).double())


@pytest.mark.parametrize("dtype", TYPES)
def test_quantise_ties_extremes_and_nonfinite_blocks(dev, dtype):
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2, 0.3, 1.2, 1.3, 5.5, 6.0, 7.0, 7.9, 0.0, -0.0]
    rows = []
    for scale in (1.0, 2.0 ** -3, 2.0 ** 9):
        for top in (4.0, 6.0, 7.75):  # the block's largest magnitude stays in [4, 8) times its scale
            r = [top] + ties + [-v for v in ties]
            rows.append([v * scale for v in (r + [0.0] * 64)[:64]])
    rows.append([0.0] * 64)
    tiny, huge = torch.finfo(TYPES[dtype]).smallest_normal, torch.finfo(TYPES[dtype]).max
    rows.append([tiny, -tiny, tiny / 2, 0.0] * 16)
    rows.append([huge, -huge, huge / 4, 0.0] * 16)
    for bad in (float("nan"), float("inf"), float("-inf")):
        rows.append([1.0] * 5 + [bad] + [2.0] * 26 + [3.0] * 32)  # the first block is lost, the second is not
    x = torch.tensor(rows, dtype=torch.float64).to(TYPES[dtype]).to(dev)
    got = U.dequantize_mxfp4(U.quantize_mxfp4(x))
    want = decode(*encode(x))
    assert bool(torch.isnan(want[-3:, :32]).all()) and bool(torch.isfinite(want[-3:, 32:]).all())
    same(got, want)


def test_quantise_takes_views_and_any_alignment(dev):
    x = data((9, 70), "bfloat16", 3, dev)
    for v in (x[:, 1:], x[1:, :33], x.t(), x[::2], x[3:4, 5:]):
        same(U.dequantize_mxfp4(U.quantize_mxfp4(v)), decode(*encode(v)))
    flat = data((1, 641), "float32", 4, dev).view(-1)[1:].view(10, 64)  # contiguous, 4 bytes off
    assert flat.is_contiguous() and flat.data_ptr() % 16 == 4
    same(U.dequantize_mxfp4(U.quantize_mxfp4(flat)), decode(*encode(flat)))


@pytest.mark.parametrize("shape", [(1, 5), (3, 64), (2, 70, 300), (130, 1024)])
def test_prepared_weight_is_the_checkpoint(dev, shape):
    g = torch.Generator().manual_seed(7)
    codes = torch.randint(0, 16, shape, generator=g)
    scales = torch.randint(0, 256, (*shape[:-1], -(-shape[-1] // 32)), generator=g)  # 255: NaN
    scales = torch.where(scales == 254, 100, scales)
    c, s = stored(codes, scales)
    junk = c.clone()
    if shape[-1] % 32:
        junk[..., (shape[-1] + 1) // 2:] = 0x7f  # codes behind K are dropped
    q = U.prepare_mxfp4_weight(junk.to(dev), s.to(dev), shape[-1])
    same(U.dequantize_mxfp4(q), decode(codes, scales).float().double())  # 4 and 6 times 2^126 round to infinity


PRODUCTS = [(1, 1, 1), (1, 16, 33), (2, 40, 256), (5, 33, 300), (16, 64, 512), (17, 130, 2088), (31, 257, 96), (64, 64, 64), (65, 100, 1000),
            (128, 512, 768), (129, 255, 513), (200, 700, 320), (256, 256, 4096), (300, 1516, 256), (1000, 520, 776), (1, 4096, 4096), (3, 2049, 3000)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype,out", [("bfloat16", "bfloat16"), ("float16", "float32"), ("float32", "float16")])
def test_dense_matches_64_bit_sums(dev, m, n, k, dtype, out):
    x, w = data((m, k), dtype, m + n, dev), data((n, k), "float32", k, dev)
    x *= 2.0 ** -4
    xd, wd = decode(*encode(x)), decode(*encode(w))
    wq = U.quantize_mxfp4(w)
    got = U.dense_mxfp4(x, wq, out)
    near(got, xd, wd, out)
    assert torch.equal(got, U.dense_mxfp4(U.quantize_mxfp4(x), wq, out))  # quantised on the way or before: the same bits


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("m", [1, 16, 17, 130])
def test_dense_of_unaligned_rows(dev, m, dtype):
    """Contiguous rows that begin one element into their memory: the products of the same values, one row or several."""
    k, n = 712, 200
    x, w = data((m, k), dtype, m, dev), data((n, k), "float32", 7, dev)
    wq = U.quantize_mxfp4(w)
    off = torch.cat((x.new_zeros(1), x.view(-1)))[1:].view(m, k)
    assert off.data_ptr() % 16 == x.element_size()
    near(U.dense_mxfp4(off, wq, "float32"), decode(*encode(x)), decode(*encode(w)), "float32")


def test_dense_large_tiles(dev):
    """Several hundred rows and columns of tiles, uneven on every side; the sums in 64 bits on the GPU."""
    for m, n, k in ((2100, 2300, 1100), (4096, 1024, 2048), (700, 6000, 288)):
        x, w = data((m, k), "bfloat16", m, dev), data((n, k), "bfloat16", n, dev)
        q, wq = U.quantize_mxfp4(x), U.quantize_mxfp4(w)
        xd, wd = U.dequantize_mxfp4(q).double(), U.dequantize_mxfp4(wq).double()
        got = U.dense_mxfp4(x, wq)
        err, bound = (got.double() - xd @ wd.T).abs(), (k * 2.0 ** -23 + 2.0 ** -24) * (xd.abs() @ wd.abs().T)
        assert bool((err <= bound).all()), (m, n, k)


@pytest.mark.parametrize("m", [1, 40, 300])
def test_dense_keeps_nan_in_its_row_and_column(dev, m):
    k, n = 700, 200
    x, w = data((m, k), "bfloat16", 5, dev), data((n, k), "bfloat16", 6, dev)
    x[m // 2, 650] = float("inf")
    w[77, 10] = float("nan")
    got = U.dense_mxfp4(x, U.quantize_mxfp4(w)).isnan().cpu()
    want = torch.zeros((m, n), dtype=torch.bool)
    want[m // 2], want[:, 77] = True, True
    assert torch.equal(got, want)


def test_dense_without_rows(dev):
    w = U.quantize_mxfp4(data((40, 64), "bfloat16", 1, dev))
    assert U.dense_mxfp4(torch.empty((0, 64), dtype=torch.bfloat16, device=dev), w).shape == (0, 40)
    q = U.quantize_mxfp4(torch.empty((0, 64), device=dev))
    assert U.dequantize_mxfp4(q).shape == (0, 64) and U.dense_mxfp4(q, w).shape == (0, 40)


def test_refusals(dev):
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device=dev)
    w = U.quantize_mxfp4(torch.zeros((8, 64), device=dev))
    with pytest.raises(ValueError, match="GPU"):
        U.quantize_mxfp4(torch.zeros((4, 64)))
    with pytest.raises(TypeError, match="dtype"):
        U.quantize_mxfp4(torch.zeros((4, 64), dtype=torch.float64, device=dev))
    with pytest.raises(ValueError, match="two axes or three"):
        U.quantize_mxfp4(torch.zeros((64,), device=dev))
    with pytest.raises(ValueError, match="K must be positive"):
        U.quantize_mxfp4(torch.zeros((4, 0), device=dev))
    with pytest.raises(ValueError, match="out_dtype"):
        U.dequantize_mxfp4(w, "int8")
    with pytest.raises(TypeError, match="Mxfp4Tensor"):
        U.dense_mxfp4(x, x)
    with pytest.raises(ValueError, match="rows, 64"):
        U.dense_mxfp4(x[:, :32], w)
    with pytest.raises(ValueError, match="2 axes"):
        U.dense_mxfp4(x, U.quantize_mxfp4(torch.zeros((2, 8, 64), device=dev)))
    with pytest.raises(TypeError, match="dtype"):
        U.dense_mxfp4(x.to(torch.int32), w)
    with pytest.raises(ValueError, match="out_dtype"):
        U.dense_mxfp4(x, w, "int32")
    c, s = torch.zeros((8, 32), dtype=torch.uint8, device=dev), torch.zeros((8, 2), dtype=torch.uint8, device=dev)
    assert U.prepare_mxfp4_weight(c, s).shape == (8, 64)
    for bad in ((c, s[:, :1]), (c[:4], s), (c, s, 32), (c, s, 65)):
        with pytest.raises(ValueError):
            U.prepare_mxfp4_weight(*bad)
    with pytest.raises(TypeError):
        U.prepare_mxfp4_weight(c, s.to(torch.int8))
