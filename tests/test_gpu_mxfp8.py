"""MXFP8 checkpoints on the GPU: every value against the definition in 64 bits.  A power of two and a rounding to three mantissa bits are
exact arithmetic there, so nothing may differ."""
import math

import pytest
import torch

import unit_amd as U

pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
# the 8-bit floats' magnitudes: eight subnormal ones (0 among them), then eight per exponent, 480 not among them
ELEMENTS = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1], dtype=torch.float64)


def values(x):
    """what x's checkpoint stands for, in 64 bits, on the CPU"""
    x = x.cpu().double()
    k = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -k % 32)).unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(torch.where(top > 0, top, torch.ones_like(top)))
    power = (exponent - 9 + (mantissa > 0.875)).clamp(-127, 127)  # 448 = 0.875 * 2^9
    power = torch.where(top > 0, power, torch.full_like(power, -127))
    scale = torch.ldexp(torch.ones_like(top), power)
    a = (b / scale).abs()
    middle = (ELEMENTS[1:] + ELEMENTS[:-1]) / 2
    i = torch.bucketize(a, middle)
    i = i + ((i % 2 == 1) & (a == middle[i.clamp(max=len(middle) - 1)]))  # a tie goes to the even mantissa
    v = torch.copysign(ELEMENTS[i.clamp(max=len(ELEMENTS) - 1)] * scale, b)
    v = torch.where(torch.isfinite(top), v, torch.full_like(v, math.nan))
    return v.flatten(-2)[..., :k]


def same(got, want):
    got = got.cpu().double()
    assert got.shape == want.shape
    assert bool(((got == want) | (got.isnan() & want.isnan())).all()), (got[got != want][:5], want[got != want][:5])


SHAPES = [(1, 1), (1, 32), (1, 33), (3, 31), (7, 64), (33, 257), (2, 5, 40), (1, 4096), (300, 1333), (1031, 96), (5, 2, 1032), (2100, 2085)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES)
def test_there_and_back(dev, shape, dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(shape, generator=g) * torch.exp(3 * torch.randn(shape[:-1] + (1,), generator=g))
    x = (x * (torch.rand(shape, generator=g) > 0.1)).to(TYPES[dtype])
    q = U.quantize_mxfp8(x.to(dev))
    assert q.shape == shape and q.device == dev
    want = values(x)
    same(U.dequantize_mxfp8(q, dtype), want)  # the type that was quantised holds every value
    same(U.dequantize_mxfp8(q), want)
    codes = math.prod(shape[:-1]) * -(-shape[-1] // 32) * 32
    assert q.buf.numel() == codes + codes // 32


def test_storage_is_as_documented(dev):
    x = torch.zeros((2, 40))
    x[0, 0], x[0, 39], x[1, 3] = 448.0, -3.0, 0.5
    b = U.quantize_mxfp8(x.to(dev)).buf.cpu()
    codes, scales = b[:128].view(2, 64), b[128:].view(2, 2)
    # 448 = 1.75 * 2^8, exponent bias 7; -3 is scaled to -384 = -1.5 * 2^8, 0.5 to 256
    assert codes[0, 0] == 0x7e and codes[0, 39] == 0x80 | 0x7c and codes[1, 3] == 0x78 and int((codes != 0).sum()) == 3
    assert scales.tolist() == [[127, 127 - 7], [127 - 9, 0]]


@pytest.mark.parametrize("dtype", TYPES)
def test_every_rounding(dev, dtype):
    """Each element, each middle between two, and the neighbours of both, in one block with 448 and at every scale."""
    t = TYPES[dtype]
    points = torch.cat((ELEMENTS, (ELEMENTS[1:] + ELEMENTS[:-1]) / 2))
    up = torch.nextafter(points.float(), torch.tensor(math.inf)).double()
    down = torch.nextafter(points.float(), torch.tensor(0.0)).double()
    v = torch.cat((points, up, down)).clamp(max=448.0)
    v = torch.cat((v, -v))
    v = torch.nn.functional.pad(v, (0, -len(v) % 31)).view(-1, 31)
    v = torch.cat((torch.full((len(v), 1), 448.0, dtype=torch.float64), v), 1)
    powers = [0, 5, -6] if dtype == "float16" else [0, 60, -60, 119, -118]
    for p in powers:
        x = torch.ldexp(v, torch.tensor(p)).to(t)
        x[:, 0] = torch.ldexp(torch.tensor(448.0), torch.tensor(p)).to(t)
        same(U.dequantize_mxfp8(U.quantize_mxfp8(x.to(dev)), dtype), values(x))


@pytest.mark.parametrize("dtype", TYPES)
def test_largest_magnitudes_choose_the_scale(dev, dtype):
    """Nothing above 448 times the scale: the line between two scales is 1.75 times a power of two."""
    t, eps = TYPES[dtype], torch.finfo(TYPES[dtype]).eps
    tops = torch.tensor([s * m * 2.0 ** p for p in (-14, -3, 0, 9, 15) for s in (1.0, 1.75, 1.75 + 2 * eps, 2 - eps, 1.5) for m in (1.0, -1.0)])
    x = torch.zeros((len(tops), 32), dtype=t)
    x[:, 7], x[:, 30] = tops.to(t), (tops / 1000).to(t)
    same(U.dequantize_mxfp8(U.quantize_mxfp8(x.to(dev)), dtype), values(x).to(t).double())  # float16's largest becomes 2^16: infinite


@pytest.mark.parametrize("dtype", TYPES)
def test_extremes(dev, dtype):
    info = torch.finfo(TYPES[dtype])
    x = torch.zeros((8, 96), dtype=TYPES[dtype])
    x[0, 5], x[0, 40] = info.max, -info.max
    x[1, 1], x[1, 64] = info.smallest_normal, info.smallest_normal * info.eps  # subnormal
    x[2, 3], x[3, 33], x[4, 95] = math.inf, math.nan, -math.inf
    x[5] = info.max
    x[6, ::2] = info.smallest_normal * info.eps * 7
    # the largest finite values are nearest to a power of two that their type does not hold
    same(U.dequantize_mxfp8(U.quantize_mxfp8(x.to(dev)), dtype), values(x).to(TYPES[dtype]).double())


def test_rows_that_begin_anywhere_and_other_strides(dev):
    x = torch.randn(20 * 77 + 1, generator=torch.Generator().manual_seed(2)).to(dev)
    part = x[1:].view(20, 77)
    same(U.dequantize_mxfp8(U.quantize_mxfp8(part)), values(part))
    same(U.dequantize_mxfp8(U.quantize_mxfp8(part.t())), values(part.t()))
    same(U.dequantize_mxfp8(U.quantize_mxfp8(part[::3, 5:50])), values(part[::3, 5:50]))


def test_no_rows(dev):
    q = U.quantize_mxfp8(torch.zeros((0, 70), device=dev))
    assert U.dequantize_mxfp8(q, "bfloat16").shape == (0, 70)


def test_refusals(dev):
    x = torch.zeros((4, 64), device=dev)
    with pytest.raises(TypeError, match="x: expected dtype"):
        U.quantize_mxfp8(x.double())
    with pytest.raises(ValueError, match="two axes or three"):
        U.quantize_mxfp8(x[0])
    with pytest.raises(ValueError, match="GPU"):
        U.quantize_mxfp8(x.cpu())
    with pytest.raises(ValueError, match="positive"):
        U.quantize_mxfp8(x[:, :0])
    q = U.quantize_mxfp8(x)
    with pytest.raises(ValueError, match="out_dtype"):
        U.dequantize_mxfp8(q, "float64")
    with pytest.raises(TypeError, match="Mxfp8Tensor"):
        U.dequantize_mxfp8(x)
    with pytest.raises(ValueError, match="needed"):
        U.dequantize_mxfp8(U.Mxfp8Tensor(q.buf[:100], (4, 64)))
