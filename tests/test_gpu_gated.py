"""Gated feed-forward products on the GPU, forward and gradients, against sums in 64 bits.

Tolerances.  K terms summed in float32 in any order are off by at most K * 2^-23 times the sum of their magnitudes (2^-24 a rounding,
doubled for adders that truncate): d(g), d(u) for the pre-activations.  The sigmoid's argument ζ = z (c1 + c3 z^2) takes four roundings,
its exponential and reciprocal one step each, the sum one: s is off by at most 2^-22 (8 + |ζ|) of itself, and by 2^-126 where it would be
subnormal.  |act'| <= 1.2, |act''| <= 1.  Hence
  h       1.2 d(g) |u| + |act(g)| d(u) + 1.2 d(g) d(u) + |h| 2^-22 (8 + |ζ|), and its rounding: 2^-24, 2^-11, 2^-8 of it
  act'    2^-22 (8 + |ζ|) (s + |z| s |ζ'|): s and z s (1 - s) ζ' with (1 - s) off by as much as s
and the gradients' products like every product, on gate gradients that are off by that and by their rounding to 16 bits."""
import math

import pytest
import torch

import unit_amd as U

pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -126, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -126}  # half of the smallest step
C = math.sqrt(8 / math.pi)


def randn(shape, dtype, seed, dev, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(TYPES[dtype]).to(dev)


def lots(sizes, rows):
    """(group, its rows) as the sizes give them, clamped to what is left; without sizes all of them"""
    if sizes is None:
        yield None, slice(0, rows)
        return
    at = 0
    for g, s in enumerate(sizes):
        n = min(max(s, 0), rows - at)
        yield g, slice(at, at + n)
        at += n


def products(x, w, sizes):
    """x . w^T by group"""
    out = x.new_zeros((x.shape[0], w.shape[-2]))
    for g, r in lots(sizes, x.shape[0]):
        out[r] = x[r] @ (w if g is None else w[g]).T
    return out


def activation(z, act):
    """act(z), act'(z), and the relative error that its sigmoid may have"""
    zeta = z if act == "silu" else C * (z + 0.044715 * z ** 3)
    rise = torch.ones_like(z) if act == "silu" else C * (1 + 3 * 0.044715 * z ** 2)
    s = torch.sigmoid(zeta)
    rel = 2.0 ** -22 * (8 + zeta.abs())
    return z * s, s + z * s * torch.sigmoid(-zeta) * rise, rel, rel * (s + z.abs() * s * rise) + 2.0 ** -126


def forward(x, w, sizes, act):
    """h, pre (rows, 2, N) and how far either may be off before it is rounded"""
    n, k = w.shape[-2] // 2, w.shape[-1]
    pre = products(x.double(), w.double(), sizes).unflatten(-1, (2, n))
    off = k * 2.0 ** -23 * products(x.double().abs(), w.double().abs(), sizes).unflatten(-1, (2, n))
    (g, u), (dg, du) = pre.unbind(1), off.unbind(1)
    a, _, rel, _ = activation(g, act)
    h = a * u
    return h, 1.2 * dg * u.abs() + a.abs() * du + 1.2 * dg * du + h.abs() * rel + u.abs() * 2.0 ** -126, pre, off


def gradients(x, w, dy, sizes, act, pre, pre_off, dtype):
    """ddata, dweight and how far either may be off before it is rounded"""
    n, k = w.shape[-2] // 2, w.shape[-1]
    x, w, dy = x.double(), w.double(), dy.double()
    (g, u), (og, ou) = pre.unbind(1), pre_off.unbind(1)
    a, slope, rel, slope_off = activation(g, act)
    dpre = torch.cat((dy * u * slope, dy * a), 1)
    off = torch.cat((dy.abs() * (u.abs() * (slope_off + og) + ou * (slope.abs() + slope_off + og)), dy.abs() * (a.abs() * rel + 1.2 * og)), 1)
    off = off + 3 * 2.0 ** -24 * dpre.abs()  # two products in float32
    off = off + ROUND[dtype] * (dpre.abs() + off) + TINY[dtype]
    dx, dxo, dw, dwo = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(w)
    for e, r in lots(sizes, x.shape[0]):
        we = w if e is None else w[e]
        dx[r], dxo[r] = dpre[r] @ we, off[r] @ we.abs() + 2 * n * 2.0 ** -23 * (dpre[r].abs() + off[r]) @ we.abs()
        part, part_off = dpre[r].T @ x[r], off[r].T @ x[r].abs() + (r.stop - r.start) * 2.0 ** -23 * (dpre[r].abs() + off[r]).T @ x[r].abs()
        if e is None:
            dw, dwo = part, part_off
        else:
            dw[e], dwo[e] = part, part_off
    return dx, dxo, dw, dwo


def near(got, want, off, out):
    assert got.dtype == TYPES[out] and got.shape == want.shape
    err, bound = (got.double() - want).abs(), off * (1 + ROUND[out]) + ROUND[out] * want.abs() + TINY[out]
    assert bool((err <= bound).all()), (float((err - bound).max()), float(err.max()), int((err > bound).sum()))


CASES = [  # group sizes (None: one weight), rows beside them, N, K
    (None, 1, 8, 8),
    (None, 1, 64, 256),
    (None, 5, 200, 520),
    (None, 16, 1032, 328),
    (None, 17, 136, 72),
    (None, 65, 72, 1032),
    (None, 333, 264, 136),
    (None, 700, 776, 512),
    (None, 2000, 1032, 264),
    ([1], 0, 8, 8),
    ([0, 1, 0], 0, 64, 64),
    ([3, 0, 0, 5], 2, 72, 40),
    ([0, 0, 0], 7, 64, 128),
    ([1] * 40, 0, 136, 264),
    ([16, 17, 15, 1, 32, 33], 3, 200, 512),
    ([100, 1, 28], 0, 520, 776),
    ([129, 0, 127, 65], 0, 392, 520),
    ([513, 3, 0, 700], 40, 520, 248),
    ([5, 0, 9] * 30, 11, 96, 192),     # more groups than a wave has lanes
    ([0] * 300 + [70] + [0] * 50 + [1], 0, 64, 72),
    ([0] * 70 + [3] + [0] * 80 + [9, 1] + [0] * 20, 3, 72, 200),  # the same of at most 16 rows
]


def operands(case, dtype, dev):
    sizes, spare, n, k = case
    rows = spare + sum(sizes or [])
    lead = () if sizes is None else (len(sizes),)
    x, w = randn((rows, k), dtype, 1, dev), randn(lead + (2 * n, k), dtype, 2, dev, 1.5 * k ** -0.5)
    return x, w, randn((rows, n), dtype, 3, dev, 2.0 ** -5), None if sizes is None else torch.tensor(sizes, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype,out,act", [("float16", "float32", "silu"), ("bfloat16", "bfloat16", "gelu_tanh"), ("float16", "float16", "gelu_tanh"),
                                           ("bfloat16", "float32", "silu")])
def test_forward(dev, case, dtype, out, act):
    sizes = CASES[case][0]
    x, w, _, s = operands(CASES[case], dtype, dev)
    h, off, pre, pre_off = forward(x, w, sizes, act)
    got = U.gated_dense(x, w, s, act, out)
    near(got, h, off, out)
    long = None if s is None else s.long()
    again, kept = U.gated_dense(x, w, long, act, out, keep="pre")
    assert torch.equal(got, again)  # the same bits, whatever is kept
    near(kept, pre, pre_off, dtype)
    again, kept = U.gated_dense(x, w, s, act, out, keep="mxfp8")
    assert torch.equal(got, again) and kept.shape == pre.shape
    n = pre.shape[-1]
    top = torch.nn.functional.pad(pre.abs() + pre_off, (0, -n % 32)).unflatten(-1, (-1, 32)).amax(-1)
    mantissa, exponent = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(top), exponent - 9 + (mantissa > 0.875)).repeat_interleave(32, -1)[..., :n]
    err = (U.dequantize_mxfp8(kept).double() - pre).abs()
    assert bool((err <= pre_off + torch.maximum(2.0 ** -4 * (pre.abs() + pre_off), 2.0 ** -10 * scale)).all())


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype,out,wout,act", [("float16", "float32", "float32", "gelu_tanh"), ("bfloat16", "bfloat16", "float32", "silu"),
                                                ("float16", "float16", "float16", "silu"), ("bfloat16", "float32", "bfloat16", "gelu_tanh")])
def test_gradients(dev, case, dtype, out, wout, act):
    sizes = CASES[case][0]
    x, w, dy, s = operands(CASES[case], dtype, dev)
    _, _, exact, sums_off = forward(x, w, sizes, act)
    _, kept = U.gated_dense(x, w, s, act, keep="pre")

    def check(got, x, pre, off):
        dx, dxo, dw, dwo = gradients(x, w, dy, sizes, act, pre, off, dtype)
        near(got[0], dx, dxo, out)
        near(got[1], dw, dwo, wout)

    args = dict(activation=act, out_dtype=out, weight_out_dtype=wout)
    got = U.gated_dense_grad(x, w, dy, s, pre=kept, **args)
    check(got, x, kept.double(), torch.zeros_like(exact))
    for a, b in zip(got, U.gated_dense_grad(x, w, dy, None if s is None else s.long(), pre=kept, **args)):
        assert torch.equal(a, b)
    # from the rows alone: pre-activations may be rounded to 16 bits on the way
    check(U.gated_dense_grad(x, w, dy, s, **args), x, exact, sums_off + ROUND[dtype] * (exact.abs() + sums_off) + TINY[dtype])
    # both kept in 8 bits: exact functions of what the checkpoints stand for
    x8, kept8 = U.quantize_mxfp8(x), U.quantize_mxfp8(kept)
    check(U.gated_dense_grad(x8, w, dy, s, pre=kept8, **args), U.dequantize_mxfp8(x8), U.dequantize_mxfp8(kept8).double(), torch.zeros_like(exact))
    # the rows alone, in 8 bits
    x8v = U.dequantize_mxfp8(x8)
    _, _, exact8, off8 = forward(x8v, w, sizes, act)
    check(U.gated_dense_grad(x8, w, dy, s, **args), x8v, exact8, off8 + ROUND[dtype] * (exact8.abs() + off8) + TINY[dtype])


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_gradients_are_the_differences_of_the_forward(dev, act):
    """Central differences of the kernels' own forward in float32 results.  A step of 2^-4 in one element of the gate's or the up projection's
    row changes one pre-activation of a row by 2^-4 x; the third derivative, at most 2, leaves h^2 / 6 of it, the sums K * 2^-22 of their
    magnitudes over the step."""
    n, k, rows, step = 16, 24, 9, 2.0 ** -4
    x, w, dy = randn((rows, k), "float16", 5, dev, 0.5), randn((2 * n, k), "float16", 6, dev, 0.25), torch.ones((rows, n), dtype=torch.float16, device=dev)
    w = (w * 16).round() / 16  # steps of 2^-4 are exact
    x = (x * 16).round() / 16
    dx, dw = U.gated_dense_grad(x, w, dy, activation=act)
    loss = lambda x, w: float(U.gated_dense(x, w, activation=act).double().sum())
    for t, d, places in ((w, dw, [(0, 0), (7, 23), (15, 4), (16, 0), (31, 11), (20, 9)]), (x, dx, [(0, 0), (8, 23), (4, 10)])):
        for at in places:
            plus, minus = t.clone(), t.clone()
            plus[at] += step
            minus[at] -= step
            f = (lambda v: loss(x, v)) if t is w else (lambda v: loss(v, w))
            num = (f(plus) - f(minus)) / (2 * step)
            assert abs(num - float(d[at])) <= 0.02 * (1 + abs(num)), (at, num, float(d[at]))


def test_large_tiles(dev):
    """Tiles of the largest sizes, ragged on every side, where the rules take them; against 64 bits as above."""
    for sizes, rows, n, k in ((None, 4100, 1544, 776), ([1500, 0, 700, 1801], 4006, 1032, 520), ([256] * 12 + [9], 3081, 1280, 1032), ([500, 700, 300] * 5, 7500, 1024, 1024)):
        x, w = randn((rows, k), "bfloat16", 7, dev), randn((() if sizes is None else (len(sizes),)) + (2 * n, k), "bfloat16", 8, dev, k ** -0.5)
        s = None if sizes is None else torch.tensor(sizes, device=dev)
        h, off, pre, pre_off = forward(x, w, sizes, "silu")
        got, kept = U.gated_dense(x, w, s, "silu", "bfloat16", keep="pre")
        near(got, h, off, "bfloat16")
        near(kept, pre, pre_off, "bfloat16")
        assert torch.equal(got, U.gated_dense(x, w, s, "silu", "bfloat16")) and torch.equal(got, U.gated_dense(x, w, s, "silu", "bfloat16", keep="mxfp8")[0])


@pytest.mark.parametrize("tile", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("keep", [None, "pre", "mxfp8"])
def test_every_tile(dev, tile, keep, monkeypatch):
    """Each tile on problems that end inside it, whichever the rule would take."""
    monkeypatch.setenv("UNIT_AMD_GATED_TILE", str(tile))
    monkeypatch.setenv("UNIT_AMD_GATED_MOST", "255" if keep == "pre" else "160" if keep else "0")
    for sizes, rows, n, k in ((None, 40, 72, 136), ([70, 0, 300, 33], 410, 328, 200), ([256, 417, 160, 673, 161, 512, 0, 1], 2200, 136, 72), (None, 930, 200, 64)):
        x, w = randn((rows, k), "float16", 9, dev), randn((() if sizes is None else (len(sizes),)) + (2 * n, k), "float16", 10, dev, k ** -0.5)
        s = None if sizes is None else torch.tensor(sizes, device=dev)
        h, off, pre, pre_off = forward(x, w, sizes, "gelu_tanh")
        got = U.gated_dense(x, w, s, "gelu_tanh", "float32", keep=keep)
        near(got if keep is None else got[0], h, off, "float32")
        if keep == "pre":
            near(got[1], pre, pre_off, "float16")
        if keep == "mxfp8":
            near(U.dequantize_mxfp8(got[1]).half(), pre, pre_off + 2.0 ** -4 * pre.abs() + 2.0 ** -17 * pre.abs().amax(), "float16")


@pytest.mark.parametrize("sizes", [None, [5, 9, 3], [40, 0, 30], [300, 200, 129]])
def test_nonfinite_values_stay_in_their_rows_and_groups(dev, sizes):
    n, k = 72, 136
    spare = 6 if sizes else 20
    x, w, dy, s = operands((sizes, spare, n, k), "bfloat16", dev)
    bad = sum(sizes[:2]) if sizes else 7
    x[bad, 3], dy[bad, 5] = float("inf"), float("nan")
    if sizes:
        x[-6:], dy[-6:] = float("nan"), float("inf")  # rows of no expert
    good = torch.ones(len(x), dtype=torch.bool, device=dev)
    good[bad] = False
    for keep in ("pre", "mxfp8"):
        y, pre = U.gated_dense(x, w, s, keep=keep)
        assert bool(torch.isfinite(y[good]).all()) and not bool(torch.isfinite(y[bad]).any())
        values = U.dequantize_mxfp8(pre) if keep == "mxfp8" else pre
        assert bool(torch.isfinite(values[good]).all()) and not bool(torch.isfinite(values[bad]).any())
        if sizes:
            assert not bool(y[-6:].any()) and not bool(values[-6:].any())
        for kept in (pre, None):
            dx, dw = U.gated_dense_grad(x, w, dy, s, pre=kept)
            assert bool(torch.isfinite(dx[good]).all()) and bool(torch.isnan(dx[bad]).all())
            if sizes:
                assert not bool(dx[-6:].any()) and bool(torch.isfinite(dw[:2]).all()) and bool(torch.isnan(dw[2]).any())


@pytest.mark.parametrize("tile", [1, 2, 3, 4])
def test_every_mxfp4_tile(dev, tile, monkeypatch):
    monkeypatch.setenv("UNIT_AMD_GROUPED_TILE", str(tile))
    for sizes, rows, n, k in ((None, 40, 72, 136), ([70, 0, 300, 33], 410, 333, 600)):
        x, w = randn((rows, k), "float16", 9, dev), U.quantize_mxfp4(randn((() if sizes is None else (len(sizes),)) + (2 * n, k), "float16", 10, dev, k ** -0.5))
        s = None if sizes is None else torch.tensor(sizes, device=dev)
        h, off, _, _ = forward(U.dequantize_mxfp4(U.quantize_mxfp4(x)), U.dequantize_mxfp4(w), sizes, "gelu_tanh")
        near(U.gated_dense_mxfp4(x, w, s, "gelu_tanh"), h, off, "float32")


@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_far_pre_activations(dev, act):
    """Pre-activations from -1e30 to 1e30: the sigmoid is 0 or 1, the gradients are those of 0 and of the identity."""
    n = k = 8
    z = torch.tensor([-1e30, -1e18, -3e4, -200.0, 200.0, 3e4, 1e18, 1e30], dtype=torch.bfloat16)
    x = torch.eye(8, dtype=torch.bfloat16, device=dev)
    w = torch.cat((torch.diag(z), torch.ones((8, 8), dtype=torch.bfloat16))).to(dev)
    h, pre = U.gated_dense(x, w, activation=act, keep="pre")
    want = torch.diag(torch.where(z > 0, z.double(), torch.zeros(8, dtype=torch.float64))).to(dev)
    near(h, want, 2.0 ** -20 * want.abs(), "float32")
    dy = torch.ones((8, n), dtype=torch.bfloat16, device=dev)
    for p in (pre, None):
        dx, dw = U.gated_dense_grad(x, w, dy, activation=act, pre=p)
        assert bool(torch.isfinite(dw).all()) and bool(torch.isfinite(dx).all())
        diagonal = dw[:8].diagonal().double().cpu()
        assert torch.equal(diagonal, (z > 0).double())
        near(dw[8:].diagonal(), want.diagonal(), 2.0 ** -8 * want.diagonal().abs(), "float32")


def test_no_rows(dev):
    for s, lead in ((None, ()), (torch.zeros(3, dtype=torch.int32, device=dev), (3,))):
        x, w = torch.zeros((0, 64), dtype=torch.float16, device=dev), torch.ones(lead + (80, 64), dtype=torch.float16, device=dev)
        dy = torch.zeros((0, 40), dtype=torch.float16, device=dev)
        for keep in ("pre", "mxfp8"):
            y, pre = U.gated_dense(x, w, s, keep=keep)
            assert y.shape == (0, 40) and pre.shape == (0, 2, 40)
            for p in (pre, None):
                dx, dw = U.gated_dense_grad(x, w, dy, s, pre=p)
                assert dx.shape == (0, 64) and dw.shape == w.shape and not bool(dw.any())
        dx, dw = U.gated_dense_grad(U.quantize_mxfp8(x), w, dy, s, pre=pre)
        assert dw.shape == w.shape and not bool(dw.any())


MX_CASES = [  # group sizes, spare rows, N, K
    (None, 1, 64, 256), (None, 1, 3, 33), (None, 7, 130, 1000), (None, 33, 1000, 512), (None, 300, 77, 264), (None, 1500, 640, 520), (None, 2100, 1030, 300),
    ([0, 1, 0], 0, 64, 64), ([3, 0, 0, 5], 2, 70, 45), ([1] * 40, 0, 136, 264), ([100, 1, 28], 0, 333, 776), ([513, 3, 0, 700], 40, 520, 248), ([5, 0, 9] * 30, 11, 96, 192),
]


@pytest.mark.parametrize("case", range(len(MX_CASES)))
@pytest.mark.parametrize("dtype,out,act", [("float32", "float32", "silu"), ("bfloat16", "bfloat16", "gelu_tanh"), ("float16", "float16", "silu"), ("bfloat16", "float32", "gelu_tanh")])
def test_mxfp4(dev, case, dtype, out, act):
    sizes, spare, n, k = MX_CASES[case]
    rows = spare + sum(sizes or [])
    x, w = randn((rows, k), dtype, 1, dev), U.quantize_mxfp4(randn((() if sizes is None else (len(sizes),)) + (2 * n, k), "bfloat16", 2, dev, 1.5 * k ** -0.5))
    s = None if sizes is None else torch.tensor(sizes, device=dev)
    q = U.quantize_mxfp4(x)
    h, off, _, _ = forward(U.dequantize_mxfp4(q), U.dequantize_mxfp4(w), sizes, act)
    got = U.gated_dense_mxfp4(x, w, s, act, out)
    near(got, h, off, out)
    near(U.gated_dense_mxfp4(q, w, s, act, out), h, off, out)


def test_refusals(dev):
    x, w, dy = (torch.zeros(s, dtype=torch.float16, device=dev) for s in ((4, 64), (80, 64), (4, 40)))
    s = torch.tensor([2, 2], device=dev)
    for call, error, text in (
        (lambda: U.gated_dense(x, w, activation="relu"), ValueError, "activation"),
        (lambda: U.gated_dense(x, w, out_dtype="int8"), ValueError, "out_dtype"),
        (lambda: U.gated_dense(x, w, out_dtype="bfloat16"), ValueError, "out_dtype"),
        (lambda: U.gated_dense(x, w, keep="8"), ValueError, "keep"),
        (lambda: U.gated_dense(x, w, s), ValueError, "weight: expected 3-D"),
        (lambda: U.gated_dense(x, w[None]), ValueError, "weight: expected 2-D"),
        (lambda: U.gated_dense(x, torch.stack((w, w, w)), s), ValueError, "group_sizes: expected 3 entries"),
        (lambda: U.gated_dense(x, w[:79]), ValueError, "as many rows"),
        (lambda: U.gated_dense(x, w[:, :56]), ValueError, "data: expected"),
        (lambda: U.gated_dense(x, w.bfloat16()), TypeError, "weight: expected dtype"),
        (lambda: U.gated_dense(x.float(), w), TypeError, "data: expected dtype"),
        (lambda: U.gated_dense(x, w[:20]), ValueError, "multiples of 8"),
        (lambda: U.gated_dense(x.cpu(), w), ValueError, "GPU"),
        (lambda: U.gated_dense(x, w.cpu()), ValueError, "GPU"),
        (lambda: U.gated_dense(U.quantize_mxfp8(x), w), TypeError, "Mxfp8Tensor"),
        (lambda: U.gated_dense(x.flatten()[4:68].view(1, 64), w), ValueError, "aligned"),
        (lambda: U.gated_dense_grad(x, w, dy[:, :32]), ValueError, "grad: expected"),
        (lambda: U.gated_dense_grad(x, w, dy.bfloat16()), TypeError, "grad: expected dtype"),
        (lambda: U.gated_dense_grad(x, w, dy, pre=torch.zeros((4, 80), dtype=torch.float16, device=dev)), ValueError, "pre: expected 3-D"),
        (lambda: U.gated_dense_grad(x, w, dy, pre=torch.zeros((4, 2, 32), dtype=torch.float16, device=dev)), ValueError, "pre: expected"),
        (lambda: U.gated_dense_grad(x, w, dy, pre=torch.zeros((4, 2, 40), device=dev)), TypeError, "pre: expected dtype"),
        (lambda: U.gated_dense_grad(x, w, dy, weight_out_dtype="bfloat16"), ValueError, "out_dtype"),
        (lambda: U.gated_dense_grad(U.quantize_mxfp8(x[:3]), w, dy), ValueError, "grad: expected"),
        (lambda: U.gated_dense_mxfp4(x, w), TypeError, "Mxfp4Tensor"),
        (lambda: U.gated_dense_mxfp4(x, U.quantize_mxfp4(w[:79])), ValueError, "as many rows"),
        (lambda: U.gated_dense_mxfp4(x[:, :50], U.quantize_mxfp4(w)), ValueError, "data: expected"),
        (lambda: U.gated_dense_mxfp4(x, U.quantize_mxfp4(w), s), ValueError, "weight: expected 3 axes"),
    ):
        with pytest.raises(error, match=text):
            call()


@pytest.mark.parametrize("most", [1, 128, 255])
def test_tiles_of_two_sizes_over_many_groups(dev, most, monkeypatch):
    """More groups than a wave has lanes, with remainders of every kind: none, one row, the limit and one more, all but one row of a tile."""
    monkeypatch.setenv("UNIT_AMD_GATED_TILE", "8")
    monkeypatch.setenv("UNIT_AMD_GATED_MOST", str(most))
    sizes = [256, 0, 257, most, most + 1, 255, 512 + most, 1, 0, 31] * 7 + [700]
    rows, n, k = sum(sizes) + 9, 136, 72
    x, w = randn((rows, k), "bfloat16", 11, dev), randn((len(sizes), 2 * n, k), "bfloat16", 12, dev, k ** -0.5)
    h, off, pre, pre_off = forward(x, w, sizes, "silu")
    got, kept = U.gated_dense(x, w, torch.tensor(sizes, device=dev), "silu", "bfloat16", keep="pre")
    near(got, h, off, "bfloat16")
    near(kept, pre, pre_off, "bfloat16")


@pytest.mark.parametrize("tile", [1, 2, 3, 4, 5, 6, 7, 8])
def test_gradients_on_every_tile(dev, tile, monkeypatch):
    monkeypatch.setenv("UNIT_AMD_GATED_TILE", str(tile))
    monkeypatch.setenv("UNIT_AMD_GROUPED_TILE", str(min(tile, 5)))
    for case in ((None, 40, 72, 136), ([70, 0, 300, 33], 7, 328, 200)):
        x, w, dy, s = operands(case, "float16", dev)
        _, _, exact, off = forward(x, w, case[0], "silu")
        got = U.gated_dense_grad(x, w, dy, s, "silu")
        dx, dxo, dw, dwo = gradients(x, w, dy, case[0], "silu", exact, off + ROUND["float16"] * (exact.abs() + off) + TINY["float16"], "float16")
        near(got[0], dx, dxo, "float32")
        near(got[1], dw, dwo, "float32")


@pytest.mark.parametrize("rows,sizes", [(3, None), (70, [20, 0, 45])])
def test_the_python_path_gives_the_native_calls_results(dev, rows, sizes, monkeypatch):
    from unit_amd import gated as G, grouped
    x, w, dy, s = operands((sizes, rows - sum(sizes or []), 72, 136), "bfloat16", dev)

    def everything():
        wq = U.quantize_mxfp4(w)
        h, pre = U.gated_dense(x, w, s, "gelu_tanh", "bfloat16", keep="pre")
        _, pre8 = U.gated_dense(x, w, s, "gelu_tanh", "bfloat16", keep="mxfp8")
        x8 = U.quantize_mxfp8(x)
        out = [h, pre, U.dequantize_mxfp8(pre8), U.dequantize_mxfp8(x8, "bfloat16"), U.gated_dense(x, w, s), U.gated_dense_mxfp4(x, wq, s, "silu", "float16"),
               U.gated_dense_mxfp4(U.quantize_mxfp4(x), wq, s)]
        for data, kept in ((x, pre), (x, None), (x8, pre8), (x8, None)):
            out += U.gated_dense_grad(data, w, dy, s, "gelu_tanh", kept, "bfloat16", "float32")
        return out

    native = everything()
    calls = []

    class Declines:
        def __getattr__(self, name):
            return lambda *a: calls.append(name)

    monkeypatch.setattr(G, "_native_gated", Declines())
    monkeypatch.setattr(grouped, "_native_gated", Declines())
    for a, b in zip(native, everything()):
        assert a.dtype == b.dtype and torch.equal(a, b)
    assert set(calls) == {"quantize8", "dequantize8", "gated", "gated_mx", "gated_grad"}


def test_the_common_case_is_native(dev):
    """Each native call takes the operands that a user's program has, rather than leave them to the Python operator."""
    from unit_amd.grouped import _native_gated as native
    x, w, dy, _ = operands((None, 6, 72, 136), "float16", dev)
    h, pre8 = native.gated(x, w, None, "silu", "float16", "mxfp8")
    assert h.shape == (6, 72) and pre8.shape == (6, 2, 72)
    assert native.gated(x, w, None, "silu", "float32", None) is not None and native.gated(x, w, None, "silu", "float32", "pre") is not None
    x8 = native.quantize8(x)
    assert native.dequantize8(x8, "float16").shape == x.shape
    assert native.gated_mx(x, U.quantize_mxfp4(w), None, "silu", "float16").shape == (6, 72)
    for data, pre in ((x, None), (x8, None), (x, pre8), (x8, pre8)):
        assert native.gated_grad(data, w, dy, None, "silu", pre, "float16", "float32") is not None
    assert native.gated(x, w, None, "relu", "float16", None) is None and native.gated(x.float(), w, None, "silu", "float16", None) is None


@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("splits", [1, 2, 4, 16])
def test_gradients_in_one_launch(dev, tiles, splits, monkeypatch):
    """Each form of the launch, rows shared out or not, either product first, ragged on every side; with the tiles of groups beside it."""
    monkeypatch.setenv("UNIT_AMD_GATED_PAIR", str(tiles))
    monkeypatch.setenv("UNIT_AMD_GATED_SPLITS", str(splits))
    cases = [(None, 1100, 72, 136), (None, 130, 264, 328), (None, 2087, 24, 72)]
    for case in cases + ([([70, 0, 300, 33], 7, 136, 200), ([900, 0, 1], 0, 40, 264)] if splits == 1 else []):
        for dtype, out in (("bfloat16", "bfloat16"), ("float16", "float32")):
            x, w, dy, s = operands(case, dtype, dev)
            _, kept = U.gated_dense(x, w, s, "silu", keep="pre")
            got = U.gated_dense_grad(x, w, dy, s, "silu", kept, out, out)
            dx, dxo, dw, dwo = gradients(x, w, dy, case[0], "silu", kept.double(), torch.zeros_like(kept, dtype=torch.float64), dtype)
            near(got[0], dx, dxo, out)
            near(got[1], dw, dwo, out)
            for a, b in zip(got, U.gated_dense_grad(x, w, dy, s, "silu", kept, out, out)):
                assert torch.equal(a, b)


def test_gradients_of_many_rows_and_a_small_weight(dev):
    """Where the rows are shared out by the rule itself, with the other operand frozen too."""
    from unit_amd.gated import _gated_grad
    x, w, dy, _ = operands((None, 9001, 136, 72), "bfloat16", dev)
    _, kept = U.gated_dense(x, w, keep="pre")
    dx, dxo, dw, dwo = gradients(x, w, dy, None, "silu", kept.double(), torch.zeros_like(kept, dtype=torch.float64), "bfloat16")
    got = U.gated_dense_grad(x, w, dy, pre=kept)
    near(got[0], dx, dxo, "float32")
    near(got[1], dw, dwo, "float32")
    for wanted in ((True, False), (False, True)):
        one = _gated_grad(x, w, dy, None, "silu", kept, "float32", "float32", wanted)
        for have, t, want, off in zip(wanted, one, (dx, dw), (dxo, dwo)):
            assert (t is not None) == have
            if have:
                near(t, want, off, "float32")
