"""Products grouped by expert on the GPU, forward and gradients, against sums in 64 bits.

Tolerance: K terms summed in float32 in any order are off by at most K * 2^-23 times the sum of their magnitudes (2^-24 a rounding,
doubled for adders that truncate), and the result is rounded once: 2^-24, 2^-11 or 2^-8 of it (float16: 2^-25 below its normal range).
Integer-valued operands are exact."""
import pytest
import torch

import unit_amd as U

pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
ROUND = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def randn(shape, dtype, seed, dev, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(TYPES[dtype]).to(dev)


def groups(sizes, rows):
    """(group, its rows) as the sizes give them, clamped to what is left"""
    at = 0
    for g, s in enumerate(sizes):
        n = min(max(s, 0), rows - at)
        yield g, slice(at, at + n)
        at += n


def forward(x, w, sizes):
    out = x.new_zeros((x.shape[0], w.shape[1]))
    for g, r in groups(sizes, x.shape[0]):
        out[r] = x[r] @ w[g].T
    return out


def backward(x, w, dy, sizes):
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for g, r in groups(sizes, x.shape[0]):
        dx[r], dw[g] = dy[r] @ w[g], dy[r].T @ x[r]
    return dx, dw


def near(got, want, size, terms, out):
    bound = terms * 2.0 ** -23 * size + ROUND[out] * want.abs() + (2.0 ** -25 if out == "float16" else 0.0)
    err = (got.double() - want).abs()
    assert got.dtype == TYPES[out] and got.shape == want.shape
    assert bool((err <= bound).all()), (float((err - bound).max()), float(err.max()))


CASES = [  # group sizes, spare rows, N, K
    ([1], 0, 8, 8),
    ([0, 1, 0], 0, 64, 64),
    ([3, 0, 0, 5], 2, 72, 40),
    ([0, 0, 0], 7, 64, 128),
    ([1] * 40, 0, 136, 264),
    ([16, 17, 15, 1, 32, 33], 3, 200, 512),
    ([64], 0, 256, 1024),
    ([100, 1, 28], 0, 520, 776),
    ([128, 128], 1, 128, 96),
    ([129, 0, 127, 65], 0, 776, 520),
    ([255, 257, 300], 0, 264, 328),
    ([513, 3, 0, 700], 40, 1032, 248),
    ([2000], 0, 512, 256),
    ([5, 0, 9] * 30, 11, 96, 192),     # more groups than a wave has lanes
    ([0] * 300 + [70] + [0] * 50 + [1], 0, 64, 72),
]


def operands(sizes, spare, n, k, dtype, dev):
    rows = sum(sizes) + spare
    x, w = randn((rows, k), dtype, 1, dev), randn((len(sizes), n, k), dtype, 2, dev, k ** -0.5)
    return x, w, randn((rows, n), dtype, 3, dev, 2.0 ** -5), torch.tensor(sizes, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype,out", [("float16", "float32"), ("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float32")])
def test_forward(dev, case, dtype, out):
    sizes, spare, n, k = CASES[case]
    x, w, _, s = operands(sizes, spare, n, k, dtype, dev)
    got = U.grouped_dense(x, w, s, out)
    near(got, forward(x.double(), w.double(), sizes), forward(x.double().abs(), w.double().abs(), sizes), k, out)
    assert torch.equal(got, U.grouped_dense(x, w, s.long(), out))  # 8-byte sizes, and the same bits again


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype,out,wout", [("float16", "float32", "float32"), ("bfloat16", "bfloat16", "float32"), ("float16", "float16", "float16"),
                                            ("bfloat16", "float32", "bfloat16")])
def test_gradients(dev, case, dtype, out, wout):
    sizes, spare, n, k = CASES[case]
    x, w, dy, s = operands(sizes, spare, n, k, dtype, dev)
    got = U.grouped_dense_grad(x, w, dy, s, out, wout)
    want = backward(x.double(), w.double(), dy.double(), sizes)
    size = backward(x.double().abs(), w.double().abs(), dy.double().abs(), sizes)
    near(got[0], want[0], size[0], n, out)
    near(got[1], want[1], size[1], max(sizes), wout)
    again = U.grouped_dense_grad(x, w, dy, s.long(), out, wout)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_gradients_are_the_differences_of_the_forward(dev, dtype):
    """The product is linear in either operand: with integers every sum is exact, and so is the difference."""
    g = torch.Generator().manual_seed(5)
    sizes, rows, n, k = [3, 0, 20, 1], 26, 24, 40
    s = torch.tensor(sizes, dtype=torch.int64, device=dev)
    ints = lambda *shape: torch.randint(-3, 4, shape, generator=g).to(TYPES[dtype]).to(dev)
    x, w, dy = ints(rows, k), ints(4, n, k), ints(rows, n)
    loss = lambda x, w: float((U.grouped_dense(x, w, s).double() * dy.double()).sum())
    dx, dw = U.grouped_dense_grad(x, w, dy, s)
    at = loss(x, w)
    for r, c in ((0, 0), (2, 39), (3, 7), (22, 20), (23, 1), (25, 5)):  # the last two rows belong to no expert
        moved = x.clone()
        moved[r, c] += 1
        assert loss(moved, w) - at == float(dx[r, c])
    for e, r, c in ((0, 0, 0), (1, 3, 3), (2, 23, 39), (3, 11, 20)):
        moved = w.clone()
        moved[e, r, c] += 1
        assert loss(x, moved) - at == float(dw[e, r, c])
    assert bool((dx[24:] == 0).all()) and bool((dw[1] == 0).all())


def test_large_groups(dev):
    """Tiles of the largest size, ragged on every side, both directions; integer operands, so sums are exact."""
    g = torch.Generator(device=dev).manual_seed(9)
    for sizes, n, k in (([1500, 0, 700, 1801], 1544, 776), ([4000], 2048, 1032), ([300] * 12 + [9], 2056, 520), ([2100, 0, 1500, 1200, 900], 1544, 520)):
        rows = sum(sizes) + 5
        ints = lambda *shape: torch.randint(-2, 3, shape, generator=g, device=dev).to(torch.bfloat16)
        x, w, dy, s = ints(rows, k), ints(len(sizes), n, k), ints(rows, n), torch.tensor(sizes, device=dev)
        assert torch.equal(U.grouped_dense(x, w, s).double(), forward(x.double(), w.double(), sizes))
        for got, want in zip(U.grouped_dense_grad(x, w, dy, s), backward(x.double(), w.double(), dy.double(), sizes)):
            assert torch.equal(got.double(), want)


@pytest.mark.parametrize("sizes", [[5, 9, 3], [40, 0, 30], [300, 200, 129]])
def test_nonfinite_values_stay_in_their_rows_and_groups(dev, sizes):
    n, k = 72, 136
    x, w, dy, s = operands(sizes, 6, n, k, "bfloat16", dev)
    last = sum(sizes[:2])  # the first row of the last group
    x[last, 3], dy[last, 5] = float("inf"), float("nan")
    x[-6:], dy[-6:] = float("nan"), float("inf")  # rows of no expert
    y = U.grouped_dense(x, w, s)
    assert bool(torch.isfinite(y[:last]).all()) and bool(torch.isfinite(y[last + 1:]).all()) and not bool(torch.isfinite(y[last]).any())
    dx, dw = U.grouped_dense_grad(x, w, dy, s)
    assert bool(torch.isfinite(dx[:last]).all()) and bool(torch.isfinite(dx[last + 1:]).all()) and bool(torch.isnan(dx[last]).all())
    assert bool((dx[-6:] == 0).all()) and bool((y[-6:] == 0).all())
    assert bool(torch.isfinite(dw[:2]).all())
    bad = torch.zeros((n, k), dtype=torch.bool, device=dev)
    bad[5], bad[:, 3] = True, True
    assert torch.equal(~torch.isfinite(dw[2]), bad)
    w[0] = float("nan")  # another group's weight
    y, (dx, _) = U.grouped_dense(x, w, s), U.grouped_dense_grad(x, w, dy, s)
    r = slice(sizes[0], last)
    assert bool(torch.isfinite(y[r]).all()) and bool(torch.isfinite(dx[r]).all())


@pytest.mark.parametrize("sizes", [[-5, 4, 100, 2], [2 ** 31 - 1, 2 ** 31 - 1, 3, -2 ** 31], [0, 0, 0, 0], [7, 3, 0, 2 ** 31 - 1]])
def test_sizes_of_any_value_stay_in_bounds(dev, sizes):
    x, w, dy, _ = operands([10, 5, 3, 2], 0, 64, 72, "float16", dev)
    for dt in (torch.int32, torch.int64):
        s = torch.tensor(sizes, dtype=torch.int64).to(dt).to(dev)
        y, (dx, dw) = U.grouped_dense(x, w, s), U.grouped_dense_grad(x, w, dy, s)
        near(y, forward(x.double(), w.double(), sizes), forward(x.double().abs(), w.double().abs(), sizes), 72, "float32")
        want, size = (backward(*(f(t.double()) for t in (x, w, dy)), sizes) for f in (lambda t: t, torch.abs))
        near(dx, want[0], size[0], 64, "float32")
        near(dw, want[1], size[1], 20, "float32")
    wide = torch.tensor([2 ** 40, -2 ** 40, 1, 1], device=dev)  # 8-byte sizes beyond 32 bits
    assert torch.equal(U.grouped_dense(x, w, wide), U.grouped_dense(x, w, torch.tensor([20, 0, 0, 0], device=dev)))


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("dtype,out", [("bfloat16", "bfloat16"), ("float16", "float32")])
def test_mxfp4(dev, case, dtype, out):
    sizes, spare, n, k = CASES[case]
    n, k = n - 3, k + 5  # any number of columns and elements
    x, w, _, s = operands(sizes, spare, n, k, dtype, dev)
    wq = U.quantize_mxfp4(w)
    xd, wd = U.dequantize_mxfp4(U.quantize_mxfp4(x)).double(), U.dequantize_mxfp4(wq).double()
    got = U.grouped_dense_mxfp4(x, wq, s, out)
    near(got, forward(xd, wd, sizes), forward(xd.abs(), wd.abs(), sizes), k, out)
    assert torch.equal(got, U.grouped_dense_mxfp4(U.quantize_mxfp4(x), wq, s.long(), out))


def test_mxfp4_large_groups_and_nan(dev):
    g = torch.Generator(device=dev).manual_seed(11)
    sizes, n, k = [1500, 0, 700, 1801], 1500, 1000
    x = torch.randn((sum(sizes) + 9, k), generator=g, device=dev).half()
    w = torch.randn((4, n, k), generator=g, device=dev).half()
    x[-9:] = float("nan")
    x[10, 5] = float("inf")
    wq, s = U.quantize_mxfp4(w), torch.tensor(sizes, device=dev)
    got = U.grouped_dense_mxfp4(x, wq, s)
    assert bool((got[-9:] == 0).all()) and bool(got[10].isnan().all())
    xd, wd = U.dequantize_mxfp4(U.quantize_mxfp4(x)).double(), U.dequantize_mxfp4(wq).double()
    keep = torch.ones(len(x), dtype=torch.bool, device=dev)
    keep[10] = False
    near(got[keep], forward(xd, wd, sizes)[keep], forward(xd.abs(), wd.abs(), sizes)[keep], k, "float32")


@pytest.mark.parametrize("tile", [1, 2, 3, 4])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_every_tile_on_every_case(dev, case, tile, monkeypatch):
    """The tile is a matter of speed: each of the four gives the right result whatever the sizes."""
    monkeypatch.setenv("UNIT_AMD_GROUPED_TILE", str(tile))
    sizes, spare, n, k = CASES[case]
    x, w, dy, s = operands(sizes, spare, n, k, "bfloat16", dev)
    xd, wd, dyd = x.double(), w.double(), dy.double()
    near(U.grouped_dense(x, w, s), forward(xd, wd, sizes), forward(xd.abs(), wd.abs(), sizes), k, "float32")
    got, want, size = U.grouped_dense_grad(x, w, dy, s), backward(xd, wd, dyd, sizes), backward(xd.abs(), wd.abs(), dyd.abs(), sizes)
    near(got[0], want[0], size[0], n, "float32")
    near(got[1], want[1], size[1], max(sizes), "float32")
    q, wq = U.quantize_mxfp4(x), U.quantize_mxfp4(w)
    xd, wd = U.dequantize_mxfp4(q).double(), U.dequantize_mxfp4(wq).double()
    near(U.grouped_dense_mxfp4(q, wq, s), forward(xd, wd, sizes), forward(xd.abs(), wd.abs(), sizes), k, "float32")


def test_rows_of_more_than_2_31_bytes(dev):
    """2.2 GB of rows: the groups on either side of the 2^31-byte line, and the last rows; forward, both gradients."""
    n, k, rows = 64, 4096, 270_000
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randint(-2, 3, (rows, k), generator=g, device=dev, dtype=torch.int8).to(torch.bfloat16)
    w = torch.randint(-2, 3, (3, n, k), generator=g, device=dev).to(torch.bfloat16)
    dy = torch.randint(-2, 3, (rows, n), generator=g, device=dev).to(torch.bfloat16)
    sizes = [262_100, 60, 7_800]  # the line is row 262144
    s = torch.tensor(sizes, device=dev)
    y, (dx, dw) = U.grouped_dense(x, w, s), U.grouped_dense_grad(x, w, dy, s, "bfloat16")
    for e, r in ((0, slice(0, 64)), (0, slice(262_000, 262_100)), (1, slice(262_100, 262_160)), (2, slice(262_160, 262_400)), (2, slice(269_900, 269_960))):
        assert torch.equal(y[r].double(), x[r].double() @ w[e].double().T)
        assert torch.equal(dx[r].double(), (dy[r].double() @ w[e].double()).to(torch.bfloat16).double())
    assert bool((y[269_960:] == 0).all()) and bool((dx[269_960:] == 0).all())
    for e, r in ((1, slice(262_100, 262_160)), (2, slice(262_160, 269_960))):
        assert torch.equal(dw[e].double(), dy[r].double().T @ x[r].double())


def test_quantised_weights_of_more_than_2_31_bytes(dev):
    """A stack of 2.3 GB of codes: the first and the last experts, as prepared and as multiplied."""
    e, n, k = 70, 8192, 8192
    g = torch.Generator(device=dev).manual_seed(3)
    codes = torch.randint(0, 256, (e, n, k // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = torch.randint(120, 124, (e, n, k // 32), generator=g, device=dev, dtype=torch.uint8)
    w = U.prepare_mxfp4_weight(codes, scales)
    sizes = [2] + [0] * (e - 3) + [3, 40]
    x = torch.randn((45, k), generator=g, device=dev).to(torch.bfloat16)
    got = U.grouped_dense_mxfp4(x, w, torch.tensor(sizes, device=dev))
    xd = U.dequantize_mxfp4(U.quantize_mxfp4(x)).double()
    for i, r in ((0, slice(0, 2)), (e - 2, slice(2, 5)), (e - 1, slice(5, 45))):
        wd = U.dequantize_mxfp4(U.prepare_mxfp4_weight(codes[i], scales[i])).double()
        near(got[r], xd[r] @ wd.T, xd[r].abs() @ wd.abs().T, k, "float32")


def test_no_rows(dev):
    w, s = randn((3, 16, 32), "float16", 1, dev), torch.zeros(3, dtype=torch.int32, device=dev)
    x, dy = torch.empty((0, 32), dtype=torch.float16, device=dev), torch.empty((0, 16), dtype=torch.float16, device=dev)
    assert U.grouped_dense(x, w, s).shape == (0, 16)
    dx, dw = U.grouped_dense_grad(x, w, dy, s)
    assert dx.shape == (0, 32) and bool((dw == 0).all())
    assert U.grouped_dense_mxfp4(x, U.quantize_mxfp4(w), s).shape == (0, 16)


def test_views_are_taken_as_they_read(dev):
    sizes = [5, 12]
    x, w, dy, s = operands(sizes, 0, 64, 48, "float16", dev)
    want, grads = U.grouped_dense(x, w, s), U.grouped_dense_grad(x, w, dy, s)
    xt, wt, dyt = x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), dy.repeat_interleave(2, 0)[::2]
    st = torch.stack((s, s), 1)[:, 0]
    assert not (xt.is_contiguous() or wt.is_contiguous() or dyt.is_contiguous() or st.is_contiguous())
    assert torch.equal(U.grouped_dense(xt, wt, st), want)
    assert all(torch.equal(a, b) for a, b in zip(U.grouped_dense_grad(xt, wt, dyt, st), grads))
    big = randn((17, 8), "float16", 4, dev)
    assert torch.equal(U.grouped_dense(torch.cat((x[:1], x))[1:], w, s), want) and big is not None


def test_other_streams_and_graph_replays(dev):
    """On a stream of its own, and captured: sizes are read when the work runs, so a replay follows what they hold by then."""
    x, w, dy, s = operands([70, 0, 200, 30], 4, 264, 136, "bfloat16", dev)
    wq = U.quantize_mxfp4(w)
    run = lambda: (U.grouped_dense(x, w, s), *U.grouped_dense_grad(x, w, dy, s), U.grouped_dense_mxfp4(x, wq, s), U.dense_mxfp4(x, U.quantize_mxfp4(w[1])))
    eager = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for sizes in ([70, 0, 200, 30], [0, 300, 0, 0], [70, 0, 200, 30], [1, 2, 3, 4]):
        s.copy_(torch.tensor(sizes, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, run()):
            assert torch.equal(a, b), sizes


def test_refusals(dev):
    x, w, dy, s = operands([5, 12], 0, 64, 48, "float16", dev)
    with pytest.raises(ValueError, match="GPU"):
        U.grouped_dense(x.cpu(), w, s)
    with pytest.raises(ValueError, match="GPU"):
        U.grouped_dense(x, w, s.cpu())
    with pytest.raises(TypeError, match="dtype"):
        U.grouped_dense(x.float(), w, s)
    with pytest.raises(TypeError, match="dtype"):
        U.grouped_dense(x, w.bfloat16(), s)
    with pytest.raises(TypeError, match="int32 or torch.int64"):
        U.grouped_dense(x, w, s.float())
    with pytest.raises(ValueError, match="rows, 48"):
        U.grouped_dense(x[:, :40], w, s)
    with pytest.raises(ValueError, match="2 entries"):
        U.grouped_dense(x, w, s[:1])
    with pytest.raises(ValueError, match="out_dtype"):
        U.grouped_dense(x, w, s, torch.float16)
    with pytest.raises(ValueError, match="multiples of 8"):
        U.grouped_dense(x[:, :44], w[..., :44], s)
    with pytest.raises(ValueError, match="multiples of 8"):
        U.grouped_dense(x, w[:, :60], s)
    with pytest.raises(ValueError, match="must be positive"):
        U.grouped_dense(x, w[:0], s[:0])
    with pytest.raises(ValueError, match="aligned"):
        U.grouped_dense(torch.zeros(17 * 48 + 1, dtype=torch.float16, device=dev)[1:].view(17, 48), w, s)
    with pytest.raises(ValueError, match="17, 64"):
        U.grouped_dense_grad(x, w, dy[:16], s)
    with pytest.raises(ValueError, match="weight_out_dtype"):
        U.grouped_dense_grad(x, w, dy, s, weight_out_dtype="int8")
    with pytest.raises(TypeError, match="Mxfp4Tensor"):
        U.grouped_dense_mxfp4(x, w, s)
    with pytest.raises(ValueError, match="3 axes"):
        U.grouped_dense_mxfp4(x, U.quantize_mxfp4(w[0]), s)
