"""Products of expert layers and of microscaled 4-bit operands, as cases that can be timed and compared.

Operators (`case["op"]`):

  quantize     rows -> MXFP4: blocks of 32 along a row share a power of two, elements are 4-bit floats (2 exponent bits,
               1 mantissa bit); what is returned are the values that the codes stand for
  dense        y = q(x) . W^T, x a matrix of floats that is quantised on the way, W (N, K) in MXFP4
  experts      y[r] = W[e(r)] x[r], rows sorted by expert, as many rows per expert as its entry of group_sizes says
  experts_grad the gradients of the same product: dx[r] = W[e(r)]^T dy[r], dW[e] = sum over the rows of e of dy[r] x[r]^T
  experts_q    the product of `experts` on rows quantised on the way and weights in MXFP4

`own` says who computes: false, elementary torch operations in 32 bits; true, the package's operators.
listed() names twelve cases, draw(rng) takes further ones of the same ranges.
"""
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
BLOCK = 32           # elements that share a scale
MAX_FLOPS = 2.8e11   # the largest listed product
MAX_BYTES = 3.5e8    # operands and results of the largest drawn case


def listed():
    return [
        # the activations of one token in front of a quantised layer: the smallest call
        dict(name="quantize_token", op="quantize", rows=1, k=4096, dtype="bfloat16"),
        # a weight from a training run, single precision, rows that end inside a block and inside a cache line
        dict(name="quantize_ragged", op="quantize", rows=1003, k=1333, dtype="float32"),
        # the activations of a long prompt
        dict(name="quantize_prompt", op="quantize", rows=8192, k=4096, dtype="bfloat16"),
        # one token through a quantised layer: the weight is read once
        dict(name="dense_token", op="dense", rows=1, n=4096, k=4096, dtype="bfloat16", out="bfloat16"),
        # a handful of requests, nothing aligned to a tile, a reduction that ends inside a block
        dict(name="dense_ragged", op="dense", rows=333, n=1516, k=2088, dtype="float16", out="float32"),
        # a prompt through a quantised layer: the largest product
        dict(name="dense_prompt", op="dense", rows=8192, n=4096, k=4096, dtype="bfloat16", out="bfloat16"),
        # eight requests, two experts each, one new token: most experts get one row or none
        dict(name="experts_token", op="experts", rows=16, experts=16, skew=0.5, spare=0, n=2048, k=1024, dtype="float16",
             out="float16", route=1),
        # a training batch, popular and unpopular experts, a buffer whose last rows belong to no expert
        dict(name="experts_batch", op="experts", rows=16384, experts=32, skew=0.5, spare=200, n=2048, k=1024,
             dtype="bfloat16", out="bfloat16", route=2),
        # gradients of a small fine-tuning batch, ragged in every size, half precision, sums kept in single
        dict(name="experts_grad_ragged", op="experts_grad", rows=1000, experts=12, skew=0.7, spare=0, n=776, k=520,
             dtype="float16", out="float32", weight_out="float32", route=3),
        # gradients of a training batch: rows in 16 bits, weights in 32 for the optimiser
        dict(name="experts_grad_batch", op="experts_grad", rows=8192, experts=16, skew=0.5, spare=0, n=2048, k=1024,
             dtype="bfloat16", out="bfloat16", weight_out="float32", route=4),
        # thirty-two requests, two experts each, one new token, on quantised experts
        dict(name="experts_q_token", op="experts_q", rows=64, experts=64, skew=0.5, spare=0, n=2048, k=2048,
             dtype="bfloat16", out="bfloat16", route=5),
        # prompts on quantised experts
        dict(name="experts_q_prompt", op="experts_q", rows=16384, experts=64, skew=0.5, spare=0, n=2048, k=2048,
             dtype="bfloat16", out="bfloat16", route=6),
    ]


# ------------------------------------------------------------------------------------- drawn cases
def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_one(rng):
    op = rng.choice(["quantize", "dense", "experts", "experts_grad", "experts_q"])
    step = rng.choice([8, 8, 64])  # rows of 16-bit weights are whole 16-byte pieces; half of the cases are ragged beyond that
    case = dict(op=op, rows=_log_int(rng, 1, 16384))
    if op == "quantize":
        return dict(case, k=_log_int(rng, 1, 8192), dtype=rng.choice(["float32", "float16", "bfloat16"]))
    n, k = step * _log_int(rng, 64 // step, 4096 // step), step * _log_int(rng, 64 // step, 4096 // step)
    if op in ("dense", "experts_q") and rng.random() < 0.4:
        n, k = _log_int(rng, 1, 4096), _log_int(rng, 33, 4096)
    dtype = rng.choice(["float16", "bfloat16"])
    case.update(n=n, k=k, dtype=dtype, out=rng.choice(["float32", dtype]))
    if op == "dense":
        return case
    case.update(experts=_log_int(rng, 1, 128), skew=rng.choice([0.0, 0.5, 1.0]), route=rng.randrange(1 << 30),
                spare=rng.choice([0, 0, case["rows"] // 10]))
    if op == "experts_grad":
        case["weight_out"] = rng.choice(["float32", dtype])
    return case


def draw(rng):
    while True:
        case = _draw_one(rng)
        w = work(case)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return case


# ------------------------------------------------------------------------------------- inputs and state
def _sizes(case, seed):
    """Rows of each expert: how many is the case's, which expert gets them the seed's."""
    r = random.Random(case["route"])
    e = case["experts"]
    chosen = r.choices(range(e), [(i + 1.0) ** -case["skew"] for i in range(e)], k=case["rows"] - case["spare"])
    sizes = torch.bincount(torch.tensor(chosen, dtype=torch.int64), minlength=e).tolist()
    random.Random(seed).shuffle(sizes)
    return sizes


def _rows(rows, k, dtype, g, scale=1.0):
    """Activations: about one channel in fifty is eight times as large as the others, one row in forty is all zeros."""
    x = torch.randn((rows, k), device="cuda", generator=g) * scale
    x *= 1.0 + 7.0 * (torch.rand((k,), device="cuda", generator=g) < 0.02)
    x *= (torch.rand((rows, 1), device="cuda", generator=g) >= 0.025) | (rows < 40)
    return x.to(DTYPES[dtype])


def _weights(shape, dtype, g):
    return (torch.randn(shape, device="cuda", generator=g) / math.sqrt(shape[-1])).to(DTYPES[dtype])


def _inputs(case, seed):
    g, op = torch.Generator(device="cuda").manual_seed(seed), case["op"]
    rows, k, dtype = case["rows"], case["k"], case["dtype"]
    x = dict(x=_rows(rows, k, dtype, g))
    if op == "quantize":
        return x
    if op == "dense":
        return dict(x, w=_encode(_weights((case["n"], k), "bfloat16", g)))
    sizes = _sizes(case, seed)
    x.update(sizes=torch.tensor(sizes, dtype=torch.int32, device="cuda"), most=max(sizes))
    if op == "experts_q":
        return dict(x, w=_encode(_weights((case["experts"], case["n"], k), "bfloat16", g)))
    x["w"] = _weights((case["experts"], case["n"], k), dtype, g)
    if op == "experts_grad":
        x["dy"] = _rows(rows, case["n"], dtype, g, 2.0 ** -7)
    return x


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own and case["op"] in ("dense", "experts_q"):
        # a quantised checkpoint's codes and scales, laid out once when the model is loaded
        import unit_amd as U
        state["w"] = U.prepare_mxfp4_weight(*state["w"], case["k"])
    return state


# ------------------------------------------------------------------------------------- the plain forms
def _blocks(x):
    """(..., K) -> float (..., K / 32 rounded up, 32), zeros behind the end."""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK))
    return x.unflatten(-1, (-1, BLOCK))


def _power(biased):
    """2^(biased - 127), biased 0..254, put together from its bits."""
    return torch.where(biased > 0, biased << 23, 1 << 22).int().view(torch.float32)


def _quantized(x):
    """Blocks of floats -> magnitude index 0..7 with the sign in bit 3, and the biased exponent of each block's scale:
    the largest magnitude's binary exponent less 2 (the largest element, 6, is 1.5 * 2^2); 255 where a block holds an
    infinity or NaN.  Rounding to the nearest element, ties to the even index, magnitudes above 6 become 6."""
    b = _blocks(x)
    top = b.abs().amax(-1)
    scale = (torch.frexp(top).exponent.int() - 3 + 127).clamp(0, 254)
    scale = torch.where(top > 0, scale, torch.zeros_like(scale))
    y = b * _power(254 - scale).unsqueeze(-1)
    a = y.abs()
    index = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    scale = torch.where(torch.isfinite(top), scale, torch.full_like(scale, 255))
    return index + 8 * torch.signbit(b), scale


def _values(index, scale):
    """What the codes stand for, (..., K rounded up to whole blocks) in single precision."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=index.device)
    v = table[index.long()] * _power(scale.int().clamp(max=254)).unsqueeze(-1)
    return torch.where((scale == 255).unsqueeze(-1), math.nan, v).flatten(-2)


def _encode(w):
    """The storage of a checkpoint: two codes a byte, the even element in the low half, and a byte of scale per block."""
    index, scale = _quantized(w)
    pairs = index.flatten(-2).unflatten(-1, (-1, 2)).to(torch.uint8)
    return pairs[..., 0] + 16 * pairs[..., 1], scale.to(torch.uint8)


def _decode(codes, scales):
    index = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, BLOCK))
    return _values(index, scales)


def _places(sizes, rows, most):
    """Where row r of the sorted rows stands in a buffer of `most` rows per expert; rows of no expert go behind its end."""
    ends = sizes.long().cumsum(0)
    r = torch.arange(rows, device=sizes.device)
    e = torch.searchsorted(ends, r, right=True)
    starts = torch.cat((ends - sizes, ends[-1:]))
    return torch.where(e < len(sizes), e * most + r - starts[e], len(sizes) * most)


def _spread(x, places, experts, most):
    buf = x.new_zeros((experts * most + 1, x.shape[1]))
    buf[places] = x
    return buf[:-1].view(experts, most, -1)


def _collect(y, places):
    y = y.flatten(0, 1)
    return torch.cat((y, y.new_zeros((1, y.shape[1]))))[places]


def _plain(state):
    case, x = state["case"], state["x"]
    op = case["op"]
    if op == "quantize":
        return _values(*_quantized(x))[:, :case["k"]].to(x.dtype)
    out = DTYPES[case["out"]]
    if op == "dense":
        return (_values(*_quantized(x)) @ _decode(*state["w"]).t()).to(out)
    most = max(1, state["most"])
    places = _places(state["sizes"], case["rows"], most)
    w = _decode(*state["w"]) if op == "experts_q" else state["w"].float()
    x = _spread(_values(*_quantized(x)) if op == "experts_q" else x.float(), places, len(w), most)
    if op != "experts_grad":
        return _collect(torch.bmm(x, w.transpose(1, 2).contiguous()), places).to(out)
    dy = _spread(state["dy"].float(), places, len(w), most)
    dw = torch.bmm(dy.transpose(1, 2).contiguous(), x)
    return _collect(torch.bmm(dy, w), places).to(out), dw.to(DTYPES[case["weight_out"]])


def run(state):
    if not own:
        return _plain(state)
    import unit_amd as U
    case = state["case"]
    op = case["op"]
    if op == "quantize":
        return U.dequantize_mxfp4(U.quantize_mxfp4(state["x"]), out_dtype=case["dtype"])
    if op == "dense":
        return U.dense_mxfp4(state["x"], state["w"], out_dtype=case["out"])
    if op == "experts":
        return U.grouped_dense(state["x"], state["w"], state["sizes"], out_dtype=case["out"])
    if op == "experts_grad":
        return U.grouped_dense_grad(state["x"], state["w"], state["dy"], state["sizes"], out_dtype=case["out"],
                                    weight_out_dtype=case["weight_out"])
    return U.grouped_dense_mxfp4(state["x"], state["w"], state["sizes"], out_dtype=case["out"])


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    elements = (0.0, 1.0, 2.0, 4.0, 0.5, 1.5, 3.0, 6.0)  # even mantissas first: the first of two equally near ones is kept

    def two(power):  # its exact power, from its bits
        return ((power + 1023) << 52).view(torch.float64)

    def nearest(x):
        x = x.double()
        k = x.shape[-1]
        whole = torch.zeros((*x.shape[:-1], -(-k // BLOCK) * BLOCK), dtype=torch.float64, device=x.device)
        whole[..., :k] = x
        b = whole.view(*x.shape[:-1], -1, BLOCK)
        top = b.abs().max(-1, keepdim=True).values
        power = torch.floor(torch.log2(torch.where(top > 0, top, 2.0 ** -130))).long()
        power = power - (two(power) > top).long() * (top > 0) + (two(power + 1) <= top).long()
        unit = two(torch.clamp(power - 2, -127, 127))
        a, best, far = (b / unit).abs(), torch.zeros_like(b), torch.full_like(b, math.inf)
        for v in elements:
            d = (a - v).abs()
            best = torch.where(d < far, v, best)
            far = torch.minimum(d, far)
        return (torch.sign(b) * best * unit).flatten(-2)

    def stored(codes, scales):
        half = torch.stack((codes.int() % 16, codes.int() // 16), -1).flatten(-2)
        m = half % 8
        v = torch.where(m < 2, 0.5 * m.double(), (1.0 + 0.5 * (m % 2)) * two(m.long() // 2 - 1))
        return torch.where(half < 8, v, -v) * two(scales.long() - 127).repeat_interleave(BLOCK, -1)

    if op == "quantize":
        return nearest(s["x"])[:, :case["k"]]
    if op == "dense":
        return nearest(s["x"]) @ stored(*s["w"]).T
    x = nearest(s["x"]) if op == "experts_q" else s["x"].double()
    y = torch.zeros((case["rows"], case["k"] if op == "experts_grad" else case["n"]), dtype=torch.float64, device="cuda")
    dw = torch.zeros((case["experts"], case["n"], case["k"]), dtype=torch.float64, device="cuda") if op == "experts_grad" else None
    at = 0
    for e, size in enumerate(s["sizes"].tolist()):
        rows = slice(at, at + size)
        at += size
        if not size:
            continue
        w = stored(s["w"][0][e], s["w"][1][e]) if op == "experts_q" else s["w"][e].double()
        if op == "experts_grad":
            dy = s["dy"][rows].double()
            y[rows] = dy @ w
            dw[e] = dy.T @ x[rows]
        else:
            y[rows] = x[rows] @ w.T
    return (y, dw) if op == "experts_grad" else y


# ------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    rows, k, op = case["rows"], case["k"], case["op"]
    es = BYTES[case["dtype"]]
    if op == "quantize":
        # the floats in, codes and scales out, their values out; a scaling each way per element
        return {"bytes": rows * (2 * k * es + -(-k // BLOCK) * 17), "flops": 2 * rows * k}
    n, eo = case["n"], BYTES[case["out"]]
    if op == "dense":
        return {"bytes": rows * k * es + n * -(-k // BLOCK) * 17 + rows * n * eo, "flops": 2 * rows * n * k}
    taken = case["rows"] - case["spare"]
    busy = sum(s > 0 for s in _sizes(case, 0))  # an expert without rows leaves its weight unread
    if op == "experts":
        return {"bytes": (taken * k + busy * n * k) * es + rows * n * eo, "flops": 2 * taken * n * k}
    if op == "experts_q":
        return {"bytes": taken * k * es + busy * n * -(-k // BLOCK) * 17 + rows * n * eo, "flops": 2 * taken * n * k}
    return {"bytes": (taken * (n + k) + busy * n * k) * es + rows * k * eo + case["experts"] * n * k * BYTES[case["weight_out"]],
            "flops": 4 * taken * n * k}
