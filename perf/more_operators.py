"""Gated feed-forward products, their gradients and 8-bit activation checkpoints, as cases that can be timed and compared.

Operators (`case["op"]`):

  gated       h[r] = act(gate . x[r]) * (up . x[r]); a weight (2 N, K) holds gate's rows, then up's.  With `experts`, rows are sorted by
              expert and each expert has such a weight.  keep "pre": gate . x and up . x come back too, (rows, 2, N)
  gated_q     the same with rows that are quantised on the way to MXFP4 and weights in MXFP4
  checkpoint  rows -> MXFP8: blocks of 32 along a row share the smallest power of two for which their largest magnitude is at most
              448, elements are 8-bit floats (4 exponent bits, 3 mantissa bits); what is returned are the values they stand for
  gated_grad  the gradients of `gated` for dy: dx and dweight, from kept pre-activations (kept "pre") or from the rows alone ("rows")
  gated_step  a training step that keeps rows and pre-activations in MXFP8 between `gated` and `gated_grad`: h, dx, dweight

act is "silu", z / (1 + exp(-z)), or "gelu_tanh", z (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2.

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
MAX_BYTES = 5.0e8    # operands and results of the largest drawn case


def listed():
    return [
        # one token through the block of a served model: the weight is read once
        dict(name="gated_token", op="gated", rows=1, experts=0, n=4096, k=2048, act="silu", dtype="bfloat16", out="bfloat16", keep=""),
        # a handful of requests, nothing aligned to a tile, results for a loss in single precision
        dict(name="gated_ragged", op="gated", rows=333, experts=0, n=1512, k=2088, act="gelu_tanh", dtype="float16", out="float32", keep=""),
        # a prompt: the largest product
        dict(name="gated_prompt", op="gated", rows=8192, experts=0, n=4096, k=2048, act="silu", dtype="bfloat16", out="bfloat16", keep=""),
        # a training batch over experts, popular and unpopular ones, a buffer whose last rows belong to none, pre-activations kept
        dict(name="gated_experts_batch", op="gated", rows=16384, experts=32, skew=0.5, spare=200, n=1024, k=1024, act="silu",
             dtype="bfloat16", out="bfloat16", keep="pre", route=1),
        # thirty-two requests, two experts each, one new token, on quantised experts
        dict(name="gated_q_token", op="gated_q", rows=64, experts=64, skew=0.5, spare=0, n=1024, k=2048, act="silu", dtype="bfloat16",
             out="bfloat16", route=2),
        # a prompt on a quantised block
        dict(name="gated_q_prompt", op="gated_q", rows=8192, experts=0, n=4096, k=2048, act="gelu_tanh", dtype="bfloat16", out="bfloat16"),
        # rows of a small model kept in 8 bits, single precision, rows that end inside a block and inside a cache line
        dict(name="checkpoint_ragged", op="checkpoint", rows=1003, k=1333, dtype="float32"),
        # the hidden activations of a training batch, kept and restored
        dict(name="checkpoint_batch", op="checkpoint", rows=8192, k=4096, dtype="bfloat16"),
        # gradients of a small fine-tuning batch, ragged in every size, from its rows alone
        dict(name="gated_grad_ragged", op="gated_grad", rows=1000, experts=12, skew=0.7, spare=0, n=776, k=520, act="gelu_tanh",
             dtype="float16", kept="rows", route=3),
        # gradients of a training batch, pre-activations kept in 16 bits
        dict(name="gated_grad_batch", op="gated_grad", rows=8192, experts=16, skew=0.5, spare=0, n=2048, k=1024, act="silu",
             dtype="bfloat16", kept="pre", route=4),
        # a training step of a small dense block on 8-bit checkpoints
        dict(name="gated_step_small", op="gated_step", rows=777, experts=0, n=1032, k=776, act="silu", dtype="float16"),
        # a training step over experts on 8-bit checkpoints
        dict(name="gated_step_batch", op="gated_step", rows=8192, experts=16, skew=0.5, spare=100, n=1024, k=1024, act="silu",
             dtype="bfloat16", route=5),
    ]


# ------------------------------------------------------------------------------------- drawn cases
def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_one(rng):
    op = rng.choice(["gated", "gated", "gated_q", "checkpoint", "gated_grad", "gated_step"])
    rows = _log_int(rng, 1, 16384)
    if op == "checkpoint":
        return dict(op=op, rows=rows, k=_log_int(rng, 1, 8192), dtype=rng.choice(["float32", "float16", "bfloat16"]))
    step = rng.choice([8, 8, 64])  # rows of 16-bit weights are whole 16-byte pieces; half of the cases are ragged beyond that
    dtype = rng.choice(["float16", "bfloat16"])
    case = dict(op=op, rows=rows, experts=rng.choice([0, _log_int(rng, 1, 128)]), n=step * _log_int(rng, 64 // step, 4096 // step),
                k=step * _log_int(rng, 64 // step, 4096 // step), act=rng.choice(["silu", "gelu_tanh"]), dtype=dtype)
    if op == "gated_q" and rng.random() < 0.4:
        case.update(n=_log_int(rng, 1, 4096), k=_log_int(rng, 33, 4096))
    if case["experts"]:
        case.update(skew=rng.choice([0.0, 0.5, 1.0]), route=rng.randrange(1 << 30), spare=rng.choice([0, 0, rows // 10]))
    if op in ("gated", "gated_q"):
        case["out"] = rng.choice(["float32", dtype])
    if op == "gated":
        case["keep"] = rng.choice(["", "pre"])
    if op == "gated_grad":
        case["kept"] = rng.choice(["pre", "rows"])
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


def _inputs(case, seed):
    g, op = torch.Generator(device="cuda").manual_seed(seed), case["op"]
    rows, k, dtype = case["rows"], case["k"], case["dtype"]
    x = dict(x=_rows(rows, k, dtype, g))
    if op == "checkpoint":
        return x
    n, e = case["n"], case["experts"]
    w = (torch.randn(((e,) if e else ()) + (2 * n, k), device="cuda", generator=g) / math.sqrt(k)).to(DTYPES["bfloat16" if op == "gated_q" else dtype])
    x["w"] = _encode(w) if op == "gated_q" else w
    if e:
        sizes = _sizes(case, seed)
        x.update(sizes=torch.tensor(sizes, dtype=torch.int32, device="cuda"), most=max(sizes))
    if op in ("gated_grad", "gated_step"):
        x["dy"] = _rows(rows, n, dtype, g, 2.0 ** -7)
    if op == "gated_grad" and case["kept"] == "pre":
        x["pre"] = _pre_activations(x["x"].float(), w.float(), x).to(x["x"].dtype)
    return x


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if own and case["op"] == "gated_q":
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


def _quantized4(x):
    """MXFP4: magnitude index 0..7 with the sign in bit 3, and the biased exponent of each block's scale: the largest magnitude's binary
    exponent less 2.  Rounding to the nearest element, ties to the even index, magnitudes above 6 become 6."""
    b = _blocks(x)
    top = b.abs().amax(-1)
    scale = (torch.frexp(top).exponent.int() - 3 + 127).clamp(0, 254)
    scale = torch.where(top > 0, scale, torch.zeros_like(scale))
    a = (b * _power(254 - scale).unsqueeze(-1)).abs()
    index = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    return index + 8 * torch.signbit(b), scale


def _values4(index, scale):
    """What the codes stand for, (..., K rounded up to whole blocks) in single precision."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=index.device)
    return (table[index.long()] * _power(scale.int()).unsqueeze(-1)).flatten(-2)


def _encode(w):
    """The storage of a checkpoint: two codes a byte, the even element in the low half, and a byte of scale per block."""
    index, scale = _quantized4(w)
    pairs = index.flatten(-2).unflatten(-1, (-1, 2)).to(torch.uint8)
    return pairs[..., 0] + 16 * pairs[..., 1], scale.to(torch.uint8)


def _decode(codes, scales):
    index = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).unflatten(-1, (-1, BLOCK))
    return _values4(index, scales)


def _kept8(x):
    """The values of x's MXFP8 checkpoint, in single precision."""
    b = _blocks(x)
    top = b.abs().amax(-1)
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    scale = (exponent.int() - 9 + (mantissa > 0.875).int() + 127).clamp(0, 254)
    scale = torch.where(top > 0, scale, torch.zeros_like(scale))
    y = b * _power(254 - scale).unsqueeze(-1)
    step = torch.frexp(y).exponent.int().clamp(min=-5) - 4  # 2^-9 below the normal range, three mantissa bits in it
    v = torch.round(torch.ldexp(y, -step)) * _power(step + 127)
    return (v * _power(scale).unsqueeze(-1)).flatten(-2)[..., :x.shape[-1]]


def _places(sizes, rows, most):
    """Where row r of the sorted rows stands in a buffer of `most` rows per expert; rows of no expert go behind its end."""
    ends = sizes.long().cumsum(0)
    r = torch.arange(rows, device=sizes.device)
    e = torch.searchsorted(ends, r, right=True)
    starts = torch.cat((ends - sizes, ends[-1:]))
    return torch.where(e < len(sizes), e * most + r - starts[e], len(sizes) * most)


def _by_expert(x, s):
    """(rows, c) -> (experts, most, c), one expert without sizes"""
    if "sizes" not in s:
        return x.unsqueeze(0)
    buf = x.new_zeros((len(s["sizes"]) * s["most"] + 1, x.shape[1]))
    buf[_places(s["sizes"], len(x), s["most"])] = x
    return buf[:-1].view(len(s["sizes"]), s["most"], -1)


def _by_row(y, s, rows):
    y = y.flatten(0, 1)
    return torch.cat((y, y.new_zeros((1, y.shape[1]))))[_places(s["sizes"], rows, s["most"])] if "sizes" in s else y


def _pre_activations(x, w, s):
    """(rows, 2, N): gate . x, up . x"""
    w = w if w.dim() == 3 else w.unsqueeze(0)
    return _by_row(torch.bmm(_by_expert(x, s), w.transpose(1, 2).contiguous()), s, len(x)).unflatten(-1, (2, -1))


def _act(z, act):
    """act(z) and its derivative"""
    c = math.sqrt(8.0 / math.pi)
    share = torch.sigmoid(z if act == "silu" else c * (z + 0.044715 * z ** 3))  # (1 + tanh(a)) / 2 = sigmoid(2 a)
    slope = 1.0 if act == "silu" else c * (1.0 + 3 * 0.044715 * z ** 2)
    return z * share, share + z * share * (1.0 - share) * slope


def _gradients(x, w, dy, pre, s, case):
    g, u = pre.unbind(1)
    a, d = _act(g, case["act"])
    dpre = _by_expert(torch.cat((dy * u * d, dy * a), 1), s)
    dw = torch.bmm(dpre.transpose(1, 2).contiguous(), _by_expert(x, s))
    dx = _by_row(torch.bmm(dpre, w if w.dim() == 3 else w.unsqueeze(0)), s, len(x))
    dtype = DTYPES[case["dtype"]]
    return dx.to(dtype), (dw if w.dim() == 3 else dw[0]).to(dtype)


def _plain(s):
    case, x = s["case"], s["x"]
    op = case["op"]
    if op == "checkpoint":
        return _kept8(x).to(x.dtype)
    if op == "gated_q":
        x, w = _values4(*_quantized4(x)), _decode(*s["w"])
    else:
        x, w = x.float(), s["w"].float()
    if op == "gated_grad" and case["kept"] == "pre":
        return _gradients(x, w, s["dy"].float(), s["pre"].float(), s, case)
    pre = _pre_activations(x, w, s)
    if op == "gated_grad":
        return _gradients(x, w, s["dy"].float(), pre, s, case)
    h = _act(pre[:, 0], case["act"])[0] * pre[:, 1]
    if op == "gated_step":
        return h.to(DTYPES[case["dtype"]]), *_gradients(_kept8(x), w, s["dy"].float(), _kept8(pre), s, case)
    h = h.to(DTYPES[case["out"]])
    return (h, pre.to(DTYPES[case["dtype"]])) if op == "gated" and case["keep"] else h


def run(state):
    if not own:
        return _plain(state)
    import unit_amd as U
    case, x, sizes = state["case"], state["x"], state.get("sizes")
    op, dtype = case["op"], case["dtype"]
    if op == "checkpoint":
        return U.dequantize_mxfp8(U.quantize_mxfp8(x), out_dtype=dtype)
    if op == "gated":
        return U.gated_dense(x, state["w"], sizes, activation=case["act"], out_dtype=case["out"], keep=case["keep"] or None)
    if op == "gated_q":
        return U.gated_dense_mxfp4(x, state["w"], sizes, activation=case["act"], out_dtype=case["out"])
    if op == "gated_grad":
        return U.gated_dense_grad(x, state["w"], state["dy"], sizes, activation=case["act"], pre=state.get("pre"), out_dtype=dtype,
                                  weight_out_dtype=dtype)
    h, pre = U.gated_dense(x, state["w"], sizes, activation=case["act"], out_dtype=dtype, keep="mxfp8")
    rows = U.quantize_mxfp8(x)
    return h, *U.gated_dense_grad(rows, state["w"], state["dy"], sizes, activation=case["act"], pre=pre, out_dtype=dtype, weight_out_dtype=dtype)


# ------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]

    def two(power):  # its exact power, from its bits
        return ((power + 1023) << 52).view(torch.float64)

    def blocks(x):
        k = x.shape[-1]
        whole = torch.zeros((*x.shape[:-1], -(-k // BLOCK) * BLOCK), dtype=torch.float64, device=x.device)
        whole[..., :k] = x
        b = whole.view(*x.shape[:-1], -1, BLOCK)
        top = b.abs().max(-1, keepdim=True).values
        power = torch.floor(torch.log2(torch.where(top > 0, top, 2.0 ** -130))).long()
        power = power - (two(power) > top).long() * (top > 0) + (two(power + 1) <= top).long()
        return b, top, power

    def nearest(b, unit, elements):
        """b / unit to the nearest of the elements, which ascend from 0 and alternate between even and odd codes; ties to even"""
        t = torch.tensor(elements, dtype=torch.float64, device=b.device)
        middle = (t[1:] + t[:-1]) / 2
        a = (b / unit).abs()
        i = torch.bucketize(a, middle)  # the lower one on a tie
        i = i + ((i % 2 == 1) & (a == middle[i.clamp(max=len(middle) - 1)]))
        return (torch.sign(b) * t[i] * unit).flatten(-2)

    def four(x):
        b, _, power = blocks(x.double())
        return nearest(b, two(torch.clamp(power - 2, -127, 127)), (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0))[..., :x.shape[-1]]

    def eight(x):
        b, top, power = blocks(x.double())
        power = power - 8
        power = torch.clamp(power + (top > 448.0 * two(power)).long(), -127, 127)
        normal = [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1]  # 480 is not among them
        return nearest(b, two(power), [m * 2.0 ** -9 for m in range(8)] + normal)[..., :x.shape[-1]]

    def stored(codes, scales):
        half = torch.stack((codes.int() % 16, codes.int() // 16), -1).flatten(-2)
        m = half % 8
        v = torch.where(m < 2, 0.5 * m.double(), (1.0 + 0.5 * (m % 2)) * two(m.long() // 2 - 1))
        return (torch.where(half < 8, v, -v) * two(scales.long() - 127).repeat_interleave(BLOCK, -1))[..., :case["k"]]

    if op == "checkpoint":
        return eight(s["x"])
    n, k, rows = case["n"], case["k"], case["rows"]
    w = stored(*s["w"]) if op == "gated_q" else s["w"]
    x = four(s["x"]) if op == "gated_q" else s["x"].double()
    lots = [(slice(0, rows), None)]
    if "sizes" in s:
        lots, at = [], 0
        for e, size in enumerate(s["sizes"].tolist()):
            lots += [(slice(at, at + size), e)] if size else []
            at += size

    def weight(e):
        return (w if e is None else w[e]).double()

    if op == "gated_grad" and case["kept"] == "pre":
        pre = s["pre"].double().flatten(1)
    else:
        pre = torch.zeros((rows, 2 * n), dtype=torch.float64, device="cuda")
        for r, e in lots:
            pre[r] = x[r] @ weight(e).T

    def activation(z):
        if case["act"] == "silu":
            return z / (1 + torch.exp(-z))
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))

    h = activation(pre[:, :n]) * pre[:, n:]
    if op == "gated_q" or op == "gated" and not case["keep"]:
        return h
    if op == "gated":
        return h, pre.view(rows, 2, n)
    if op == "gated_step":
        x, pre = eight(x), eight(pre.view(rows, 2, n)).flatten(1)
    z = pre[:, :n].clone().requires_grad_()
    dy = s["dy"].double()
    slope, = torch.autograd.grad(activation(z).sum(), z)
    dpre = torch.cat((dy * pre[:, n:] * slope, dy * activation(z.detach())), 1)
    dx, dw = torch.zeros((rows, k), dtype=torch.float64, device="cuda"), torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    for r, e in lots:
        dx[r] = dpre[r] @ weight(e)
        if e is None:
            dw = dpre[r].T @ x[r]
        else:
            dw[e] = dpre[r].T @ x[r]
    return (h, dx, dw) if op == "gated_step" else (dx, dw)


# ------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    rows, k, op = case["rows"], case["k"], case["op"]
    es = BYTES[case["dtype"]]
    if op == "checkpoint":
        # the floats in, codes and scales out, their values out; a scaling each way per element
        return {"bytes": rows * (2 * k * es + -(-k // BLOCK) * 33), "flops": 2 * rows * k}
    n = case["n"]
    taken = rows - case.get("spare", 0)
    busy = sum(s > 0 for s in _sizes(case, 0)) if case["experts"] else 1  # an expert without rows leaves its weight unread
    held = busy * 2 * n * (-(-k // BLOCK) * 17 if op == "gated_q" else k * es)
    product = 4 * taken * n * k
    if op in ("gated", "gated_q"):
        return {"bytes": taken * k * es + held + rows * n * BYTES[case["out"]] + (rows * 2 * n * es if case.get("keep") else 0), "flops": product}
    gradients = (taken * (k + n) + rows * k + max(1, case["experts"]) * 2 * n * k) * es
    if op == "gated_step":
        # h too, and the checkpoints written and read: the two halves are calls of their own
        kept = taken * (-(-k // BLOCK) + 2 * -(-n // BLOCK)) * 33
        return {"bytes": held + gradients + rows * n * es + 2 * kept, "flops": 3 * product}
    if case["kept"] == "rows":
        return {"bytes": held + gradients, "flops": 3 * product}
    return {"bytes": held + gradients + taken * 2 * n * es, "flops": 2 * product}
