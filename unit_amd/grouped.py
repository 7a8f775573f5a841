"""Products of expert layers and of MXFP4 operands: operators on torch tensors that live on the MI355X, like those of ops.py
(same helpers, same manner: raw device pointers to the C ABI, torch allocates the results and workspaces).  No counterpart in
the reference, whose dense operators (apps/cpu/relay/int8-gemm.py:14-16, apps/gpu/gemm.py:8-20) these stand beside.

  quantize_mxfp4, dequantize_mxfp4   floats <-> 4-bit floats with a power of two per 32 elements
  quantize_mxfp8, dequantize_mxfp8   floats <-> 8-bit floats with a power of two per 32 elements: activations kept for a backward pass
  prepare_mxfp4_weight               a checkpoint's codes and scales, laid out once for the products
  dense_mxfp4                        x . W^T with both operands in MXFP4
  grouped_dense, grouped_dense_grad  rows sorted by expert times their expert's weight, and the gradients
  grouped_dense_mxfp4                the same product with MXFP4 operands
"""
import contextlib
import ctypes
import math

import torch

from . import _lib
from ._lib import check
from .ops import _Calls, _dev, _device, _stream

__all__ = ["Mxfp4Tensor", "Mxfp8Tensor", "quantize_mxfp8", "dequantize_mxfp8", "quantize_mxfp4", "dequantize_mxfp4", "prepare_mxfp4_weight", "dense_mxfp4", "grouped_dense",
           "grouped_dense_grad", "grouped_dense_mxfp4"]

_MXFP4, _MXFP8 = 3, 4
_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_OUT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _out_dtype(name, arg="out_dtype"):
    try:
        return _OUT[name]
    except (KeyError, TypeError):
        raise ValueError(f"{arg}: expected 'float32', 'float16' or 'bfloat16', got {name!r}") from None


def _floats(t, name, dtypes, ndim=None):
    t = _dev(t, name, None, ndim)
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: expected dtype {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    return t


def _sizes(group_sizes, data):
    s = _dev(group_sizes, "group_sizes", None, 1)
    if s.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"group_sizes: expected dtype torch.int32 or torch.int64, got {s.dtype}")
    _same_device(s, "group_sizes", data)
    return s


def _same_device(t, name, data):
    if t.device != data.device:
        raise ValueError(f"{name}: lives on {t.device}, the data on {data.device}")


def _on(t):
    """the device that t lives on as the current one, so that its current stream is what the work runs on"""
    if _device is not None and t.device.index == _device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


class _GroupedCalls(_Calls):
    """The common case of this module's operators as native functions, like ops._Calls."""

    _NAMES = ("quantize", "dequantize", "product_mx", "grouped", "grouped_grad")
    _LIBRARY = ("unit_mxfp4_bytes", "unit_quantize_mxfp4", "unit_dequantize_mxfp4", "unit_mxfp4_workspace_bytes", "unit_dense_mxfp4",
                "unit_grouped_dense", "unit_grouped_dense_grad_data", "unit_grouped_dense_grad_weight", "unit_grouped_dense_mxfp4")

    def _bind(self, calls, addresses):
        calls.bind_grouped(addresses, Mxfp4Tensor)


_native = _GroupedCalls()


# ------------------------------------------------------------------------------- MXFP4
def _mxfp4_bytes(rows, k):
    codes, scales = ctypes.c_size_t(), ctypes.c_size_t()
    check(_lib.load().unit_mxfp4_bytes(rows, k, ctypes.byref(codes), ctypes.byref(scales)))
    return codes.value, scales.value


class Mxfp4Tensor:
    """A matrix (rows, K), or a stack of them, in MXFP4: along the last axis blocks of 32 elements share a power of two, elements
    are 4-bit floats (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives).  `buf` holds the codes, then the scales, in the layout that
    the products read (include/unit_amd.h); made by quantize_mxfp4 and prepare_mxfp4_weight, read back by dequantize_mxfp4."""

    __slots__ = ("buf", "shape")

    def __init__(self, buf, shape):
        self.buf, self.shape = buf, shape

    @property
    def device(self):
        return self.buf.device

    def _pointers(self):
        """addresses of codes and scales, rows, K"""
        rows = math.prod(self.shape[:-1])
        codes, scales = _mxfp4_bytes(rows, self.shape[-1])
        if self.buf.numel() < codes + scales:
            raise ValueError(f"{self!r}: a buffer of {self.buf.numel()} bytes, {codes + scales} needed")
        return self.buf.data_ptr(), self.buf.data_ptr() + codes, rows, self.shape[-1]

    def __repr__(self):
        return f"Mxfp4Tensor(shape={self.shape}, device='{self.device}')"


def _mxfp4_empty(shape, device):
    return Mxfp4Tensor(torch.empty((sum(_mxfp4_bytes(math.prod(shape[:-1]), shape[-1])),), dtype=torch.uint8, device=device), tuple(shape))


def quantize_mxfp4(x):
    """x (rows, K) or (E, rows, K) float32, float16 or bfloat16 -> Mxfp4Tensor of the same shape.

    The scale of a block is the power of two below its largest magnitude, divided by 4 and at least 2^-127; elements are
    x / scale rounded to the nearest 4-bit float, ties to the even mantissa, magnitudes above 6 to 6.  A block that holds an
    infinity or a NaN becomes NaN throughout."""
    q = _native.quantize(x)
    if q is not None:
        return q
    x = _floats(x, "x", tuple(_CODE))
    if x.dim() not in (2, 3):
        raise ValueError(f"x: expected two axes or three, got shape {tuple(x.shape)}")
    with _on(x):
        q = _mxfp4_empty(x.shape, x.device)
        codes, scales, rows, k = q._pointers()
        check(_lib.load().unit_quantize_mxfp4(x.data_ptr(), _CODE[x.dtype], rows, k, codes, scales, _stream()))
    return q


def _mxfp4(q, name):
    if not isinstance(q, Mxfp4Tensor):
        raise TypeError(f"{name}: expected an Mxfp4Tensor, got {type(q).__name__}")
    return q


def dequantize_mxfp4(q, out_dtype="float32"):
    """The values that an Mxfp4Tensor stands for (rounded once where out_dtype does not hold them)."""
    out = _native.dequantize(q, out_dtype)
    if out is not None:
        return out
    codes, scales, rows, k = _mxfp4(q, "q")._pointers()
    dt = _out_dtype(out_dtype)
    with _on(q.buf):
        out = torch.empty(q.shape, dtype=dt, device=q.device)
        check(_lib.load().unit_dequantize_mxfp4(codes, scales, rows, k, out.data_ptr(), _CODE[dt], _stream()))
    return out


def prepare_mxfp4_weight(codes, scales, k=None):
    """The storage of a quantised checkpoint -> Mxfp4Tensor (N, k) or (E, N, k), accepted by dense_mxfp4 and grouped_dense_mxfp4.

    codes  uint8 (N, 16 * b) or (E, N, 16 * b): two codes a byte, the even element in the low half
    scales uint8 (N, b) or (E, N, b): biased exponents, 255 for NaN;  k at most 32 * b and more than 32 * (b - 1), 32 * b unless given"""
    codes, scales = _dev(codes, "codes", torch.uint8), _dev(scales, "scales", torch.uint8)
    _same_device(scales, "scales", codes)
    if codes.dim() not in (2, 3) or codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != 16 * scales.shape[-1]:
        raise ValueError(f"codes {tuple(codes.shape)}, scales {tuple(scales.shape)}: expected (..., 16 * b) and (..., b)")
    b = scales.shape[-1]
    k = 32 * b if k is None else int(k)
    if not 32 * (b - 1) < k <= 32 * b:
        raise ValueError(f"k: {k} elements do not fill {b} blocks of 32")
    with _on(codes):
        q = _mxfp4_empty((*codes.shape[:-1], k), codes.device)
        to, sto, rows, _ = q._pointers()
        check(_lib.load().unit_prepare_mxfp4(codes.data_ptr(), scales.data_ptr(), rows, k, to, sto, _stream()))
    return q


def _mxfp4_product(data, weight, group_sizes, out_dtype, ndim):
    dt = _out_dtype(out_dtype)
    if len(_mxfp4(weight, "weight").shape) != ndim:
        raise ValueError(f"weight: expected {ndim} axes, got shape {weight.shape}")
    n, k = weight.shape[-2:]
    quantised = isinstance(data, Mxfp4Tensor)
    if not quantised:
        data = _floats(data, "data", tuple(_CODE), 2)
    if len(data.shape) != 2 or data.shape[1] != k:
        raise ValueError(f"data: expected (rows, {k}), got {tuple(data.shape)}")
    _same_device(weight, "weight", data)
    sizes = None
    if ndim == 3:
        sizes = _sizes(group_sizes, data)
        if sizes.shape[0] != weight.shape[0]:
            raise ValueError(f"group_sizes: expected {weight.shape[0]} entries, got {sizes.shape[0]}")
    rows, ws, L = data.shape[0], None, _lib.load()
    with _on(weight.buf):
        if quantised:
            operand = (*data._pointers()[:2], _MXFP4)
        else:
            need = ctypes.c_size_t()
            check(L.unit_mxfp4_workspace_bytes(rows, k, ctypes.byref(need)))
            ws = torch.empty((need.value,), dtype=torch.uint8, device=data.device)
            operand = (data.data_ptr(), None, _CODE[data.dtype])
        codes, scales = weight._pointers()[:2]
        out = torch.empty((rows, n), dtype=dt, device=data.device)
        tail = (None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), _stream())
        if ndim == 2:
            check(L.unit_dense_mxfp4(*operand, codes, scales, out.data_ptr(), _CODE[dt], rows, n, k, *tail))
        else:
            check(L.unit_grouped_dense_mxfp4(*operand, codes, scales, sizes.data_ptr(), sizes.element_size(), out.data_ptr(), _CODE[dt],
                                             rows, weight.shape[0], n, k, *tail))
    return out


def dense_mxfp4(data, weight, out_dtype="float32"):
    """out (M, N) = q(data) . weight^T, products and sums in float32, rounded once to out_dtype.

    data (M, K) float32, float16 or bfloat16, quantised on the way as quantize_mxfp4 does, or an Mxfp4Tensor;
    weight an Mxfp4Tensor (N, K)"""
    out = _native.product_mx(data, weight, None, out_dtype)
    return _mxfp4_product(data, weight, None, out_dtype, 2) if out is None else out


def grouped_dense_mxfp4(data, weight, group_sizes, out_dtype="float32"):
    """grouped_dense with MXFP4 operands: data as in dense_mxfp4, weight an Mxfp4Tensor (E, N, K)."""
    out = _native.product_mx(data, weight, group_sizes, out_dtype) if group_sizes is not None else None
    return _mxfp4_product(data, weight, group_sizes, out_dtype, 3) if out is None else out


# ------------------------------------------------------------------------------- MXFP8
def _mxfp8_bytes(rows, k):
    codes, scales = ctypes.c_size_t(), ctypes.c_size_t()
    check(_lib.load().unit_mxfp8_bytes(rows, k, ctypes.byref(codes), ctypes.byref(scales)))
    return codes.value, scales.value


class Mxfp8Tensor:
    """Rows in MXFP8: along the last axis blocks of 32 elements share a power of two, elements are 8-bit floats (e4m3: three mantissa
    bits, up to 448).  33 bytes for 32 elements: what a training step keeps of its activations until the backward pass.  `buf` holds the
    codes, then the scales (include/unit_amd.h); made by quantize_mxfp8 and gated_dense, read back by dequantize_mxfp8."""

    __slots__ = ("buf", "shape")

    def __init__(self, buf, shape):
        self.buf, self.shape = buf, shape

    @property
    def device(self):
        return self.buf.device

    def _pointers(self):
        """addresses of codes and scales, rows, length of a row"""
        rows = math.prod(self.shape[:-1])
        codes, scales = _mxfp8_bytes(rows, self.shape[-1])
        if self.buf.numel() < codes + scales:
            raise ValueError(f"{self!r}: a buffer of {self.buf.numel()} bytes, {codes + scales} needed")
        return self.buf.data_ptr(), self.buf.data_ptr() + codes, rows, self.shape[-1]

    def __repr__(self):
        return f"Mxfp8Tensor(shape={self.shape}, device='{self.device}')"


class _GatedCalls(_Calls):
    """The common case of MXFP8 and of the gated products (gated.py) as native functions, like ops._Calls."""

    _NAMES = ("quantize8", "dequantize8", "gated", "gated_mx", "gated_grad")
    _LIBRARY = ("unit_mxfp4_bytes", "unit_mxfp4_workspace_bytes", "unit_mxfp8_bytes", "unit_quantize_mxfp8", "unit_dequantize_mxfp8", "unit_gated_dense",
                "unit_gated_dense_mxfp4", "unit_gated_dense_grad_ws_bytes", "unit_gated_dense_grad")

    def _bind(self, calls, addresses):
        calls.bind_gated(addresses, Mxfp4Tensor, Mxfp8Tensor)


_native_gated = _GatedCalls()


def _mxfp8_empty(shape, device):
    return Mxfp8Tensor(torch.empty((sum(_mxfp8_bytes(math.prod(shape[:-1]), shape[-1])),), dtype=torch.uint8, device=device), tuple(shape))


def quantize_mxfp8(x):
    """x of two or three axes, float32, float16 or bfloat16 -> Mxfp8Tensor of the same shape.

    The scale of a block is the smallest power of two, 2^-127 at least, for which its largest magnitude is at most 448; elements are
    x / scale rounded to the nearest 8-bit float, ties to the even mantissa, so nothing saturates.  A block that holds an infinity or
    a NaN becomes NaN throughout."""
    q = _native_gated.quantize8(x)
    if q is not None:
        return q
    x = _floats(x, "x", tuple(_CODE))
    if x.dim() not in (2, 3):
        raise ValueError(f"x: expected two axes or three, got shape {tuple(x.shape)}")
    with _on(x):
        q = _mxfp8_empty(x.shape, x.device)
        codes, scales, rows, k = q._pointers()
        check(_lib.load().unit_quantize_mxfp8(x.data_ptr(), _CODE[x.dtype], rows, k, codes, scales, _stream()))
    return q


def dequantize_mxfp8(q, out_dtype="float32"):
    """The values that an Mxfp8Tensor stands for, rounded once where out_dtype does not hold them.  The type that was quantised holds them all
    but for the power of two above its largest value, which magnitudes within a thirty-second of it become: infinite."""
    out = _native_gated.dequantize8(q, out_dtype)
    if out is not None:
        return out
    dt = _out_dtype(out_dtype)
    if not isinstance(q, Mxfp8Tensor):
        raise TypeError(f"q: expected an Mxfp8Tensor, got {type(q).__name__}")
    with _on(q.buf):
        codes, scales, rows, k = q._pointers()
        out = torch.empty(q.shape, dtype=dt, device=q.device)
        check(_lib.load().unit_dequantize_mxfp8(codes, scales, rows, k, out.data_ptr(), _CODE[dt], _stream()))
    return out


# ------------------------------------------------------------------------------- 16-bit operands
_NAME = {v: k for k, v in _OUT.items()}
_HALVES = (torch.float16, torch.bfloat16)


def _grouped(data, weight, group_sizes, read=True):
    """read: the rows' elements are, not their shape alone"""
    if isinstance(data, Mxfp8Tensor) or not read:
        weight = _floats(weight, "weight", _HALVES, 3)
    else:
        data = _floats(data, "data", _HALVES, 2)
        weight = _dev(weight, "weight", data.dtype, 3)
    _same_device(weight, "weight", data)
    sizes = _sizes(group_sizes, data)
    e, n, k = weight.shape
    if len(data.shape) != 2 or data.shape[1] != k:
        raise ValueError(f"data: expected (rows, {k}), got {tuple(data.shape)}")
    if sizes.shape[0] != e:
        raise ValueError(f"group_sizes: expected {e} entries, got {sizes.shape[0]}")
    return data, weight, sizes, e, n, k


def grouped_dense(data, weight, group_sizes, out_dtype="float32"):
    """Rows sorted by expert times their expert's weight: out[r] = weight[e(r)] . data[r].

    data (rows, K) float16 or bfloat16; weight (E, N, K) of the same type, N and K multiples of 8;
    group_sizes (E,) int32 or int64 on the GPU: how many rows each expert has, in order.  Nothing waits for its values: a size
    counts as min(max(size, 0), rows left), and rows behind the last expert's give zeros.  float32 sums, rounded once."""
    out = _native.grouped(data, weight, group_sizes, out_dtype)
    if out is not None:
        return out
    dt = _out_dtype(out_dtype)
    if isinstance(data, Mxfp8Tensor):
        raise TypeError("data: expected a torch.Tensor, got Mxfp8Tensor (which grouped_dense_grad takes)")
    data, weight, sizes, e, n, k = _grouped(data, weight, group_sizes)
    with _on(data):
        out = torch.empty((data.shape[0], n), dtype=dt, device=data.device)
        check(_lib.load().unit_grouped_dense(data.data_ptr(), weight.data_ptr(), sizes.data_ptr(), sizes.element_size(), out.data_ptr(),
                                             _CODE[data.dtype], _CODE[dt], data.shape[0], e, n, k, _stream()))
    return out


def grouped_dense_grad(data, weight, grad, group_sizes, out_dtype="float32", weight_out_dtype="float32"):
    """The gradients of grouped_dense for grad (rows, N), of data's type: (ddata (rows, K), dweight (E, N, K)), in out_dtype and
    weight_out_dtype.  ddata is zero in rows of no expert, dweight for experts without rows; sums in float32, in the order of
    the rows whatever runs beside it.  data may be kept in MXFP8 (rows, K), grad is then of weight's type and so are the rows again."""
    both = _native.grouped_grad(data, weight, grad, group_sizes, out_dtype, weight_out_dtype)
    if both is not None:
        return both
    return _grouped_grad(data, weight, grad, group_sizes, out_dtype, weight_out_dtype)


def _grouped_grad(data, weight, grad, group_sizes, out_dtype, weight_out_dtype, wanted=(True, True)):
    """(ddata, dweight), None in the place of one that is not wanted: it costs neither time nor memory"""
    dt, wdt = _out_dtype(out_dtype), _out_dtype(weight_out_dtype, "weight_out_dtype")
    data, weight, sizes, e, n, k = _grouped(data, weight, group_sizes, wanted[1])
    grad = _dev(grad, "grad", weight.dtype, 2)
    _same_device(grad, "grad", data)
    rows = data.shape[0]
    if tuple(grad.shape) != (rows, n):
        raise ValueError(f"grad: expected ({rows}, {n}), got {tuple(grad.shape)}")
    L = _lib.load()
    ddata = dweight = None
    with _on(weight):
        tail = (rows, e, n, k, _stream())
        if wanted[0]:
            ddata = torch.empty((rows, k), dtype=dt, device=weight.device)
            check(L.unit_grouped_dense_grad_data(grad.data_ptr(), weight.data_ptr(), sizes.data_ptr(), sizes.element_size(), ddata.data_ptr(),
                                                 _CODE[weight.dtype], _CODE[dt], *tail))
        if wanted[1]:
            if isinstance(data, Mxfp8Tensor):
                data = dequantize_mxfp8(data, _NAME[weight.dtype])
            dweight = torch.empty((e, n, k), dtype=wdt, device=weight.device)
            check(L.unit_grouped_dense_grad_weight(data.data_ptr(), grad.data_ptr(), sizes.data_ptr(), sizes.element_size(), dweight.data_ptr(),
                                                   _CODE[weight.dtype], _CODE[wdt], *tail))
    return ddata, dweight
