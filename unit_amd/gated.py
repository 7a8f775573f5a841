"""Gated feed-forward products, h = act(gate . x) * (up . x): operators on torch tensors that live on the MI355X, in the manner of
grouped.py, whose products by expert they extend.  No counterpart in the reference.

  gated_dense         both projections, the activation and the product in one kernel; dense, or rows sorted by expert
  gated_dense_mxfp4   the same with MXFP4 operands
  gated_dense_grad    the gradients, from what gated_dense kept (16 bits, or MXFP8) or from the rows alone

A weight holds gate's N rows, then up's: (2 N, K), or (E, 2 N, K) by expert.
"""
import ctypes

import torch

from . import _lib
from ._lib import check
from .grouped import _CODE, _HALVES, _MXFP4, _MXFP8, Mxfp4Tensor, Mxfp8Tensor, _floats, _mxfp4, _mxfp8_empty, _native_gated, _on, _out_dtype, _same_device, _sizes
from .ops import _dev, _stream

__all__ = ["gated_dense", "gated_dense_mxfp4", "gated_dense_grad"]

_ACTIVATION = {"silu": 0, "gelu_tanh": 1}


def _activation(name):
    try:
        return _ACTIVATION[name]
    except (KeyError, TypeError):
        raise ValueError(f"activation: expected 'silu' or 'gelu_tanh', got {name!r}") from None


def _gated(data, weight, group_sizes, read=True):
    """data, weight, the groups as the library takes them, (rows, groups, N, K); read: the rows' elements are, not their shape alone"""
    if not isinstance(data, Mxfp8Tensor) and read:
        data = _floats(data, "data", _HALVES, 2)
    weight = _floats(weight, "weight", _HALVES, 2 if group_sizes is None else 3)
    if not isinstance(data, Mxfp8Tensor) and weight.dtype != data.dtype:
        raise TypeError(f"weight: expected dtype {data.dtype}, got {weight.dtype}")
    _same_device(weight, "weight", data)
    e, sizes = _groups(weight, group_sizes, data)
    n2, k = weight.shape[-2:]
    if n2 % 2:
        raise ValueError(f"weight: expected as many rows of the gate as of the up projection, got {n2} in all")
    if len(data.shape) != 2 or data.shape[1] != k:
        raise ValueError(f"data: expected (rows, {k}), got {tuple(data.shape)}")
    return data, weight, sizes, (data.shape[0], e, n2 // 2, k)


def _groups(weight, group_sizes, data):
    if group_sizes is None:
        return 1, None
    sizes = _sizes(group_sizes, data)
    if sizes.shape[0] != weight.shape[0]:
        raise ValueError(f"group_sizes: expected {weight.shape[0]} entries, got {sizes.shape[0]}")
    return weight.shape[0], sizes


def _group_args(sizes):
    return (None, 4) if sizes is None else (sizes.data_ptr(), sizes.element_size())


def gated_dense(data, weight, group_sizes=None, activation="silu", out_dtype="float32", keep=None):
    """out[r] = act(gate . data[r]) * (up . data[r]), (rows, N), in one kernel: sums, activation and product in float32, rounded once.

    data (rows, K) float16 or bfloat16; weight (2 N, K) of the same type, gate's rows first, N and K multiples of 8; with group_sizes
    (E,), weight (E, 2 N, K) and rows sorted by expert as in grouped_dense (rows of no expert give zeros).
    activation "silu", z / (1 + exp(-z)), or "gelu_tanh", z (1 + tanh(sqrt(2 / pi) (z + 0.044715 z^3))) / 2.
    keep: what comes back beside out for gated_dense_grad's `pre`, gate . data[r] and up . data[r] as (rows, 2, N): "pre" a tensor of
    data's type, "mxfp8" an Mxfp8Tensor, a quarter of a float32's size; None nothing, and out alone is returned.  out is the same to the bit."""
    done = _native_gated.gated(data, weight, group_sizes, activation, out_dtype, keep)
    if done is not None:
        return done
    act, dt = _activation(activation), _out_dtype(out_dtype)
    if keep not in (None, "pre", "mxfp8"):
        raise ValueError(f"keep: expected None, 'pre' or 'mxfp8', got {keep!r}")
    data, weight, sizes, (rows, e, n, k) = _gated(_tensor(data), weight, group_sizes)
    with _on(data):
        out = torch.empty((rows, n), dtype=dt, device=data.device)
        pre = _forward(data, weight, sizes, act, (rows, e, n, k), out, keep)
    return out if keep is None else (out, pre)


def _tensor(data):
    if isinstance(data, Mxfp8Tensor):
        raise TypeError("data: expected a torch.Tensor, got Mxfp8Tensor (which gated_dense_grad takes)")
    return data


def _forward(data, weight, sizes, act, shape, out, keep):
    rows, e, n, k = shape
    pre, kept = None, (None, None, 0)
    if keep == "pre":
        pre = torch.empty((rows, 2, n), dtype=data.dtype, device=data.device)
        kept = pre.data_ptr(), None, _CODE[data.dtype]
    elif keep == "mxfp8":
        pre = _mxfp8_empty((rows, 2, n), data.device)
        kept = *pre._pointers()[:2], _MXFP8
    check(_lib.load().unit_gated_dense(data.data_ptr(), weight.data_ptr(), *_group_args(sizes), out.data_ptr(), _CODE[data.dtype], _CODE[out.dtype], act,
                                       *kept, rows, e, n, k, _stream()))
    return pre


def gated_dense_mxfp4(data, weight, group_sizes=None, activation="silu", out_dtype="float32"):
    """gated_dense with MXFP4 operands: data (rows, K) float32, float16 or bfloat16, quantised on the way as quantize_mxfp4 does, or an
    Mxfp4Tensor; weight an Mxfp4Tensor (2 N, K), with group_sizes (E, 2 N, K); N and K of any size."""
    out = _native_gated.gated_mx(data, weight, group_sizes, activation, out_dtype)
    if out is not None:
        return out
    act, dt = _activation(activation), _out_dtype(out_dtype)
    ndim = 2 if group_sizes is None else 3
    if len(_mxfp4(weight, "weight").shape) != ndim:
        raise ValueError(f"weight: expected {ndim} axes, got shape {weight.shape}")
    n2, k = weight.shape[-2:]
    if n2 % 2:
        raise ValueError(f"weight: expected as many rows of the gate as of the up projection, got {n2} in all")
    quantised = isinstance(data, Mxfp4Tensor)
    if not quantised:
        data = _floats(data, "data", tuple(_CODE), 2)
    if len(data.shape) != 2 or data.shape[1] != k:
        raise ValueError(f"data: expected (rows, {k}), got {tuple(data.shape)}")
    _same_device(weight, "weight", data)
    e, sizes = _groups(weight, group_sizes, data)
    rows, L = data.shape[0], _lib.load()
    with _on(weight.buf):
        if quantised:
            operand, work = (*data._pointers()[:2], _MXFP4), (None, 0)
        else:
            need = ctypes.c_size_t()
            check(L.unit_mxfp4_workspace_bytes(rows, k, ctypes.byref(need)))
            ws = torch.empty((need.value,), dtype=torch.uint8, device=data.device)
            operand, work = (data.data_ptr(), None, _CODE[data.dtype]), (ws.data_ptr(), ws.numel())
        out = torch.empty((rows, n2 // 2), dtype=dt, device=weight.device)
        check(L.unit_gated_dense_mxfp4(*operand, *weight._pointers()[:2], *_group_args(sizes), out.data_ptr(), _CODE[dt], act, rows, e, n2 // 2, k, *work,
                                       _stream()))
    return out


def gated_dense_grad(data, weight, grad, group_sizes=None, activation="silu", pre=None, out_dtype="float32", weight_out_dtype="float32"):
    """The gradients of gated_dense for grad (rows, N), of weight's type: (ddata (rows, K), dweight of weight's shape), in out_dtype and
    weight_out_dtype, zero in rows of no expert and for experts without rows.

    data as in gated_dense, or an Mxfp8Tensor of it; pre what gated_dense kept (either form), or None: the pre-activations are then
    computed from data again.  The gate's own gradients, grad * up * act'(gate) and grad * act(gate), are computed in float32 and
    rounded to weight's type, which the products after them take; those sum in float32 and round once."""
    both = _native_gated.gated_grad(data, weight, grad, group_sizes, activation, pre, out_dtype, weight_out_dtype)
    return _gated_grad(data, weight, grad, group_sizes, activation, pre, out_dtype, weight_out_dtype) if both is None else both


def _gated_grad(data, weight, grad, group_sizes, activation, pre, out_dtype, weight_out_dtype, wanted=(True, True)):
    """(ddata, dweight), None in the place of one that is not wanted"""
    act, dt, wdt = _activation(activation), _out_dtype(out_dtype), _out_dtype(weight_out_dtype, "weight_out_dtype")
    read = wanted[1] or pre is None  # dx from kept pre-activations takes nothing from the rows
    data, weight, sizes, (rows, e, n, k) = _gated(data, weight, group_sizes, read)
    grad = _dev(grad, "grad", weight.dtype, 2)
    _same_device(grad, "grad", weight)
    if tuple(grad.shape) != (rows, n):
        raise ValueError(f"grad: expected ({rows}, {n}), got {tuple(grad.shape)}")
    if pre is not None:
        if not isinstance(pre, Mxfp8Tensor):
            pre = _dev(pre, "pre", weight.dtype, 3)
        if tuple(pre.shape) != (rows, 2, n):
            raise ValueError(f"pre: expected ({rows}, 2, {n}), got {tuple(pre.shape)}")
        _same_device(pre, "pre", weight)
    L, code = _lib.load(), _CODE[weight.dtype]
    x = (None, None, code) if not read else (*data._pointers()[:2], _MXFP8) if isinstance(data, Mxfp8Tensor) else (data.data_ptr(), None, code)
    kept = (None, None, 0) if pre is None else (*pre._pointers()[:2], _MXFP8) if isinstance(pre, Mxfp8Tensor) else (pre.data_ptr(), None, code)
    need = ctypes.c_size_t()
    workspace = L.unit_gated_dense_grad_ws_bytes if all(wanted) else L.unit_gated_dense_grad_one_ws_bytes
    check(workspace(x[2], code, rows, e, n, k, ctypes.byref(need)))
    with _on(weight):
        ws = torch.empty((need.value,), dtype=torch.uint8, device=weight.device)
        ddata = torch.empty((rows, k), dtype=dt, device=weight.device) if wanted[0] else None
        dweight = torch.empty(weight.shape, dtype=wdt, device=weight.device) if wanted[1] else None
        result = lambda t, d: (None, 0) if t is None else (t.data_ptr(), _CODE[d])  # noqa: E731
        check(L.unit_gated_dense_grad(*x, weight.data_ptr(), grad.data_ptr(), *kept, *_group_args(sizes), *result(ddata, dt), *result(dweight, wdt), code, act,
                                      rows, e, n, k, ws.data_ptr(), ws.numel(), _stream()))
    return ddata, dweight
