"""What the C ABI of the gated products and of MXFP8 refuses before anything touches a device, its size formulas, and what the Python
operators refuse on the CPU."""
import ctypes

import pytest
import torch

import unit_amd as U
from unit_amd import gated as G


@pytest.fixture(scope="module")
def L():
    from unit_amd import _lib
    return _lib.load()


def said(L, rc, text):
    assert rc == -1 and text in L.unit_last_error().decode(), (rc, L.unit_last_error())


def test_mxfp8_buffers(L):
    c, s = ctypes.c_size_t(), ctypes.c_size_t()
    for rows, k in ((0, 1), (1, 1), (3, 32), (3, 33), (1 << 20, 4096), (1 << 30, 100)):
        assert L.unit_mxfp8_bytes(rows, k, ctypes.byref(c), ctypes.byref(s)) == 0
        assert (c.value, s.value) == (rows * -(-k // 32) * 32, rows * -(-k // 32))
    said(L, L.unit_mxfp8_bytes(-1, 5, ctypes.byref(c), ctypes.byref(s)), "must not be negative")
    said(L, L.unit_mxfp8_bytes(5, 0, ctypes.byref(c), ctypes.byref(s)), "must be positive")
    said(L, L.unit_mxfp8_bytes(1 << 40, 1 << 20, ctypes.byref(c), ctypes.byref(s)), "elements")
    said(L, L.unit_mxfp8_bytes(4, 4, None, ctypes.byref(s)), "null")


def test_mxfp8_arguments(L):
    said(L, L.unit_quantize_mxfp8(16, 3, 4, 64, 16, 16, None), "dtype")
    said(L, L.unit_quantize_mxfp8(None, 0, 4, 64, 16, 16, None), "null")
    said(L, L.unit_quantize_mxfp8(16, 0, 4, 64, 16, None, None), "null")
    said(L, L.unit_quantize_mxfp8(16, 0, 4, 64, 8, 16, None), "aligned")
    said(L, L.unit_quantize_mxfp8(17, 1, 4, 64, 16, 16, None), "aligned to its elements")
    said(L, L.unit_dequantize_mxfp8(16, 16, 4, 64, 8, 0, None), "aligned")
    said(L, L.unit_dequantize_mxfp8(16, 16, 4, 64, 16, 7, None), "dtype")


def test_gated_arguments(L):
    ok = dict(x=16, w=16, sizes=16, size_bytes=4, out=16, dtype=1, out_dtype=0, act=0, pre=None, pre_scales=None, pre_dtype=0, rows=4, groups=2, n=16, k=16, stream=None)
    call = lambda **change: L.unit_gated_dense(*{**ok, **change}.values())
    for change, text in ((dict(x=None), "null"), (dict(w=None), "null"), (dict(out=None), "null"), (dict(sizes=None), "null"), (dict(size_bytes=2), "4- or 8-byte"),
                         (dict(sizes=12, size_bytes=8), "aligned"), (dict(x=8), "aligned"), (dict(w=8), "aligned"), (dict(out=8), "aligned"), (dict(dtype=0), "dtype"),
                         (dict(dtype=3), "dtype"), (dict(out_dtype=2), "out_dtype"), (dict(act=2), "activation"), (dict(act=-1), "activation"),
                         (dict(pre=16, pre_dtype=2), "pre_dtype"), (dict(pre=16, pre_dtype=3), "pre_dtype"), (dict(pre=16, pre_dtype=4), "null"),
                         (dict(pre=8, pre_dtype=1), "aligned"), (dict(rows=-1), "not negative"), (dict(groups=0), "positive"), (dict(n=12), "multiples of 8"),
                         (dict(k=4), "multiples of 8"), (dict(n=1 << 16, k=1 << 15), "2^31"), (dict(n=1 << 22), "2^21"), (dict(groups=1 << 21), "2^20")):
        said(L, call(**change), text)


def test_gated_mxfp4_arguments(L):
    ok = dict(x=16, xs=None, x_dtype=1, wc=16, ws=16, sizes=None, size_bytes=4, out=16, out_dtype=0, act=1, rows=4, groups=1, n=8, k=64, work=16, bytes=1 << 20, stream=None)
    call = lambda **change: L.unit_gated_dense_mxfp4(*{**ok, **change}.values())
    for change, text in ((dict(bytes=16), "needed"), (dict(work=None), "null"), (dict(x=None), "null"), (dict(x_dtype=3), "null"), (dict(x_dtype=4), "x_dtype"),
                         (dict(out_dtype=3), "out_dtype"), (dict(act=7), "activation"), (dict(rows=-1), "not negative"), (dict(n=0), "positive"), (dict(out=8), "aligned"),
                         (dict(n=1 << 20, k=1 << 13), "2^31"), (dict(groups=2), "null"), (dict(wc=None), "null"), (dict(ws=None), "null")):
        said(L, call(**change), text)


def test_gated_gradient_arguments(L):
    need = ctypes.c_size_t()
    assert L.unit_gated_dense_grad_ws_bytes(1, 1, 4, 2, 16, 16, ctypes.byref(need)) == 0 and need.value == 256
    assert L.unit_gated_dense_grad_ws_bytes(4, 2, 1000, 2, 24, 40, ctypes.byref(need)) == 0 and need.value == 1000 * 96 + 80128  # parts begin on 256 bytes
    # one group of many rows and a small weight: float32 sums of the parts that its rows are shared out to
    assert L.unit_gated_dense_grad_ws_bytes(1, 1, 10000, 1, 64, 64, ctypes.byref(need)) == 0 and need.value > 10000 * 256 and (need.value - 10000 * 256) % (64 * 64 * 8) == 0
    assert L.unit_gated_dense_grad_ws_bytes(1, 1, 0, 2, 16, 16, ctypes.byref(need)) == 0 and need.value == 0
    said(L, L.unit_gated_dense_grad_ws_bytes(2, 1, 4, 2, 16, 16, ctypes.byref(need)), "x_dtype")
    said(L, L.unit_gated_dense_grad_ws_bytes(1, 1, 4, 2, 16, 16, None), "null")
    ok = dict(x=16, x_scales=None, x_dtype=1, w=16, dh=16, pre=16, pre_scales=None, pre_dtype=1, sizes=16, size_bytes=4, dx=16, dx_dtype=0, dw=16, dw_dtype=1, dtype=1,
              act=0, rows=4, groups=2, n=16, k=16, ws=16, bytes=1 << 20, stream=None)
    call = lambda **change: L.unit_gated_dense_grad(*{**ok, **change}.values())
    for change, text in ((dict(x=None), "null"), (dict(w=None), "null"), (dict(dh=None), "null"), (dict(ws=None), "null"), (dict(sizes=None), "null"),
                         (dict(pre=None, x=None, dw=None), "null"), (dict(x_dtype=4), "null"), (dict(pre_dtype=4), "null"), (dict(x_dtype=2), "x_dtype"),
                         (dict(pre_dtype=2), "pre_dtype"), (dict(dtype=0, x_dtype=0), "dtype"), (dict(dx_dtype=2), "dx"), (dict(dw_dtype=2), "dw"), (dict(act=2), "activation"),
                         (dict(rows=-1), "negative"), (dict(groups=0), "positive"), (dict(n=12), "multiples of 8"), (dict(k=12), "multiples of 8"), (dict(n=1 << 22), "2^21"),
                         (dict(n=1 << 16, k=1 << 15), "2^31"), (dict(bytes=100), "needed"), (dict(size_bytes=3), "4- or 8-byte"), (dict(x=8), "aligned"), (dict(w=8), "aligned"),
                         (dict(dh=8), "aligned"), (dict(pre=8), "aligned"), (dict(dx=8), "aligned"), (dict(dw=8), "aligned"), (dict(ws=8), "aligned")):
        said(L, call(**change), text)


def test_operators_refuse_by_name_before_they_look_for_a_gpu():
    x, w = torch.zeros((4, 64), dtype=torch.float16), torch.zeros((80, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="activation: expected"):
        U.gated_dense(x, w, activation="relu")
    with pytest.raises(ValueError, match="activation: expected"):
        U.gated_dense(x, w, activation=["silu"])
    with pytest.raises(ValueError, match="keep: expected"):
        U.gated_dense(x, w, keep="mxfp4")
    with pytest.raises(ValueError, match="out_dtype: expected"):
        U.gated_dense_mxfp4(x, w, out_dtype="half")
    with pytest.raises(ValueError, match="weight_out_dtype: expected"):
        U.gated_dense_grad(x, w, x, weight_out_dtype=None)
    for call in (lambda: U.gated_dense(x, w), lambda: U.gated_dense_grad(x, w, x[:, :40]), lambda: U.quantize_mxfp8(x)):
        with pytest.raises(ValueError, match="must live on the GPU"):
            call()
    with pytest.raises(TypeError, match="torch.Tensor"):
        U.quantize_mxfp8([1.0])
    with pytest.raises(TypeError, match="Mxfp4Tensor"):
        U.gated_dense_mxfp4(x, w)
    assert set(G._ACTIVATION) == {"silu", "gelu_tanh"}
