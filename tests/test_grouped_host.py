"""What the C ABI of the grouped and MXFP4 products refuses before anything touches a device, and its size formulas."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def L():
    from unit_amd import _lib
    return _lib.load()


def said(L, rc, text):
    assert rc == -1 and text in L.unit_last_error().decode(), (rc, L.unit_last_error())


def test_mxfp4_buffers(L):
    c, s = ctypes.c_size_t(), ctypes.c_size_t()
    for rows, k in ((0, 1), (1, 1), (3, 256), (3, 257), (1 << 20, 4096)):
        assert L.unit_mxfp4_bytes(rows, k, ctypes.byref(c), ctypes.byref(s)) == 0
        stages = -(-k // 256)
        assert (c.value, s.value) == (rows * stages * 128, rows * stages * 8 + 1024)
        if rows < 1 << 20:
            assert L.unit_mxfp4_workspace_bytes(rows, k, ctypes.byref(c)) == 0 and c.value == rows * stages * 136 + 1024
    said(L, L.unit_mxfp4_bytes(-1, 5, ctypes.byref(c), ctypes.byref(s)), "must not be negative")
    said(L, L.unit_mxfp4_bytes(5, 0, ctypes.byref(c), ctypes.byref(s)), "must be positive")
    said(L, L.unit_mxfp4_bytes(1 << 40, 1 << 20, ctypes.byref(c), ctypes.byref(s)), "elements")
    said(L, L.unit_mxfp4_workspace_bytes(4, 4, None), "not null")


def test_mxfp4_arguments(L):
    said(L, L.unit_quantize_mxfp4(16, 3, 4, 64, 16, 16, None), "dtype")
    said(L, L.unit_quantize_mxfp4(None, 0, 4, 64, 16, 16, None), "null")
    said(L, L.unit_quantize_mxfp4(16, 0, 4, 64, 8, 16, None), "aligned")
    said(L, L.unit_quantize_mxfp4(18, 0, 4, 64, 16, 16, None), "aligned to its elements")
    said(L, L.unit_dequantize_mxfp4(16, 16, 4, 64, 8, 0, None), "aligned")
    said(L, L.unit_dequantize_mxfp4(16, 16, 4, 64, 16, 7, None), "dtype")
    said(L, L.unit_prepare_mxfp4(16, None, 4, 64, 16, 16, None), "null")
    ok = [16, None, 1, 16, 16, 16, 0, 4, 8, 64, 16, 1 << 20, None]

    def dense(**change):
        names = "x xs x_dtype wc ws out out_dtype m n k work bytes stream".split()
        return L.unit_dense_mxfp4(*[change.get(n, v) for n, v in zip(names, ok)])
    said(L, dense(bytes=16), "needed")
    said(L, dense(work=None), "null")
    said(L, dense(x_dtype=3), "null")
    said(L, dense(x_dtype=4), "x_dtype")
    said(L, dense(out_dtype=3), "out_dtype")
    said(L, dense(m=-1), "not negative")
    said(L, dense(n=0), "positive")
    said(L, dense(out=8), "aligned")
    said(L, dense(n=1 << 22, k=1 << 12), "2^31")


def test_grouped_arguments(L):
    for f in (L.unit_grouped_dense, L.unit_grouped_dense_grad_data, L.unit_grouped_dense_grad_weight):
        ok = dict(a=16, b=16, sizes=16, size_bytes=4, out=16, dtype=1, out_dtype=0, rows=4, groups=2, n=16, k=16, stream=None)
        call = lambda **change: f(*{**ok, **change}.values())
        for change, text in ((dict(a=None), "null"), (dict(b=None), "null"), (dict(sizes=None), "null"), (dict(out=None), "null"), (dict(size_bytes=2), "4- or 8-byte"),
                             (dict(sizes=12, size_bytes=8), "aligned"), (dict(a=8), "aligned"), (dict(b=8), "aligned"), (dict(out=8), "aligned"), (dict(dtype=0), "dtype"),
                             (dict(dtype=3), "dtype"), (dict(out_dtype=3), "out_dtype"), (dict(rows=-1), "not negative"), (dict(groups=0), "positive"),
                             (dict(n=12), "multiples of 8"), (dict(k=4), "multiples of 8"), (dict(n=1 << 16, k=1 << 16), "2^31"), (dict(groups=1 << 21), "2^20")):
            said(L, call(**change), text)
