"""The workspace of a gradient of which one operand alone is asked for: its own size, without a device."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def L():
    from unit_amd import _lib
    return _lib.load()


def size(f, *args):
    need = ctypes.c_size_t()
    assert f(*args, ctypes.byref(need)) == 0
    return need.value


@pytest.mark.parametrize("rows,groups,n,k", [(10000, 1, 64, 64), (16384, 1, 512, 512), (4, 2, 16, 16), (1000, 2, 24, 40), (0, 1, 16, 16)])
def test_one_gradient_takes_no_sums(L, rows, groups, n, k):
    lines = lambda b: -(-b // 256) * 256
    dpre = lines(rows * n * 4)
    assert size(L.unit_gated_dense_grad_one_ws_bytes, 1, 1, rows, groups, n, k) == dpre
    assert size(L.unit_gated_dense_grad_one_ws_bytes, 4, 2, rows, groups, n, k) == dpre + lines(rows * k * 2)
    both = size(L.unit_gated_dense_grad_ws_bytes, 1, 1, rows, groups, n, k)
    assert both > dpre if groups == 1 and rows > 4096 else both == dpre


def test_it_refuses_as_the_other_does(L):
    need = ctypes.c_size_t()
    for args, text in (((2, 1, 4, 2, 16, 16), "x_dtype"), ((1, 0, 4, 2, 16, 16), "dtype"), ((1, 1, -1, 2, 16, 16), "negative"), ((1, 1, 4, 2, 12, 16), "multiples of 8")):
        assert L.unit_gated_dense_grad_one_ws_bytes(*args, ctypes.byref(need)) == -1 and text in L.unit_last_error().decode()
    assert L.unit_gated_dense_grad_one_ws_bytes(1, 1, 4, 2, 16, 16, None) == -1
    # a workspace of that size is one for a single gradient only, refused where both are asked for
    for dx, dw, refused in ((16, 16, True), (16, None, False), (None, 16, False)):
        need = size(L.unit_gated_dense_grad_one_ws_bytes, 1, 1, 10000, 1, 64, 64) - (0 if refused else 1)
        assert L.unit_gated_dense_grad(16, None, 1, 16, 16, 16, None, 1, None, 4, dx, 0, dw, 1, 1, 0, 10000, 1, 64, 64, 16, need, None) == -1
        said = L.unit_last_error().decode()
        assert "needed" in said and (f", {need + 1} needed" in said) == (not refused)
