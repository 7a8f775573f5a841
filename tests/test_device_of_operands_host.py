"""The expert and MXFP4 operators on operands of another device than the current one: everything that they launch runs with the operands' device as
the current one, on that device's stream, so that the steps of one operator, and those of the layer, are ordered.  On the CPU, with the library's
launches, the streams and the change of device noted in the place of being done."""
import contextlib

import pytest
import torch

import unit_amd as U
from unit_amd import _lib, gated, grouped

SIZES = ("unit_mxfp4_bytes", "unit_mxfp8_bytes", "unit_mxfp4_workspace_bytes", "unit_gated_dense_grad_ws_bytes", "unit_gated_dense_grad_one_ws_bytes")


@pytest.fixture
def noted(monkeypatch):
    """(launches: name and the tensor whose device is current), streams asked for with no such tensor"""
    real, current, launches, stray = _lib.load(), [None], [], []

    class Library:
        def __getattr__(self, name):
            if name in SIZES:
                return getattr(real, name)
            return lambda *args: launches.append((name, current[-1])) or 0

    @contextlib.contextmanager
    def on(t):
        current.append(t)
        yield
        current.pop()

    def stream():
        if current[-1] is None:
            stray.append(1)
        return None

    class Declined:
        def __getattr__(self, name):
            return lambda *args: None

    library = Library()
    monkeypatch.setattr(_lib, "load", lambda: library)
    for module in (grouped, gated):
        monkeypatch.setattr(module, "_on", on)
        monkeypatch.setattr(module, "_stream", stream)
        monkeypatch.setattr(module, "_dev", lambda t, name, dtype=None, ndim=None: t.contiguous())
    monkeypatch.setattr(grouped, "_native", Declined())
    monkeypatch.setattr(grouped, "_native_gated", Declined())
    monkeypatch.setattr(gated, "_native_gated", Declined())
    return launches, stray


def calls():
    x, w, dy = (torch.zeros(s, dtype=torch.bfloat16) for s in ((5, 64), (3, 32, 64), (5, 32)))
    sizes, codes, scales = torch.tensor([2, 0, 3]), torch.zeros((3, 32, 32), dtype=torch.uint8), torch.zeros((3, 32, 2), dtype=torch.uint8)
    w4 = lambda: U.prepare_mxfp4_weight(codes, scales)
    one = lambda: U.prepare_mxfp4_weight(codes[0], scales[0])
    return {
        "quantize_mxfp4": lambda: U.quantize_mxfp4(x),
        "dequantize_mxfp4": lambda: U.dequantize_mxfp4(w4()),
        "dense_mxfp4": lambda: U.dense_mxfp4(x, one()),
        "dense_mxfp4 of codes": lambda: U.dense_mxfp4(U.quantize_mxfp4(x), one()),
        "grouped_dense_mxfp4": lambda: U.grouped_dense_mxfp4(x, w4(), sizes),
        "grouped_dense": lambda: U.grouped_dense(x, w, sizes),
        "grouped_dense_grad": lambda: U.grouped_dense_grad(x, w, dy, sizes),
        "grouped_dense_grad of 8 bits": lambda: U.grouped_dense_grad(U.quantize_mxfp8(x), w, dy, sizes),
        "gated_dense": lambda: U.gated_dense(x, w, sizes, keep="pre"),
        "gated_dense_mxfp4": lambda: U.gated_dense_mxfp4(x, w4(), sizes),
        "gated_dense_grad": lambda: U.gated_dense_grad(x, w, dy[:, :16].contiguous(), sizes),
        "mxfp8": lambda: U.dequantize_mxfp8(U.quantize_mxfp8(x)),
    }


@pytest.mark.parametrize("name", calls())
def test_every_launch_runs_on_the_operands_device(noted, name):
    launches, stray = noted
    calls()[name]()
    assert launches and not stray
    assert all(t is not None for _, t in launches), launches
