"""What layerNorm, dropout and gatedMatMul decide on the host -- which views are taken as they lie, which arguments are refused, what
reaches the C ABI -- against a library that only records its calls (no GPU)."""
import ctypes as C

import numpy as np
import pytest

from neureka_amd import HipDevice, IllegalArgumentException, IllegalStateException, NDConfiguration, Tensor
from neureka_amd import device as device_module
from neureka_amd.ndim import Layout


class Recorder:
    """Entry points that do nothing but note their arguments; nk_alloc hands out distinct addresses."""

    def __init__(self):
        self.calls, self.next = [], 1 << 20

    def __getattr__(self, name):
        def call(*args):
            if name == "nk_alloc":
                C.cast(args[2], C.POINTER(C.c_uint64))[0] = self.next
                self.next += (int(args[1]) + 4095) & ~4095
            elif name not in ("nk_free", "nk_fill", "nk_h2d", "nk_d2h"):
                self.calls.append((name, args))
            return 0
        return call

    def last(self, name):
        found = [args for n, args in self.calls if n == name]
        assert found, f"{name} was not called"
        return found[-1]


def recording_device():
    dev = HipDevice.__new__(HipDevice)
    dev._lib, dev.handle, dev.index, dev._disposed, dev._data_objects, dev._stored = Recorder(), 1, 0, False, 0, {}
    return dev


@pytest.fixture
def dev():
    return recording_device()


def on(dev, shape, dtype=np.float32):
    return Tensor.of(dtype, shape, np.zeros(shape, dtype)).to(dev)


def test_which_views_are_rows():
    t = NDConfiguration.ofShape((4, 6))
    assert t.asRows() == (0, 4, 6, 6) and t.asDense() == 0
    assert NDConfiguration.ofShape((2, 3, 5)).asRows() == (0, 6, 5, 5)
    assert NDConfiguration.ofShape((7,)).asRows() == (0, 1, 7, 7)
    assert t.sliced((4, 3), (0, 2), (1, 1)).asRows() == (2, 4, 3, 6) and t.sliced((4, 3), (0, 2), (1, 1)).asDense() is None
    assert t.sliced((2, 6), (1, 0), (1, 1)).asRows() == (6, 2, 6, 6) and t.sliced((2, 6), (1, 0), (1, 1)).asDense() == 6
    assert t.sliced((2, 6), (0, 0), (2, 1)).asRows() == (0, 2, 6, 12)                       # every second row
    assert t.sliced((4, 3), (0, 0), (1, 2)).asRows() is None                                # every second column
    assert t.sliced((1, 3), (2, 1), (1, 1)).asRows() == (13, 1, 3, 3) and t.sliced((1, 3), (2, 1), (1, 1)).asDense() == 13
    assert t.newReshaped((1, 0)).asRows() is None
    assert NDConfiguration.ofShape((4, 6, 5)).sliced((4, 3, 5), (0, 0, 0), (1, 1, 1)).asRows() is None     # rows at two different steps
    assert NDConfiguration.virtualOf((4, 6)).asRows() is None and NDConfiguration.virtualOf((4, 6)).asDense() is None
    assert NDConfiguration.ofShape((4, 6), Layout.COLUMN_MAJOR).asDense() is None


def test_which_matrices_are_dense_by_columns():
    t = NDConfiguration.ofShape((4, 6))
    assert t.asDenseColumns() is None and t.newReshaped((1, 0)).asDenseColumns() == 0
    assert NDConfiguration.ofShape((4, 6), Layout.COLUMN_MAJOR).asDenseColumns() == 0
    assert NDConfiguration.ofShape((4, 1)).asDenseColumns() == 0 and NDConfiguration.ofShape((1, 4)).asDenseColumns() == 0
    assert NDConfiguration.ofShape((2, 3, 4)).asDenseColumns() is None and NDConfiguration.virtualOf((4, 6)).asDenseColumns() is None


def test_norm_passes_a_slice_by_its_pitch(dev):
    t = on(dev, (5, 10))
    gain = on(dev, (4,))
    t[1:4, 3:7].layerNorm(gain, gain, 0.5)
    args = dev._lib.last("nk_layer_norm")
    assert args[1:6] == (0, 3, 4, t._data.ptr + 13 * 4, 10) and args[6] == args[7] == gain._data.ptr and args[8] == 0.5 and args[10:] == (0, 0)
    assert not [n for n, _ in dev._lib.calls if n == "nk_activation"]                       # nothing was copied
    t[0:5, 0:10:2].layerNorm(on(dev, (5,)), on(dev, (5,)))
    assert [n for n, _ in dev._lib.calls if n == "nk_activation"]


def test_norm_keeps_statistics_only_for_a_graph(dev):
    x, gain, bias = on(dev, (3, 8)), on(dev, (8,)), on(dev, (1, 8))
    x.layerNorm(gain, bias)
    assert dev._lib.last("nk_layer_norm")[10:] == (0, 0)
    bias.setRqsGradient(True)
    y = x.layerNorm(gain, bias)
    mean, rstd = dev._lib.last("nk_layer_norm")[10:]
    assert mean and rstd
    y.backward(1.0)
    args = dev._lib.last("nk_layer_norm_backward")
    assert args[7:9] == (mean, rstd) and args[10:12] == (0, 0) and args[12] == bias.gradient._data.ptr
    assert x.gradient is None and gain.gradient is None and bias.gradient.shape == (1, 8)


def test_gated_layouts_that_reach_the_library(dev):
    x, w, v = on(dev, (2, 3, 8)), on(dev, (8, 5)), on(dev, (5, 8))
    assert x.gatedMatMul(w, w).shape == (2, 3, 5)
    assert dev._lib.last("nk_gated_matmul")[1:10] == (13, 0, 0, 6, 8, 5, x._data.ptr, w._data.ptr, w._data.ptr)
    x.gatedMatMul(v.T(), v.T(), "gelu")
    assert dev._lib.last("nk_gated_matmul")[1:10] == (6, 0, 1, 6, 8, 5, x._data.ptr, v._data.ptr, v._data.ptr)
    copies = len([n for n, _ in dev._lib.calls if n == "nk_activation"])
    x.gatedMatMul(w, v.T())                                                                 # one of each: copied to rows
    assert dev._lib.last("nk_gated_matmul")[3] == 0 and len([n for n, _ in dev._lib.calls if n == "nk_activation"]) == copies + 1


def test_refusals_reach_no_kernel(dev):
    x, w, gain = on(dev, (4, 6)), on(dev, (6, 5)), on(dev, (6,))
    refused = [lambda: x.layerNorm(on(dev, (5,)), gain), lambda: x.layerNorm(gain, on(dev, (6,), np.float64)), lambda: x.layerNorm(gain, gain, -1.0),
               lambda: x.layerNorm(gain, gain, float("nan")), lambda: x.dropout(1.1, 0), lambda: x.dropout(float("nan"), 0), lambda: x.dropout(0.5, -1),
               lambda: x.dropout(0.5, 1 << 64), lambda: x.dropout(0.5, 0, 1 << 64), lambda: x.gatedMatMul(w, on(dev, (6, 4))), lambda: x.gatedMatMul(on(dev, (5, 6)), on(dev, (5, 6))),
               lambda: x.gatedMatMul(w, w, "exp"), lambda: x.gatedMatMul(w, on(dev, (6, 5), np.float64)),
               lambda: on(dev, (4, 6), np.int32).layerNorm(on(dev, (6,), np.int32), on(dev, (6,), np.int32)), lambda: on(dev, (4,), np.int64).dropout(0.5, 0),
               lambda: dev.launch_layer_norm(x[0:4, 0:3], on(dev, (4, 3)), on(dev, (3,)), on(dev, (3,))),                  # a drain that is not dense
               lambda: dev.launch_gated_matmul("silu", on(dev, (4, 5)), x.T().T()[0:4, 0:6:2], on(dev, (3, 5)), on(dev, (3, 5)))]
    for call in refused:
        with pytest.raises(IllegalArgumentException):
            call()
    with pytest.raises(IllegalArgumentException):
        from neureka_amd import execute
        execute("dropout", [x], d=0)
    assert not [n for n, _ in dev._lib.calls if n.startswith(("nk_layer", "nk_dropout", "nk_gated"))]


def test_tensors_of_another_device_are_refused(dev):
    other = recording_device()
    x, gain, w = on(dev, (4, 6)), on(other, (6,)), on(other, (6, 6))
    for call in (lambda: x.layerNorm(gain, gain), lambda: x.gatedMatMul(w, w), lambda: dev.launch_dropout(on(other, (4, 6)), x, 0.5, 1),
                 lambda: dev.launch_layer_norm(on(dev, (4, 6)), x, gain, gain), lambda: dev.launch_gated_matmul("silu", on(dev, (4, 6)), x, w, w)):
        with pytest.raises(IllegalStateException):
            call()
    assert not [n for n, _ in dev._lib.calls + other._lib.calls if n.startswith(("nk_layer", "nk_dropout", "nk_gated"))]


def test_an_error_of_another_shape_or_type_is_refused(dev):
    y = on(dev, (4, 6)).setRqsGradient(True).gatedMatMul(on(dev, (6, 5)), on(dev, (6, 5)))
    for bad in (on(dev, (4, 6)), on(dev, (4, 5), np.float64)):
        with pytest.raises(IllegalArgumentException):
            y.backward(bad)


def test_the_recorder_stands_for_the_real_table():
    """Every entry point used here exists with that many arguments."""
    from neureka_amd import _lib
    for name, count in (("nk_layer_norm", 12), ("nk_layer_norm_backward", 13), ("nk_dropout", 11), ("nk_gated_matmul", 13), ("nk_gated_matmul_backward", 16)):
        assert len(_lib.SYMBOLS[name][1]) == count
    assert device_module.HipDevice.GATED_ACTIVATIONS == ("idy", "relu", "sig", "silu", "gelu", "tanh")
