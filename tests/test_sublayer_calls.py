"""Calls of layerNorm, dropout and gatedMatMul that reach them through `execute`, and errors that come back padded to another rank,
against a library that only records its calls (no GPU)."""
import numpy as np
import pytest

from neureka_amd import IllegalArgumentException, execute
from test_sublayer_host import on, recording_device


@pytest.fixture
def dev():
    return recording_device()


def test_execute_fills_in_what_the_methods_fill_in(dev):
    x, g, w = on(dev, (4, 6)), on(dev, (6,)), on(dev, (6, 5))
    execute("layerNorm", [x, g, g])
    assert dev._lib.last("nk_layer_norm")[8] == 1e-5
    execute("gatedMatMul", [x, w, w])
    assert dev._lib.last("nk_gated_matmul")[1] == 13                          # silu, as Tensor.gatedMatMul
    execute("dropout", [x], args={"probability": 0.5, "seed": 3})
    assert dev._lib.last("nk_dropout")[7:10] == (0.5, 3, 0)


@pytest.mark.parametrize("op,count,args", [("dropout", 1, {}), ("dropout", 1, {"probability": 0.5}), ("dropout", 1, {"seed": 1}), ("dropout", 2, {"probability": 0.5, "seed": 1}),
                                           ("layerNorm", 1, {}), ("layerNorm", 2, {}), ("layerNorm", 4, {}), ("layerNorm", 3, {"eps": 1e-5}), ("gatedMatMul", 2, {}),
                                           ("gatedMatMul", 3, {"activation": "silu", "keep": True})])
def test_execute_refuses_operands_and_arguments_that_do_not_fit(dev, op, count, args):
    operands = [on(dev, (6, 6)) for _ in range(count)]
    with pytest.raises(IllegalArgumentException):
        execute(op, operands, args=args)
    assert not [n for n, _ in dev._lib.calls if n.startswith(("nk_layer", "nk_dropout", "nk_gated"))]


@pytest.mark.parametrize("padded", [(1, 4, 6), (4, 6, 1), (1, 1, 4, 6), (4, 1, 6)])
def test_an_error_padded_to_another_rank_is_taken(dev, padded):
    """An operand of lower rank is padded with axes of one element, and its error comes back in that shape: the same rows."""
    g, w = on(dev, (6,)), on(dev, (6, 6))
    for entry, at, f in (("nk_layer_norm_backward", 9, lambda x: x.layerNorm(g, g)), ("nk_dropout", 5, lambda x: x.dropout(0.5, 1)),
                         ("nk_gated_matmul_backward", 12, lambda x: x.gatedMatMul(w, w))):
        x, error = on(dev, (4, 6)).setRqsGradient(True), on(dev, padded)
        f(x).backward(error)
        assert x.gradient.shape == (4, 6) and dev._lib.last(entry)[at] == error._data.ptr
    x = on(dev, (4, 6)).setRqsGradient(True)
    (x.layerNorm(g, g) * on(dev, (1, 4, 6))).backward(1.0)                    # as a residual stream with a batch axis has it
    assert x.gradient.shape == (4, 6)


def test_a_padded_error_may_be_a_view(dev):
    g = on(dev, (6,))
    x, wide = on(dev, (4, 6)).setRqsGradient(True), on(dev, (1, 4, 9))
    x.layerNorm(g, g).backward(wide[0:1, 0:4, 2:8])
    assert x.gradient.shape == (4, 6)


@pytest.mark.parametrize("other", [(4, 5), (6, 4), (2, 4, 6), (24,), (2, 2, 6), (1, 6, 4), (1, 24)])
def test_errors_of_other_shapes_stay_refused(dev, other):
    g = on(dev, (6,))
    y = on(dev, (4, 6)).setRqsGradient(True).layerNorm(g, g)
    with pytest.raises(IllegalArgumentException):
        y.backward(on(dev, other))
