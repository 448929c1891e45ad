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
