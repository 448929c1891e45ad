"""What the entry points of layerNorm, dropout and gatedMatMul take and refuse, and which kernels a product runs."""
import numpy as np
import pytest

from test_gpu_sublayer import dropped, get, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [np.float32, np.float64])
def test_a_dropout_onto_a_part_of_its_own_source_is_refused(device, dt):
    from neureka_amd import HipError
    x = np.random.default_rng(1).standard_normal((64, 60)).astype(dt)
    t = put(device, x)
    square = t[0:60, 0:60]
    for what, drain, source in (("shifted by a row", t[1:64, 0:60], t[0:63, 0:60]), ("shifted back", t[0:63, 0:60], t[1:64, 0:60]), ("by a column", t[0:64, 1:60], t[0:64, 0:59]),
                                ("transposed", square.T(), square), ("a stride apart", t[0:32, 0:60], t[0:64:2, 0:60]), ("corners", t[0:40, 0:40], t[24:64, 20:60])):
        with pytest.raises(HipError, match="overlaps"):
            device.launch_dropout(drain, source, 0.5, 1)
    assert get(t).tobytes() == x.tobytes()
    (p, _, c), = device._ops(t)
    twice = np.array([64, 60, 60, 0, 60, 1, 0, 0, 1, 1], np.int32)            # shape, strides (the columns all the same element), indices map, offset, spread
    other = put(device, x)
    lib = device._lib
    assert lib.nk_dropout(device.handle, 0 if dt == np.float32 else 1, 2, other._data.ptr, twice.ctypes.data_as(type(c)), p, c, 0.5, 1, 0, 64 * 60) != 0
    assert b"holds one element" in lib.nk_last_error()


def test_a_dropout_between_parts_that_share_nothing_runs(device):
    """Halves, alternating columns, a block and the transpose of its neighbour: in one buffer, with no element in common; in place."""
    x = np.random.default_rng(2).standard_normal((64, 60)).astype(np.float32)
    for drain, source in ((np.s_[0:64, 0:30], np.s_[0:64, 30:60]), (np.s_[0:64, 0:60:2], np.s_[0:64, 1:60:2]), (np.s_[0:32, 0:60], np.s_[32:64, 0:60]), (np.s_[0:64:2, 3:60], np.s_[1:64:2, 0:57]),
                          (np.s_[5:64:3, 7:60:2], np.s_[5:64:3, 7:60:2])):
        t, want = put(device, x), x.copy()
        want[drain] = dropped(np.ascontiguousarray(x[source]), 7, 2, 0.3)
        device.launch_dropout(t[drain], t[source], 0.3, 7, 2)
        assert get(t).tobytes() == want.tobytes()
    t, want = put(device, x), x.copy()
    want[0:30, 0:30] = dropped(np.ascontiguousarray(x[0:30, 30:60].T), 7, 2, 0.3)
    device.launch_dropout(t[0:30, 0:30], t[0:30, 30:60].T(), 0.3, 7, 2)
    assert get(t).tobytes() == want.tobytes()


@pytest.mark.parametrize("padded", [(1, 7, 12), (7, 12, 1), (7, 1, 12)])
def test_gradients_of_padded_errors(device, padded):
    """The same gradients, bit for bit, from an error that has further axes of one element, dense or a view."""
    rng = np.random.default_rng(3)
    x, g, w, e = (rng.standard_normal(s).astype(np.float32) for s in ((7, 12), (12,), (12, 12), (7, 12)))
    tg, tw = put(device, g), put(device, w)
    wide = np.full(tuple(n + 2 for n in padded), np.nan, np.float32)
    wide[1:-1, 1:-1, 1:-1] = e.reshape(padded)
    part = put(device, wide)[tuple(slice(1, n + 1) for n in padded)]
    for f in (lambda t: t.layerNorm(tg, tg), lambda t: t.dropout(0.4, 5, 6), lambda t: t.gatedMatMul(tw, tw)):
        seen = []
        for error in (put(device, e), put(device, e.reshape(padded)), part):
            t = put(device, x).setRqsGradient(True)
            f(t).backward(error)
            assert t.gradient.shape == (7, 12)
            seen.append(get(t.gradient).tobytes())
        assert seen[0] == seen[1] == seen[2]


def test_a_norm_inside_a_residual_stream_of_higher_rank(device):
    rng = np.random.default_rng(4)
    x, g, b, r = (rng.standard_normal(s).astype(np.float32) for s in ((7, 12), (12,), (12,), (1, 7, 12)))
    t = put(device, x).setRqsGradient(True)
    (t.layerNorm(put(device, g), put(device, b)) * put(device, r)).backward(1.0)
    alone = put(device, x).setRqsGradient(True)
    alone.layerNorm(put(device, g), put(device, b)).backward(put(device, r[0]))
    assert get(t.gradient).tobytes() == get(alone.gradient).tobytes()


# which kernels the shapes of the other tests are meant to run: forward, d_X, the weights' gradients
PATHS = {
    np.float32: [((1, 3001, 1301), "few_rows_split", "few_rows_split", "three_planes"), ((20, 3001, 1301), "few_rows_split", "few_rows_split", "three_planes"),
                 ((16, 64, 65), "few_rows", "few_rows", "three_planes"), ((17, 100, 48), "few_rows", "few_rows", "three_planes"),
                 ((40, 500, 701), "few_rows", "few_rows_split", "three_planes"), ((64, 1501, 700), "few_rows_split", "few_rows_split", "three_planes"),
                 ((33, 1700, 1600), "tiles_three_planes_split", "three_planes_split", "three_planes"), ((150, 50, 70), "tiles_three_planes", "three_planes", "three_planes"),
                 ((2500, 64, 65), "tiles_three_planes", "three_planes", "three_planes_split"), ((300, 1000, 500), "tiles_three_planes_split", "three_planes_split", "three_planes"),
                 ((1301, 1307, 1299), "tiles_two_planes_split", "two_planes_split", "two_planes_split"), ((1300, 1310, 1290), "tiles_two_planes_split", "two_planes_split", "two_planes_split"),
                 ((4099, 500, 1100), "tiles_two_planes", "two_planes_split", "two_planes_split"), ((700, 3000, 1100), "tiles_two_planes_split", "two_planes_split", "two_planes"),
                 ((1200, 1400, 1310), "tiles_two_planes_split", "two_planes_split", "two_planes_split"), ((1200, 2048, 1290), "tiles_two_planes_split", "two_planes_split", "two_planes"),
                 ((1300, 1210, 1408), "tiles_two_planes_split", "two_planes_split", "two_planes_split"), ((2048, 1200, 4096), "tiles_two_planes", "two_planes_split", "two_planes")],
    np.float64: [((1, 3001, 1301), "few_rows_split", "few_rows_split", "tiles"), ((16, 64, 65), "few_rows", "few_rows", "tiles"), ((40, 500, 701), "tiles_split", "tiles_split", "tiles"),
                 ((150, 50, 70), "tiles", "tiles", "tiles"), ((513, 48, 192), "tiles", "tiles_split", "tiles_split"), ((300, 1000, 500), "tiles_split", "tiles_split", "tiles")]}


@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("dt,shape,forward,d_x,weights", [(dt, *p) for dt, paths in PATHS.items() for p in paths])
def test_which_kernels_a_product_runs(device, dt, shape, forward, d_x, weights, along):
    from neureka_amd import _lib
    M, K, N = shape
    zeros = lambda *s: put(device, np.zeros(s, dt))
    x, w, y, e = zeros(M, K), zeros(N, K).T() if along else zeros(K, N), zeros(M, N), zeros(M, N)
    device.launch_gated_matmul("silu", y, x, w, w)
    assert _lib.last_path() == "gated_" + forward
    dx, dg, du = zeros(M, K), zeros(K, N), zeros(K, N)
    for wanted, path in (((dx, dg, du), f"gated_backward_x_{d_x}_w_{weights}"), ((dx, None, None), f"gated_backward_x_{d_x}"), ((None, dg, du), f"gated_backward_w_{weights}")):
        device.launch_gated_matmul_backward("silu", x, w, w, y, y, e, *wanted)
        assert _lib.last_path() == path
