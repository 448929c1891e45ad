"""Products of gatedMatMul that take two half-precision planes, on operands whose small entries decide the result: entries far below the
largest of their row or column, met by zeros (or by very little) where that row is large.  Every result has to be as exact as its own
terms allow, whatever the rest of its row holds."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = np.finfo(np.float32).eps / 2                             # the most that one rounding changes a value, relative to it


def put(device, a):
    from neureka_amd import Tensor
    return Tensor.of(a.dtype, a.shape, a).to(device)


def close(got, want, amount, terms, what):
    """`terms` products of `amount` together, each off by a few units (22 bits and a sign hold an operand to two), and a chain of
    additions that is off like a random walk, of which four standard deviations are allowed: 146 units at the 1200 terms of the shortest product
    here, which also covers the most that the planes may be off, 2^-17 or 128 units.  A sum beyond the type is an infinity."""
    got, tol = np.asarray(got, np.float64), (8 + 4 * np.sqrt(terms)) * U * amount
    over = np.abs(want) > np.finfo(np.float32).max * (1 + U)
    want = np.where(over, np.copysign(np.inf, want), want)
    got, want, tol = (np.where(over & (got == want), 0, a) for a in (got, want, tol))
    bad = ~(np.abs(got - want) <= tol)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - want) / np.maximum(tol, 1e-300), 0)), want.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} values off, worst at {i}: got {got[i]!r}, want {want[i]!r}, allowed {tol[i]!r}")


def forward(device, x, wg, wu, along):
    """gate and up of a product, straight from the device."""
    M, N = x.shape[0], wg.shape[1]
    gate, up = (device.allocate(np.float32, M * N) for _ in range(2))
    weight = (lambda w: put(device, np.ascontiguousarray(w.T)).T()) if along else (lambda w: put(device, w))
    device.launch_gated_matmul("idy", put(device, np.zeros((M, N), np.float32)), put(device, x), weight(wg), weight(wu), gate, up)
    return [device._read_all(d).reshape(M, N) for d in (gate, up)]


def check_forward(device, x, wg, wu, along=False):
    X = x.astype(np.float64)
    for what, got, w in zip(("gate", "up"), forward(device, x, wg, wu, along), (wg, wu)):
        W = w.astype(np.float64)
        close(got, X @ W, np.abs(X) @ np.abs(W), x.shape[1], what)


def check_backward(device, x, wg, wu, e, along=False):
    """With gate = up = 1 and the identity, dg = du = e: dX = e (Wg + Wu)^T, dWg = dWu = x^T e."""
    (M, K), N = x.shape, wg.shape[1]
    one = device.allocateFromOne(np.float32, M * N, 1.0)
    d_x, d_g, d_u = (put(device, np.zeros(s, np.float32)) for s in ((M, K), (K, N), (K, N)))
    weight = (lambda w: put(device, np.ascontiguousarray(w.T)).T()) if along else (lambda w: put(device, w))
    device.launch_gated_matmul_backward("idy", put(device, x), weight(wg), weight(wu), one, one, put(device, e), d_x, d_g, d_u)
    X, G, V, E = (a.astype(np.float64) for a in (x, wg, wu, e))
    read = lambda t: t.items.reshape(t.shape)
    close(read(d_x), E @ (G + V).T, np.abs(E) @ (np.abs(G) + np.abs(V)).T, 2 * N, "dX")
    for what, got in (("dWg", d_g), ("dWu", d_u)):
        close(read(got), X.T @ E, np.abs(X.T) @ np.abs(E), M, what)


def hidden(rng, outer, length, inner, which, scale):
    """x[outer, length] whose entries at `which` are `scale` times smaller than the others, w[length, inner] that is zero at the others."""
    x, w = rng.standard_normal((outer, length)).astype(np.float32), np.zeros((length, inner), np.float32)
    x[:, which] /= np.float32(scale)
    w[which] = rng.standard_normal((len(which), inner)).astype(np.float32)
    return x, w


# the small entries: a run of 64; every other one; every 64th; three and thirty-two anywhere
PLACES = {"run": lambda n: np.arange(64), "every other": lambda n: np.arange(0, n, 2), "every 64th": lambda n: np.arange(5, n, 64),
          "three": lambda n: np.array([1, n // 2, n - 1]), "some": lambda n: np.arange(7, n, n // 32)}


@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("binades", [18, 21, 23, 26, 40])
@pytest.mark.parametrize("place", list(PLACES))
def test_small_entries_that_alone_meet_something(device, along, binades, place):
    rng = np.random.default_rng(binades)
    M, K, N = 1200, 2048, 1290
    x, wg = hidden(rng, M, K, N, PLACES[place](K), 2.0 ** binades)
    wu = np.where(wg != 0, rng.standard_normal((K, N)).astype(np.float32), np.float32(0))
    check_forward(device, x, wg, wu, along)
    # and the other way round: small rows of the weights, an input that is zero elsewhere
    check_forward(device, np.ascontiguousarray(wg.T), np.ascontiguousarray(x.T), np.ascontiguousarray(x[::-1].T), along)


@pytest.mark.parametrize("binades", [21, 26, 40])
@pytest.mark.parametrize("place", list(PLACES))
def test_small_entries_that_alone_meet_something_in_gradients(device, binades, place):
    """dX: small columns of the error against weights that are zero elsewhere.  dW: a channel of x that is small on some tokens, and an
    error that is zero on all others (a mask over tokens)."""
    rng = np.random.default_rng(binades + 1)
    M, K, N = 1300, 1210, 1408
    e, w = hidden(rng, M, N, K, PLACES[place](N), 2.0 ** binades)
    check_backward(device, rng.standard_normal((M, K)).astype(np.float32), np.ascontiguousarray(w.T), np.ascontiguousarray(w[:, ::-1].T), e)
    x, e = hidden(rng, K, M, N, PLACES[place](M), 2.0 ** binades)
    check_backward(device, np.ascontiguousarray(x.T), *(rng.standard_normal((K, N)).astype(np.float32) for _ in range(2)), e)


def test_single_results_from_small_entries(device):
    """A few rows with three small entries, a few columns that are zero elsewhere: only where they cross does a result hang on the small
    entries; everything around is an ordinary product."""
    rng = np.random.default_rng(3)
    M, K, N = 1300, 2048, 1290
    x, wg, wu = (rng.standard_normal(s).astype(np.float32) for s in ((M, K), (K, N), (K, N)))
    at, rows = [9, 1024, 2046], [0, 7, 255, 256, 700, M - 1]
    x[np.ix_(rows, at)] *= np.float32(2.0 ** -27)
    for w, columns in ((wg, [5, 900, N - 1]), (wu, [5, 64])):
        held = w[np.ix_(at, columns)]
        w[:, columns] = 0
        w[np.ix_(at, columns)] = held
    check_forward(device, x, wg, wu)
    check_forward(device, x, wg, wu, along=True)


def crossing(b, at, columns):
    """b[:, columns] zero everywhere but at `at`."""
    held = b[np.ix_(at, columns)]
    b[:, columns] = 0
    b[np.ix_(at, columns)] = held


@pytest.mark.parametrize("along", [False, True])
def test_single_results_from_small_entries_in_gradients(device, along):
    rng = np.random.default_rng(8)
    M, K, N = 1300, 1210, 1409
    x, wg, wu, e = (rng.standard_normal(s).astype(np.float32) for s in ((M, K), (K, N), (K, N), (M, N)))
    g, u = wg.T.copy(), wu.T.copy()
    for w in (g, u):                                        # d_X: rows of e against columns of both weights' transposes
        crossing(w, [3, 800, N - 1], [0, 33, 1000, K - 1])
    e[np.ix_([1, 130, 131, M - 1], [3, 800, N - 1])] *= np.float32(2.0 ** -26)
    check_backward(device, x, np.ascontiguousarray(g.T), np.ascontiguousarray(u.T), e, along)
    x, e = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal((M, N)).astype(np.float32)
    crossing(e, [7, 640, M - 1], [4, 500, N - 1])           # the weights' gradients: columns of x against columns of e
    x[np.ix_([7, 640, M - 1], [2, 300, 301, K - 1])] *= np.float32(2.0 ** -26)
    check_backward(device, x, wg, wu, e, along)


@pytest.mark.parametrize("binades", [10, 16, 17, 18, 19, 20, 21, 22, 23])
@pytest.mark.parametrize("along", [False, True])
def test_scales_within_a_row_that_undo_each_other(device, along, binades):
    """Every other column of x scaled down, the matching rows of the weights scaled up: both halves count alike."""
    rng = np.random.default_rng(binades)
    M, K, N = 1200, 1400, 1310
    by = np.where(np.arange(K) % 2, 2.0 ** binades, 1.0).astype(np.float32)
    x = rng.uniform(0.5, 1, (M, K)).astype(np.float32) * rng.choice([-1, 1], (M, K)).astype(np.float32) / by
    wg, wu = (rng.uniform(0.5, 1, (K, N)).astype(np.float32) * rng.choice([-1, 1], (K, N)).astype(np.float32) * by[:, None] for _ in range(2))
    check_forward(device, x, wg, wu, along)


@pytest.mark.parametrize("along", [False, True])
def test_a_product_that_is_not_split_into_parts(device, along):
    rng = np.random.default_rng(4)
    M, K, N = 2048, 1200, 4096
    x, wg = hidden(rng, M, K, N, np.arange(3, K, 100), 2.0 ** 24)
    wu = rng.standard_normal((K, N)).astype(np.float32)
    wu[:, 17] = wg[:, 18]
    check_forward(device, x, wg, wu, along)


def test_empty_rows_and_columns_and_sparse_operands(device):
    """Rows and columns of zeros beside rows with small entries; operands with one entry in fifty, half of them 2^-22 of the rest."""
    rng = np.random.default_rng(5)
    M, K, N = 1200, 1400, 1310
    x, wg, wu = (rng.standard_normal(s).astype(np.float32) for s in ((M, K), (K, N), (K, N)))
    x[:, :3] *= np.float32(2.0 ** -25)
    x[3:40], wg[:, 100:400], wu[:, 1309] = 0, 0, 0
    check_forward(device, x, wg, wu)
    for a in (x, wg, wu):
        a *= (rng.random(a.shape) < 0.02)
        a[rng.random(a.shape) < 0.5] *= np.float32(2.0 ** -22)
    check_forward(device, x, wg, wu)


def test_rows_at_the_ends_of_the_range(device):
    """Rows near the least and the largest floats, with entries down to the least of all."""
    rng = np.random.default_rng(6)
    M, K, N = 1200, 1400, 1310
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[:300] *= np.float32(2.0 ** -105)
    x[300:600] *= np.float32(2.0 ** 120)
    x[::3, 17] = np.float32(2.0 ** -149)
    x[1::3, 18] = np.float32(2.0 ** -127)
    wg, wu = (rng.standard_normal((K, N)).astype(np.float32) for _ in range(2))
    wg[:, 40], wu[:, 41] = 0, 0
    wg[17, 40], wu[18, 41] = 2.0 ** 100, 2.0 ** 90
    check_forward(device, x, wg, wu)


@pytest.mark.parametrize("exponent", [-100, -110, -114, -118, -122, -125])
def test_three_planes_at_the_lower_end_of_the_range(device, exponent):
    """Products that take three bfloat16 numbers: below 2^-110 the last of them ends at multiples of 2^-133, so an operand is off by at
    most 2^-134, and every result by that times what it meets."""
    from neureka_amd import _lib
    rng = np.random.default_rng(7)
    M, K, N = 150, 200, 100
    x = (rng.standard_normal((M, K)) * 2.0 ** exponent).astype(np.float32)
    w = (rng.standard_normal((K, N)) * 2.0 ** 100).astype(np.float32)
    X, W = x.astype(np.float64), w.astype(np.float64)
    for got in forward(device, x, w, w, False):
        assert "three_planes" in _lib.last_path()
        tol = (8 + 4 * np.sqrt(K)) * U * (np.abs(X) @ np.abs(W)) + 2.0 ** -134 * np.abs(W).sum(0)
        bad = np.abs(got - X @ W) > tol
        assert not bad.any(), (bad.sum(), (np.abs(got - X @ W) / tol).max())
