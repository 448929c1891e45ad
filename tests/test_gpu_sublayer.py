"""layerNorm, dropout and gatedMatMul against their definitions in 64 bits: sizes around every tile, vector and plan border, views, both types, refusals,
gradients by formula and by differences, and the three of them together as a feed-forward sublayer.

Tolerances count roundings: u = eps / 2 is the most one rounding changes a value, relative to it."""
import numpy as np
import pytest

from helpers import assert_bits

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]


def unit(dt):
    return np.finfo(dt).eps / 2


def put(device, a):
    from neureka_amd import Tensor
    return Tensor.of(a.dtype, a.shape, a).to(device)


def get(t):
    return t.items.reshape(t.shape)


def within(got, want, tol, what):
    got, want, tol = np.asarray(got, np.float64), np.asarray(want, np.float64), np.broadcast_to(np.asarray(tol, np.float64), np.shape(want))
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    if bad.any():
        i = np.unravel_index(np.argmax(np.where(bad, np.abs(got - want) / np.maximum(tol, 1e-300), 0)), want.shape)
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} values off, worst at {i}: got {got[i]!r}, want {want[i]!r}, allowed {tol[i]!r}")


# ---- layerNorm ---------------------------------------------------------------------------------------------------

def norm_in_64_bits(x, gain, bias, error, eps):
    x, gain, bias, error = (np.asarray(a, np.float64) for a in (x, gain, bias, error))
    D = x.shape[-1]
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
    h = (x - mean) * rstd
    g = error * gain
    dx = rstd * (g - g.mean(-1, keepdims=True) - h * (g * h).mean(-1, keepdims=True))
    out = {"y": h * gain + bias, "dx": dx, "dgain": (error * h).reshape(-1, D).sum(0), "dbias": error.reshape(-1, D).sum(0)}
    # A row's sums go through at most ~20 additions in a thread, 6 across a wavefront and 16 across a block: under 48 roundings.
    # The mean is off by at most 48 u mean|x|, which enters h times rstd: H bounds |h| and what multiplies that error.
    H = np.abs(h) + rstd * np.abs(x).mean(-1, keepdims=True)
    ag = np.abs(g)
    amount = {"y": H * np.abs(gain) + np.abs(bias), "dx": rstd * (ag + ag.mean(-1, keepdims=True) + H * (ag * H).mean(-1, keepdims=True)),
              "dgain": (np.abs(error) * H).reshape(-1, D).sum(0), "dbias": np.abs(error).reshape(-1, D).sum(0)}
    return out, amount


# y: the mean's 48, half of the variance's 50, 4 of the formula, rounded up.  dx: two such chains and the sums' own.  Column sums: their
# terms' roundings and a chain of rows / blocks + 32 + 16 additions, under 64 for the sizes here.
NORM_ROUNDINGS = {"y": 80, "dx": 240, "dgain": 160, "dbias": 64}


def check_norm(device, dt, x, gain, bias, error, eps=1e-5, tx=None, te=None):
    tx = put(device, x) if tx is None else tx
    te = put(device, error) if te is None else te
    tg, tb = put(device, gain), put(device, bias)
    for t in (tx, tg, tb):
        t.setRqsGradient(True)
    y = tx.layerNorm(tg, tb, eps)
    y.backward(te)
    want, amount = norm_in_64_bits(x, gain, bias, error, eps)
    for k, t in (("y", y), ("dx", tx.gradient), ("dgain", tg.gradient), ("dbias", tb.gradient)):
        within(get(t), want[k].reshape(t.shape), NORM_ROUNDINGS[k] * unit(dt) * amount[k].reshape(t.shape), k)
    return y


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 1), (1, 2), (5, 3), (2, 63), (7, 64), (300, 65), (9, 129), (1, 255), (2, 256), (3, 257), (1025, 511), (4, 512), (3, 513),
                                       (5, 1023), (2, 1024), (3, 1025), (2, 2047), (700, 2049), (2, 4096), (3, 4097), (2, 8193), (3, 16384), (2, 16385), (65, 20001)])
def test_norm_at_every_border(device, dt, rows, cols):
    rng = np.random.default_rng(rows * 31 + cols)
    x = (rng.standard_normal((rows, cols)) * 2 + 0.5).astype(dt)
    check_norm(device, dt, x, (1 + 0.2 * rng.standard_normal(cols)).astype(dt), rng.standard_normal(cols).astype(dt), rng.standard_normal((rows, cols)).astype(dt))


@pytest.mark.parametrize("dt", DTYPES)
def test_norm_of_higher_ranks_views_and_constant_rows(device, dt):
    rng = np.random.default_rng(3)
    gain, bias = rng.standard_normal(24).astype(dt), rng.standard_normal(24).astype(dt)
    x = rng.standard_normal((2, 5, 24)).astype(dt)
    x[1, 3] = 7.25                                          # variance 0: only epsilon keeps the row finite
    check_norm(device, dt, x, gain, bias, rng.standard_normal(x.shape).astype(dt))
    # every row of a wider matrix from its third column on: rows one pitch apart, taken as they lie
    base = rng.standard_normal((9, 40)).astype(dt)
    error = rng.standard_normal((9, 24)).astype(dt)
    check_norm(device, dt, base[:, 2:26], gain, bias, error, tx=put(device, base)[:, 2:26])
    # every second column, a transpose, an error that is a view: copied first
    check_norm(device, dt, base[:, 0:40:2], gain[:20], bias[:20], error[:, :20], tx=put(device, base)[:, 0:40:2], te=put(device, error)[:, 0:20])
    check_norm(device, dt, np.ascontiguousarray(base.T), gain[:9], bias[:9], np.ascontiguousarray(error[:, :9].T.repeat(5, 0)[:40]), tx=put(device, base).T())


def test_norm_in_place_leaves_the_rows_behind_alone(device):
    rng = np.random.default_rng(4)
    held = rng.standard_normal((8, 100)).astype(np.float32)
    gain, bias = np.ones(100, np.float32), np.zeros(100, np.float32)
    t = put(device, held)
    part = t[0:5, 0:100]
    device.launch_layer_norm(part, part, put(device, gain), put(device, bias), 1e-5)
    now = get(t)
    assert_bits(now[5:], held[5:], "rows behind")
    want, amount = norm_in_64_bits(held[:5], gain, bias, held[:5], 1e-5)
    within(now[:5], want["y"], NORM_ROUNDINGS["y"] * unit(np.float32) * amount["y"], "in place")


def test_norm_passes_infinities_and_nan_on_within_their_row(device):
    x = np.ones((4, 300), np.float32) * np.arange(300, dtype=np.float32)
    x[1, 7] = np.inf
    x[2, 299] = np.nan
    y = get(put(device, x).layerNorm(put(device, np.ones(300, np.float32)), put(device, np.zeros(300, np.float32))))
    assert np.isnan(y[1]).all() and np.isnan(y[2]).all() and np.isfinite(y[[0, 3]]).all()


def test_norm_computes_only_the_gradients_asked_for_and_the_same_twice(device):
    rng = np.random.default_rng(6)
    x, e = (rng.standard_normal((3000, 700)).astype(np.float32) for _ in range(2))
    gain, bias = (rng.standard_normal(700).astype(np.float32) for _ in range(2))
    seen = []
    for wanted in ((1, 1, 1), (1, 1, 1), (0, 1, 0), (1, 0, 0), (0, 0, 1)):
        ts = [put(device, a) for a in (x, gain, bias)]
        for t, w in zip(ts, wanted):
            t.setRqsGradient(bool(w))
        ts[0].layerNorm(ts[1], ts[2]).backward(put(device, e))
        assert [t.gradient is not None for t in ts] == [bool(w) for w in wanted]
        seen.append([None if t.gradient is None else get(t.gradient) for t in ts])
    for other in seen[1:]:
        for a, b in zip(seen[0], other):
            if b is not None:
                assert_bits(b, a, "repeated")


def test_norm_refusals(device):
    from neureka_amd import HipError, IllegalArgumentException
    x, g = put(device, np.ones((4, 6), np.float32)), put(device, np.ones(6, np.float32))
    for args in ((g, put(device, np.ones(5, np.float32))), (put(device, np.ones((6, 1), np.float32)), g), (g, put(device, np.ones(6)))):
        with pytest.raises(IllegalArgumentException):
            x.layerNorm(*args)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(IllegalArgumentException):
            x.layerNorm(g, g, eps)
    with pytest.raises(IllegalArgumentException):
        put(device, np.ones((4, 6), np.int32)).layerNorm(put(device, np.ones(6, np.int32)), put(device, np.ones(6, np.int32)))
    with pytest.raises(IllegalArgumentException):
        x.setRqsGradient(True).layerNorm(g, g).backward(put(device, np.ones((4, 5), np.float32)))
    y = put(device, np.zeros((4, 6), np.float32))
    with pytest.raises(HipError):                           # the drain on the gain
        device.launch_layer_norm(y, x, y[0, 0:6], g, 1e-5)
    lib, h = device._lib, device.handle
    p, q = x._data.ptr, y._data.ptr
    for call in ((0, 0, 6, p, 6), (0, 4, 0, p, 6), (0, 4, 6, p, 5), (7, 4, 6, p, 6), (0, 40, 6, p, 6), (0, 4, 6, p, 1 << 40), (0, 1 << 30, 1 << 30, p, 1 << 30)):
        assert lib.nk_layer_norm(h, *call, g._data.ptr, g._data.ptr, 1e-5, q, 0, 0) != 0, call
    assert lib.nk_layer_norm(h, 0, 4, 6, p, 6, g._data.ptr, g._data.ptr, 1e-5, q, q, 0) != 0          # mean without rstd
    assert lib.nk_layer_norm_backward(h, 0, 4, 6, p, 6, g._data.ptr, g._data.ptr, g._data.ptr, p, 0, 0, 0) != 0


# ---- dropout -------------------------------------------------------------------------------------------------------

def kept(n, seed, offset, p):
    u = np.uint64
    low = u(0xFFFFFFFF)
    block = np.arange((n + 3) // 4, dtype=u)
    c = [block & low, block >> u(32), np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(key[0]), b & low, (a >> u(32)) ^ c[3] ^ u(key[1]), a & low]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:n] >= u(int(p * 4294967296.0))


def test_the_generator_gives_its_published_words():
    """Known answers of Philox4x32-10: counter and key all zeros, all ones (the words that the paper's authors publish)."""
    def words(counter, key):
        c, k = list(counter), list(key)
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return c
    assert words([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert words([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    # the vectorised form above draws the first of them
    assert kept(4, 0, 0, 0x6627E8D5 / 2 ** 32).tolist() == [True, True, True, True] and not kept(4, 0, 0, (0x6627E8D5 + 1) / 2 ** 32)[0]


def dropped(x, seed, offset, p):
    scale = x.dtype.type(1 / (1 - p) if p < 1 else 0)
    return np.where(kept(x.size, seed, offset, p).reshape(x.shape), x * scale, x.dtype.type(0))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 255, 1024, 1025, 4099, 100003])
@pytest.mark.parametrize("p,seed,offset", [(0.0, 0, 0), (0.1, 12345, 7), (0.5, (1 << 64) - 1, (1 << 64) - 1), (1.0, 3, 1 << 40)])
def test_dropout_is_the_generator_bit_for_bit(device, dt, n, p, seed, offset):
    x = np.random.default_rng(n).standard_normal(n).astype(dt)
    t = put(device, x).setRqsGradient(True)
    y = t.dropout(p, seed, offset)
    assert_bits(get(y), dropped(x, seed, offset, p), "forward")
    e = np.random.default_rng(n + 1).standard_normal(n).astype(dt)
    y.backward(put(device, e))
    assert_bits(get(t.gradient), dropped(e, seed, offset, p), "backward")


def test_dropout_of_views_virtual_tensors_and_in_place(device):
    from neureka_amd import Tensor, _lib
    x = np.random.default_rng(1).standard_normal((6, 7, 9)).astype(np.float32)
    t = put(device, x)
    for view, want in ((t.permute(2, 0, 1), x.transpose(2, 0, 1)), (t[1:5, 0:7:3, 2:9], x[1:5, 0:7:3, 2:9]), (t[2:4, 0:7, 0:9], x[2:4])):
        assert_bits(get(view.dropout(0.3, 99, 5)), dropped(np.ascontiguousarray(want), 99, 5, 0.3), "view")
    assert_bits(get(Tensor.of(np.float32, (5, 5), 3.0).to(device).dropout(0.4, 1)), dropped(np.full((5, 5), 3, np.float32), 1, 0, 0.4), "virtual")
    part = t[0:2, 0:7, 0:9]
    device.launch_dropout(part, part, 0.5, 11)
    assert _lib.last_path() == "dropout_dense"
    assert_bits(get(t), np.concatenate([dropped(x[:2], 11, 0, 0.5), x[2:]]), "in place, the rest untouched")


def test_dropout_clears_infinities_and_nan_where_it_drops_and_keeps_its_share(device):
    x = np.full(1 << 20, np.nan, np.float32)
    x[::2] = np.inf
    y = get(put(device, x).dropout(0.25, 2, 9))
    keep = kept(x.size, 2, 9, 0.25)
    assert (y[~keep] == 0).all() and not np.isfinite(y[keep]).any()
    # a share of 0.75 of 2^20 draws: five standard deviations are 0.0021
    assert abs(keep.mean() - 0.75) < 0.0022
    assert (kept(x.size, 2, 10, 0.25) != keep).any() and (kept(x.size, 3, 9, 0.25) != keep).any()


def test_dropout_refusals(device):
    from neureka_amd import IllegalArgumentException
    t = put(device, np.ones((3, 4), np.float32))
    for args in ((-0.1, 0), (1.5, 0), (float("nan"), 0), (0.5, -1), (0.5, 1 << 64), (0.5, 0, -1), (0.5, 0, 1 << 64)):
        with pytest.raises(IllegalArgumentException):
            t.dropout(*args)
    with pytest.raises(IllegalArgumentException):
        put(device, np.ones(4, np.int32)).dropout(0.5, 1)
    with pytest.raises(IllegalArgumentException):
        device.launch_dropout(put(device, np.ones((4, 3), np.float32)), t, 0.5, 1)
    (p, _, c), = device._ops(t)
    lib, h = device._lib, device.handle
    assert lib.nk_dropout(h, 0, 2, p, c, p, c, 0.5, 1, 0, 11) != 0 and lib.nk_dropout(h, 5, 2, p, c, p, c, 0.5, 1, 0, 12) != 0
    assert lib.nk_dropout(h, 0, 2, p, c, p, c, 2.0, 1, 0, 12) != 0 and lib.nk_dropout(h, 1, 2, p, c, p, c, 0.5, 1, 0, 12) != 0      # (as doubles it is too short)
    assert lib.nk_dropout(h, 0, 0, p, c, p, c, 0.5, 1, 0, 12) != 0 and lib.nk_dropout(h, 0, 2, p, c, p, None, 0.5, 1, 0, 12) != 0


# ---- gatedMatMul ---------------------------------------------------------------------------------------------------

def act_in_64_bits(name, g):
    """f, f' as the library defines its activations."""
    g = np.asarray(g, np.float64)
    if name == "idy":
        return g, np.ones_like(g)
    if name == "relu":
        return np.where(g >= 0, g, 0.01 * g), np.where(g >= 0, 1.0, 0.01)
    if name == "tanh":
        return np.tanh(g), 1 / np.cosh(g) ** 2
    k = 1.702 if name == "gelu" else 1.0
    s = 1 / (1 + np.exp(-k * g))
    c = 1 / (1 + np.exp(k * g))
    return (s, s * c) if name == "sig" else (g * s, s + k * g * s * c)


SHAPES = [(1, 1, 1), (1, 7, 5), (2, 16, 16), (3, 17, 33), (5, 4, 130), (15, 31, 64), (16, 64, 65), (17, 100, 48), (31, 5, 96), (33, 33, 33), (47, 129, 20), (63, 8, 256),
          (64, 40, 64), (65, 65, 65), (100, 3, 300), (127, 128, 63), (128, 16, 64), (129, 20, 129), (200, 260, 70), (257, 255, 130), (300, 64, 257), (513, 48, 192)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gated_products_of_small_integers_are_exact(device, dt, along, M, K, N):
    """With f = identity and integers every sum is exact in either type (the largest, of d_X and d_W, stays below 2^24), so every
    index is checked: H = g u, dX, dWg, dWu."""
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    x = rng.integers(-2, 3, (M, K)).astype(dt)
    wg, wu = (rng.integers(-1, 2, (K, N)).astype(dt) for _ in range(2))
    e = rng.integers(-2, 3, (M, N)).astype(dt)
    tx = put(device, x).setRqsGradient(True)
    tg, tu = ((put(device, np.ascontiguousarray(w.T)).T() if along else put(device, w)).setRqsGradient(True) for w in (wg, wu))
    y = tx.gatedMatMul(tg, tu, "idy")
    y.backward(put(device, e))
    X, G, U, E = (a.astype(np.float64) for a in (x, wg, wu, e))
    g, u = X @ G, X @ U
    dg, du = E * u, E * g
    for sums in (np.abs(dg) @ np.abs(G.T) + np.abs(du) @ np.abs(U.T), np.abs(X.T) @ np.abs(dg), np.abs(X.T) @ np.abs(du)):
        assert sums.max() < 2 ** 24                         # (a statement about the inputs, not about the kernels)
    for k, t, want in (("H", y, g * u), ("dX", tx.gradient, dg @ G.T + du @ U.T), ("dWg", tg.gradient, X.T @ dg), ("dWu", tu.gradient, X.T @ du)):
        got = get(t).astype(np.float64)
        assert got.shape == want.shape and (got == want).all(), (k, np.argwhere(got != want)[:3].tolist(), int((got != want).sum()))


def sum_roundings(n):
    """Roundings of a sum of n products: every product contributes, and the chain's roundings add up like a random walk;
    four standard deviations of that walk and eight to spare."""
    return 8 + 4 * np.sqrt(n)


def check_gated(device, dt, fun, M, K, N, along=False, seed=0, scale=1.0):
    rng = np.random.default_rng(seed + M + K + N)
    x = (scale * rng.standard_normal((M, K))).astype(dt)
    wg, wu = ((rng.standard_normal((K, N)) / np.sqrt(K)).astype(dt) for _ in range(2))
    e = rng.standard_normal((M, N)).astype(dt)
    tx = put(device, x).setRqsGradient(True)
    tg, tu = ((put(device, np.ascontiguousarray(w.T)).T() if along else put(device, w)).setRqsGradient(True) for w in (wg, wu))
    y = tx.gatedMatMul(tg, tu, fun)
    y.backward(put(device, e))
    X, G, U, E = (a.astype(np.float64) for a in (x, wg, wu, e))
    g, u = X @ G, X @ U
    f, slope = act_in_64_bits(fun, g)
    dg, du = E * u * slope, E * f
    r = unit(dt)
    tol_g, tol_u = (sum_roundings(K) * r * (np.abs(X) @ np.abs(w)) for w in (G, U))
    # |f'| <= 1.13, |f''| <= 1 for every f here (relu has no f'': its slope is compared away from the step by the caller's choice of f);
    # the activations themselves are within 1.3e-6 = 22 u of f32 at the far ends of their range
    within(get(y), f * u, 1.2 * tol_g * np.abs(u) + np.abs(f) * tol_u + 1.2 * tol_g * tol_u + 32 * r * np.abs(f * u), "H")
    tol_dg = np.abs(E) * (tol_u * 1.2 + (np.abs(u) + tol_u) * tol_g + 32 * r * np.abs(u) * (np.abs(slope) + 1))
    tol_du = np.abs(E) * (1.2 * tol_g + 32 * r * np.abs(f))
    within(get(tx.gradient), dg @ G.T + du @ U.T, tol_dg @ np.abs(G.T) + tol_du @ np.abs(U.T) + sum_roundings(2 * N) * r * (np.abs(dg) @ np.abs(G.T) + np.abs(du) @ np.abs(U.T)), "dX")
    within(get(tg.gradient), X.T @ dg, np.abs(X.T) @ tol_dg + sum_roundings(M) * r * (np.abs(X.T) @ np.abs(dg)), "dWg")
    within(get(tu.gradient), X.T @ du, np.abs(X.T) @ tol_du + sum_roundings(M) * r * (np.abs(X.T) @ np.abs(du)), "dWu")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("fun", ["idy", "sig", "silu", "gelu", "tanh"])
def test_gated_activations_and_their_gradients(device, dt, fun):
    check_gated(device, dt, fun, 70, 90, 110, seed=5)
    check_gated(device, dt, fun, 9, 40, 30, seed=6, scale=30.0)        # arguments far out


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 4096, 100), (4, 1000, 2000), (16, 3000, 70), (40, 2500, 64), (64, 777, 1111), (300, 1000, 500), (1000, 300, 200), (2500, 64, 65), (520, 520, 1030)])
def test_gated_sums_of_real_lengths(device, dt, along, M, K, N):
    check_gated(device, dt, "silu", M, K, N, along)


def test_gated_relu_keeps_a_hundredth_of_the_negative_side(device):
    x = np.array([[-3.0, 0.0, 2.0]], np.float32).T
    one = np.ones((1, 1), np.float32)
    ts = [put(device, a).setRqsGradient(True) for a in (x, one, one)]
    y = ts[0].gatedMatMul(ts[1], ts[2], "relu")
    y.backward(1.0)
    hundredth = np.float32(0.01)
    assert_bits(get(y), np.array([[9 * hundredth], [0], [4]], np.float32), "forward")
    within(get(ts[0].gradient), np.array([[-6 * 0.01], [0.0], [4.0]]), 8 * unit(np.float32), "dX: 2 x slope")


def test_gated_gradients_against_differences(device):
    rng = np.random.default_rng(8)
    x, wg, wu, e = rng.standard_normal((5, 6)), rng.standard_normal((6, 7)), rng.standard_normal((6, 7)), rng.standard_normal((5, 7))
    ts = [put(device, a).setRqsGradient(True) for a in (x, wg, wu)]
    ts[0].gatedMatMul(ts[1], ts[2], "gelu").backward(put(device, e))

    def loss(i, d):
        moved = [a + d if j == i else a for j, a in enumerate((x, wg, wu))]
        return float((get(put(device, moved[0]).gatedMatMul(put(device, moved[1]), put(device, moved[2]), "gelu")) * e).sum())
    step = 2.0 ** -17
    for i, t in enumerate(ts):
        direction = rng.standard_normal(t.shape)
        slope = (loss(i, step * direction) - loss(i, -step * direction)) / (2 * step)
        # the difference's own error: step^2 times a third derivative of order 1e3, and cancellation 1e2 * 2^-53 / step
        assert abs(slope - (get(t.gradient) * direction).sum()) < 1e3 * step ** 2 + 1e3 * 2.0 ** -53 / step


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("M", [3, 20, 150])
def test_gated_infinities_nan_and_overflow_are_those_of_the_type(device, dt, M):
    rng = np.random.default_rng(M)
    x, wg, wu = (rng.standard_normal(s).astype(dt) for s in ((M, 50), (50, 70), (50, 70)))
    big = np.finfo(dt).max
    x[0, 3], x[1, 4], x[2, 5] = np.inf, np.nan, -np.inf
    wg[7, 11], wu[8, 12] = np.inf, -np.inf
    wg[:, 13] = 0
    wg[9, 13], wg[10, 13] = big, big                        # x 2^7 overflows, to an infinity of the sum's sign
    x[:, 9], x[:, 10] = 128, 1
    x[M - 1, 9] = -128
    gate, up = (device.allocate(dt, M * 70) for _ in range(2))
    y = put(device, np.zeros((M, 70), dt))
    device.launch_gated_matmul("idy", y, put(device, x), put(device, wg), put(device, wu), gate, up)
    with np.errstate(all="ignore"):
        for name, data, w in (("gate", gate, wg), ("up", up, wu)):
            terms = x[:, :, None] * w[None]                  # rounded to the type: an overflowing product is an infinity
            want = terms.astype(np.float64).sum(1)
            got = device._read_all(data).reshape(M, 70)
            amount = np.abs(np.where(np.isfinite(terms), terms, 0)).astype(np.float64).sum(1)
            over = np.isfinite(want) & (np.abs(want) > big)
            want[over] = np.sign(want[over]) * np.inf
            assert (np.isnan(got) == np.isnan(want)).all(), (name, "NaN")
            assert (np.where(np.isinf(want), got == want, True)).all(), (name, "infinities")
            fine = np.isfinite(want)
            within(got[fine], want[fine], sum_roundings(50) * unit(dt) * amount[fine], name)


def test_gated_small_and_large_magnitudes_keep_their_digits(device):
    """Exponents from 2^-100 to 2^100 in one product: every output is as exact as its own terms allow."""
    rng = np.random.default_rng(12)
    for M in (5, 140):
        x = (rng.standard_normal((M, 64)) * 2.0 ** rng.integers(-60, 60, (M, 1))).astype(np.float32)
        wg, wu = ((rng.standard_normal((64, 96)) * 2.0 ** rng.integers(-40, 40, (1, 96))).astype(np.float32) for _ in range(2))
        gate, up = (device.allocate(np.float32, M * 96) for _ in range(2))
        device.launch_gated_matmul("idy", put(device, np.zeros((M, 96), np.float32)), put(device, x), put(device, wg), put(device, wu), gate, up)
        for data, w in ((gate, wg), (up, wu)):
            X, W = x.astype(np.float64), w.astype(np.float64)
            within(device._read_all(data).reshape(M, 96), X @ W, sum_roundings(64) * unit(np.float32) * (np.abs(X) @ np.abs(W)), "gate or up")


def test_gated_takes_higher_ranks_views_and_repeated_weights(device):
    rng = np.random.default_rng(9)
    x = rng.integers(-2, 3, (2, 3, 20)).astype(np.float32)
    w = rng.integers(-1, 2, (20, 60)).astype(np.float32)
    tx, tw = put(device, x), put(device, w).setRqsGradient(True)
    want = (x.astype(np.float64) @ w) ** 2
    y = tx.gatedMatMul(tw, tw, "idy")
    assert y.shape == (2, 3, 60) and (get(y) == want).all()
    y.backward(1.0)
    flat = x.reshape(-1, 20).astype(np.float64)
    assert (get(tw.gradient) == 2 * flat.T @ (flat @ w)).all()
    # weights that are columns of one wider matrix, one stored by rows and the other by columns, an input that is a view
    wide = put(device, w)
    both = tx.gatedMatMul(wide[0:20, 0:30], wide[0:20, 30:60], "idy")
    assert (get(both) == (x.astype(np.float64) @ w[:, :30]) * (x.astype(np.float64) @ w[:, 30:])).all()
    mixed = tx.gatedMatMul(tw, put(device, np.ascontiguousarray(w.T)).T(), "idy")
    assert (get(mixed) == want).all()
    view = put(device, np.ascontiguousarray(x.transpose(2, 0, 1))).permute(1, 2, 0)
    assert (get(view.gatedMatMul(tw, tw, "idy")) == want).all()


def test_gated_gives_the_same_bits_twice_and_leaves_other_rows_alone(device):
    rng = np.random.default_rng(10)
    for M, K, N in ((3, 2000, 300), (50, 2000, 300), (400, 2000, 300)):
        x, wg, wu = (put(device, rng.standard_normal(s).astype(np.float32)) for s in ((M, K), (K, N), (K, N)))
        held = np.full((M + 3, N), 7, np.float32)
        t = put(device, held)
        part = t[1:M + 1, 0:N]
        device.launch_gated_matmul("silu", part, x, wg, wu)
        first = get(t)
        device.launch_gated_matmul("silu", part, x, wg, wu)
        assert_bits(get(t), first, "twice")
        assert (first[[0, M + 1, M + 2]] == 7).all() and (first[1:M + 1] != 7).any(1).all()


def test_gated_refusals(device):
    from neureka_amd import HipError, IllegalArgumentException
    x, w = put(device, np.ones((4, 6), np.float32)), put(device, np.ones((6, 5), np.float32))
    for gate, up in ((w, put(device, np.ones((6, 4), np.float32))), (put(device, np.ones((5, 6), np.float32)),) * 2, (w, put(device, np.ones((6, 5)))), (put(device, np.ones(6, np.float32)),) * 2):
        with pytest.raises(IllegalArgumentException):
            x.gatedMatMul(gate, up)
    with pytest.raises(IllegalArgumentException):
        x.gatedMatMul(w, w, "softplus")
    y = x.setRqsGradient(True).gatedMatMul(w, w)
    for bad in (np.ones((4, 6), np.float32), np.ones((4, 5))):
        with pytest.raises(IllegalArgumentException):
            y.backward(put(device, bad))
    big = put(device, np.ones((6, 6), np.float32))
    with pytest.raises(HipError):                           # the drain on the input
        device.launch_gated_matmul("silu", big, big, big, big)
    lib, h = device._lib, device.handle
    p, q, r = x._data.ptr, w._data.ptr, put(device, np.ones((4, 5), np.float32))
    good = [8, 0, 0, 4, 6, 5, p, q, q, r._data.ptr, 0, 0]
    for at, value in ((0, 99), (0, 1), (1, 2), (2, 2), (3, 0), (4, -1), (5, 1 << 31), (3, 400), (4, 1 << 20), (9, 0), (10, r._data.ptr), (6, 12345)):
        bad = list(good)
        bad[at] = value
        assert lib.nk_gated_matmul(h, *bad) != 0, (at, value)


# ---- together ------------------------------------------------------------------------------------------------------

def sublayer_in_64_bits(x, gain, bias, wg, wu, wd, keep, p, error):
    """z = x + dropout((silu(n wg) * (n wu)) wd), n = norm of x, and all gradients."""
    mean = x.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + 1e-5)
    hat = (x - mean) * rstd
    n = hat * gain + bias
    g, u = n @ wg, n @ wu
    f, slope = act_in_64_bits("silu", g)
    h = f * u
    mask = keep / (1 - p)
    z = x + (h @ wd) * mask
    do = error * mask
    dh = do @ wd.T
    dg, du = dh * u * slope, dh * f
    dn = dg @ wg.T + du @ wu.T
    q = dn * gain
    dx = error + rstd * (q - q.mean(-1, keepdims=True) - hat * (q * hat).mean(-1, keepdims=True))
    return {"z": z, "x": dx, "gain": (dn * hat).sum(0), "bias": dn.sum(0), "wg": n.T @ dg, "wu": n.T @ du, "wd": h.T @ do}


@pytest.mark.parametrize("dt,tol", [(np.float32, 2.0 ** -16), (np.float64, 2.0 ** -44)])
@pytest.mark.parametrize("M,K,N", [(1, 40, 90), (37, 64, 200), (300, 96, 257)])
def test_a_feed_forward_sublayer_trains(device, dt, tol, M, K, N):
    """The operators as they are used, with matMul and the residual addition: output and all six gradients, each within `tol` of
    its own largest value (a chain of five operators with sums of up to 300 terms: 2^8 roundings of that size)."""
    rng = np.random.default_rng(M)
    a = {"x": rng.standard_normal((M, K)), "gain": 1 + 0.1 * rng.standard_normal(K), "bias": 0.1 * rng.standard_normal(K), "wg": rng.standard_normal((K, N)) / K ** 0.5,
         "wu": rng.standard_normal((K, N)) / K ** 0.5, "wd": rng.standard_normal((N, K)) / N ** 0.5}
    a = {k: v.astype(dt) for k, v in a.items()}
    error = rng.standard_normal((M, K)).astype(dt)
    t = {k: put(device, v).setRqsGradient(True) for k, v in a.items()}
    n = t["x"].layerNorm(t["gain"], t["bias"])
    h = n.gatedMatMul(t["wg"], t["wu"], "silu")
    z = t["x"] + h.matMul(t["wd"]).dropout(0.2, 77, 3)
    z.backward(put(device, error))
    want = sublayer_in_64_bits(*(a[k].astype(np.float64) for k in ("x", "gain", "bias", "wg", "wu", "wd")), kept(M * K, 77, 3, 0.2).reshape(M, K), 0.2, error.astype(np.float64))
    within(get(z), want["z"], tol * np.abs(want["z"]).max(), "z")
    for k, v in t.items():
        within(get(v.gradient), want[k].reshape(v.shape), tol * np.abs(want[k]).max(), "d" + k)


def test_operands_on_the_host_visit_the_device_and_go_back(device):
    from neureka_amd import Tensor
    rng = np.random.default_rng(14)
    x = put(device, rng.standard_normal((4, 6)).astype(np.float32)).setRqsGradient(True)
    gain, bias, w = (Tensor.of(np.float32, s, rng.standard_normal(s).astype(np.float32)).setRqsGradient(True) for s in ((6,), (6,), (6, 6)))
    y = x.layerNorm(gain, bias).gatedMatMul(w, w)
    y.backward(1.0)
    assert not any(t.isOutsourced() for t in (gain, bias, w))
    assert all(t.gradient is not None and t.gradient.shape == t.shape for t in (x, gain, bias, w))


def test_two_handles_of_the_device_do_not_mix(device):
    """A second handle has a stream and workspace of its own; tensors of the one are refused by the other."""
    from neureka_amd import HipDevice, IllegalStateException
    other = HipDevice(0)
    try:
        rng = np.random.default_rng(15)
        x, wg, wu = (rng.standard_normal(s).astype(np.float32) for s in ((30, 3000), (3000, 40), (3000, 40)))
        a = put(device, x).gatedMatMul(put(device, wg), put(device, wu))
        b = put(other, x).gatedMatMul(put(other, wg), put(other, wu))
        assert_bits(get(a), get(b), "either handle")
        mine, theirs = put(device, x[:, :40]), put(other, np.ones(40, np.float32))
        with pytest.raises(IllegalStateException):
            mine.layerNorm(theirs, theirs)
        with pytest.raises(IllegalStateException):
            device.launch_dropout(put(other, x), put(device, x), 0.5, 1)
        with pytest.raises(IllegalStateException):
            mine.gatedMatMul(put(other, wg[:40]), put(other, wu[:40]))
        del b, theirs
    finally:
        other.dispose()


# ---- products large enough for two half-precision planes -----------------------------------------------------------

LARGE = [(1300, 1310, 1290), (1111, 2000, 1003), (4099, 500, 1100), (700, 3000, 1100)]


def rows_of(device, x, wg, wu, along=False):
    """gate and up of a product, straight from the device."""
    M, N = x.shape[0], wg.shape[1]
    gate, up = (device.allocate(np.float32, M * N) for _ in range(2))
    put_w = (lambda w: put(device, np.ascontiguousarray(w.T)).T()) if along else (lambda w: put(device, w))
    device.launch_gated_matmul("idy", put(device, np.zeros((M, N), np.float32)), put(device, x), put_w(wg), put_w(wu), gate, up)
    return [device._read_all(d).reshape(M, N) for d in (gate, up)]


@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("M,K,N", LARGE)
def test_large_gated_products_and_gradients(device, along, M, K, N):
    check_gated(device, np.float32, "silu", M, K, N, along)


@pytest.mark.parametrize("along", [False, True])
def test_large_gated_products_of_integers_are_exact(device, along):
    """Integers of up to 11 bits are halves: every partial product and sum below 2^24 is exact."""
    rng = np.random.default_rng(20)
    M, K, N = 1301, 1307, 1299
    x = rng.integers(-30, 31, (M, K)).astype(np.float32)
    wg, wu = (rng.integers(-30, 31, (K, N)).astype(np.float32) for _ in range(2))
    for got, w in zip(rows_of(device, x, wg, wu, along), (wg, wu)):
        assert (got == x.astype(np.float64) @ w.astype(np.float64)).all()


def test_large_gated_rows_of_any_magnitude_keep_their_digits(device):
    """Rows and columns from 2^-100 to 2^100, zero rows and columns, and rows whose entries lie 2^30 apart (with and without a
    counterpart): each result is as exact as its own terms allow."""
    rng = np.random.default_rng(21)
    M, K, N = 1200, 1400, 1310
    x = (rng.standard_normal((M, K)) * 2.0 ** rng.integers(-50, 50, (M, 1))).astype(np.float32)
    wg, wu = ((rng.standard_normal((K, N)) * 2.0 ** rng.integers(-50, 50, (1, N))).astype(np.float32) for _ in range(2))
    x[5], wg[:, 7], wu[:, 1309] = 0, 0, 0
    x[300:310, 100] *= 2.0 ** 30                            # one entry far above its row ...
    wg[100], wu[100] = 0, 0                                 # ... that meets nothing
    wg[200, 600:640] *= 2.0 ** 30
    x[1199, :700] *= 2.0 ** -30                             # half a row far below the other half
    for got, w in zip(rows_of(device, x, wg, wu), (wg, wu)):
        X, W = x.astype(np.float64), w.astype(np.float64)
        want = X @ W
        over = np.abs(want) > np.finfo(np.float32).max       # (2^50 2^50 2^30: a few sums leave the type's range)
        assert (got[over] == np.sign(want[over]) * np.inf).all()
        within(got[~over], want[~over], (sum_roundings(K) * unit(np.float32) * (np.abs(X) @ np.abs(W)))[~over], "gate or up")


def test_large_gated_infinities_and_nan(device):
    rng = np.random.default_rng(22)
    M, K, N = 1200, 1400, 1310
    x, wg, wu = (rng.standard_normal(s).astype(np.float32) for s in ((M, K), (K, N), (K, N)))
    x[0, 3], x[700, 4], x[M - 1, K - 1] = np.inf, np.nan, -np.inf
    wg[7, 11], wu[8, N - 1] = np.inf, -np.inf
    with np.errstate(all="ignore"):
        for got, w in zip(rows_of(device, x, wg, wu), (wg, wu)):
            X, W = x.astype(np.float64), w.astype(np.float64)
            fine_x, fine_w = np.isfinite(X).all(1), np.isfinite(W).all(0)
            want = np.where(np.isfinite(X), X, 0) @ np.where(np.isfinite(W), W, 0)
            for i in np.flatnonzero(~fine_x):
                want[i] = (X[i][:, None] * W).sum(0)
            for j in np.flatnonzero(~fine_w):
                want[:, j] = (X * W[:, j]).sum(1)
            assert (np.isnan(got) == np.isnan(want)).all() and (np.where(np.isinf(want), got == want, True)).all()
            ok = np.isfinite(want)
            amount = np.abs(np.where(np.isfinite(X), X, 0)) @ np.abs(np.where(np.isfinite(W), W, 0))
            within(got[ok], want[ok], sum_roundings(K) * unit(np.float32) * amount[ok], "finite ones")


@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("spread", [12, 40])
def test_large_gated_scales_that_undo_each_other(device, along, spread):
    """The columns of x times powers of two, the rows of the weights divided by them: every product counts alike, the small entries of
    either operand no less than the large ones."""
    rng = np.random.default_rng(23)
    M, K, N = 1200, 1400, 1310
    by = 2.0 ** rng.integers(-spread, spread + 1, K)
    x = (rng.standard_normal((M, K)) * by).astype(np.float32)
    wg, wu = ((rng.standard_normal((K, N)) / by[:, None]).astype(np.float32) for _ in range(2))
    for got, w in zip(rows_of(device, x, wg, wu, along), (wg, wu)):
        X, W = x.astype(np.float64), w.astype(np.float64)
        within(got, X @ W, sum_roundings(K) * unit(np.float32) * (np.abs(X) @ np.abs(W)), "gate or up")


def test_large_gated_gradients_with_scales_that_undo_each_other(device):
    """The same for d_X (columns of the weights against those of the error) and the weights' gradients (rows of x against those of
    the error), with the products as plain factors."""
    rng = np.random.default_rng(24)
    M, K, N = 1200, 1400, 1310
    one = device.allocateFromOne(np.float32, M * N, 1.0)      # gate = up = 1, the identity: dg = du = error
    for axis in (0, 1):
        by = 2.0 ** rng.integers(-40, 41, (M, 1) if axis == 0 else (1, N))
        x = (rng.standard_normal((M, K)) * (by if axis == 0 else 1)).astype(np.float32)
        wg, wu = ((rng.standard_normal((K, N)) * (by if axis == 1 else 1)).astype(np.float32) for _ in range(2))
        e = (rng.standard_normal((M, N)) / by).astype(np.float32)
        X, G, U, E = (a.astype(np.float64) for a in (x, wg, wu, e))
        d_x, d_g, d_u = (put(device, np.zeros(s, np.float32)) for s in ((M, K), (K, N), (K, N)))
        device.launch_gated_matmul_backward("idy", put(device, x), put(device, wg), put(device, wu), one, one, put(device, e), d_x, d_g, d_u)
        r = unit(np.float32)
        within(get(d_x), E @ (G + U).T, sum_roundings(2 * N) * r * (np.abs(E) @ (np.abs(G) + np.abs(U)).T), "dX")
        for got in (d_g, d_u):
            within(get(got), X.T @ E, sum_roundings(M) * r * (np.abs(X.T) @ np.abs(E)), "dW")


def test_axes_beyond_a_launch_are_refused(device):
    """A launch has fewer than 2^32 threads: axes that would need more are refused, whatever the buffers hold."""
    from neureka_amd._lib import FUN
    lib, h, p = device._lib, device.handle, put(device, np.zeros(4, np.float32))._data.ptr
    for axis in range(3):
        axes = [1, 1, 1]
        axes[axis] = (1 << 27) - 1023
        for dt in (0, 1):
            assert lib.nk_gated_matmul(h, FUN["silu"], dt, 0, *axes, p, p, p, p, 0, 0) != 0
            assert b"2^27" in lib.nk_last_error()
    assert lib.nk_layer_norm(h, 0, 1, (1 << 27) - 1023, p, 1 << 27, p, p, 1e-5, p, 0, 0) != 0
    assert b"2^27" in lib.nk_last_error()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("M,K,N", [(100, 1, 1), (100, 1, 40), (100, 40, 1), (5, 1, 40), (5, 40, 1), (70, 2, 3), (130, 3, 2), (80, 65, 33), (80, 33, 65)])
def test_gated_products_with_thin_axes_are_exact(device, dt, along, M, K, N):
    """Axes of one to three elements and one past a tile, where columns are read by twos."""
    test_gated_products_of_small_integers_are_exact(device, dt, along, M, K, N)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("along", [False, True])
@pytest.mark.parametrize("M,K,N", [(1, 3001, 1301), (20, 3001, 1301), (40, 500, 701), (64, 1501, 700), (33, 1700, 1600)])
def test_gated_few_rows_in_parts_and_on_tiles(device, dt, along, M, K, N):
    """Parts that do not divide the contraction, and both sides of the choice between few rows and tiles."""
    check_gated(device, dt, "gelu", M, K, N, along)
