"""The operators of a transformer's feed-forward sublayer, in plain torch and as this library offers them.

    y = layer_norm(x) * gain + bias          per row of x
    h = act(x @ gate) * (x @ up)             the gated half of a feed-forward block
    y = x * keep / (1 - p)                   keep from a counter-based generator, its mask never stored

Each for training (with the gradients of every input) and, where serving calls it, forward alone.  `run` computes the
plain form while `own` is false and calls the library while it is true.
"""
import numpy as np
import torch

own = False

EPSILON = 1e-5
DTYPES = {"f32": torch.float32, "f64": torch.float64}
ACTIVATIONS = ("silu", "gelu", "sig", "relu", "tanh", "idy")
LARGEST = 4096 ** 3              # multiply-adds of one projection in the largest case


def listed():
    return [
        # the norm in front of the projections while one token is generated: latency alone
        {"name": "norm of one token", "op": "norm", "rows": 1, "cols": 1024, "dtype": "f32", "train": False},
        # the norm over a prompt
        {"name": "norm of a prompt", "op": "norm", "rows": 4096, "cols": 4096, "dtype": "f32", "train": False},
        # a training step's norm on a ragged batch of rows of no special length
        {"name": "norm trained, odd", "op": "norm", "rows": 2047, "cols": 1111, "dtype": "f32", "train": True},
        # the same in double precision, as gradient checks and scientific models run it
        {"name": "norm trained, f64", "op": "norm", "rows": 4000, "cols": 2048, "dtype": "f64", "train": True},
        # dropout behind a sublayer of a large batch, both directions
        {"name": "dropout trained", "op": "dropout", "rows": 4096, "cols": 4096, "dtype": "f32", "p": 0.1},
        # a small odd tensor in double precision
        {"name": "dropout trained, odd, f64", "op": "dropout", "rows": 777, "cols": 1111, "dtype": "f64", "p": 0.5},
        # one token through both projections: bound by reading the weights
        {"name": "gated, one token", "op": "gated", "rows": 1, "inner": 4096, "cols": 4096, "act": "silu", "dtype": "f32", "transposed": False, "train": False},
        # sixteen sequences that generate together, weights stored one row per output
        {"name": "gated, 16 tokens", "op": "gated", "rows": 16, "inner": 4096, "cols": 4096, "act": "gelu", "dtype": "f32", "transposed": True, "train": False},
        # a prompt of odd length through layers of odd widths
        {"name": "gated, odd prompt", "op": "gated", "rows": 1111, "inner": 1000, "cols": 2500, "act": "sig", "dtype": "f32", "transposed": False, "train": False},
        # a training step of a mid-size layer, and of a large one
        {"name": "gated trained", "op": "gated", "rows": 2048, "inner": 1024, "cols": 4096, "act": "silu", "dtype": "f32", "transposed": False, "train": True},
        {"name": "gated trained, large", "op": "gated", "rows": 4096, "inner": 4096, "cols": 4096, "act": "silu", "dtype": "f32", "transposed": False, "train": True},
        # a training step in double precision
        {"name": "gated trained, f64", "op": "gated", "rows": 512, "inner": 512, "cols": 2048, "act": "tanh", "dtype": "f64", "transposed": False, "train": True},
    ]


def draw(rng):
    def size(lo, hi):
        """Spread over the logarithm of the range; every other one odd."""
        n = int(round(2 ** rng.uniform(np.log2(lo), np.log2(hi))))
        return min(hi, n | 1) if rng.random() < 0.5 else max(lo, n & ~1 if n > 1 else n)
    op = rng.choice(("norm", "dropout", "gated"))
    dtype = rng.choice(("f32", "f32", "f64"))
    if op == "norm":
        cols = size(16, 16384)
        return {"op": op, "rows": size(1, max(2, min(16384, 2 ** 24 // cols))), "cols": cols, "dtype": dtype, "train": rng.random() < 0.5}
    if op == "dropout":
        cols = size(16, 16384)
        return {"op": op, "rows": size(1, max(2, min(16384, 2 ** 24 // cols))), "cols": cols, "dtype": dtype, "p": round(rng.uniform(0.05, 0.6), 3)}
    inner, cols = size(64, 4096), size(64, 4096)
    most = LARGEST if dtype == "f32" else LARGEST // 16
    train = rng.random() < 0.5
    # (relu's slope jumps at 0: where two sums of 32-bit products disagree on a sign, so do whole gradients, rightly)
    act = rng.choice([a for a in ACTIVATIONS if not (train and a == "relu")])
    return {"op": op, "rows": size(1, max(2, min(4096, most // (inner * cols)))), "inner": inner, "cols": cols, "act": act,
            "dtype": dtype, "transposed": rng.random() < 0.5, "train": train}


def work(case):
    item = 4 if case["dtype"] == "f32" else 8
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "norm":
        # x in, y out; trained: the error in and the gradient out as well; ~8 operations a value and direction
        both = 2 if case["train"] else 1
        return {"bytes": item * (2 * rows * cols * both + 2 * cols * both), "flops": 8 * rows * cols * both}
    if case["op"] == "dropout":
        # x and the error in, y and the gradient out; ten rounds of the generator for four values
        return {"bytes": item * 4 * rows * cols, "flops": 2 * rows * cols * (1 + 25)}
    inner = case["inner"]
    ends = item * (rows * inner + 2 * inner * cols + rows * cols)
    products = 4 * rows * inner * cols
    if case["train"]:
        # x, weights and the error in; h and three gradients out; two products forward, four backward
        return {"bytes": 2 * ends, "flops": 3 * products}
    return {"bytes": ends, "flops": products}


# ---- inputs ----------------------------------------------------------------------------------------------------

class _Shared:
    """A tensor of the library seen by torch without a copy (both are memory of the same card)."""

    def __init__(self, tensor):
        self.tensor = tensor                     # keeps the memory while torch looks at it
        self.__cuda_array_interface__ = {"shape": tensor.shape, "typestr": "<f8" if tensor.dtype.itemsize == 8 else "<f4",
                                         "data": (tensor._data.ptr, False), "strides": None, "version": 3}


def _seen(tensor):
    return torch.as_tensor(_Shared(tensor), device="cuda")


def _given(x):
    """The values of `x` in a tensor of the library."""
    from neureka_amd import HipDevice, Tensor
    t = Tensor.of(np.float64 if x.dtype == torch.float64 else np.float32, tuple(x.shape), 0.0).to(HipDevice.get(0)).setIsVirtual(False)
    torch.cuda.synchronize()                     # the library's own stream has filled it
    _seen(t).copy_(x)
    return t


def _inputs(case, seed):
    """The inputs as plain torch tensors, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)
    rows, cols = case["rows"], case["cols"]
    if case["op"] == "norm":
        # activations of a residual stream: channels of different spread and offset
        x = normal(rows, cols) * torch.exp(0.5 * normal(1, cols)) + 0.3 * normal(1, cols)
        given = {"x": x, "gain": 1 + 0.1 * normal(cols), "bias": 0.1 * normal(cols)}
    elif case["op"] == "dropout":
        given = {"x": normal(rows, cols)}
    else:
        inner = case["inner"]
        shape = (cols, inner) if case["transposed"] else (inner, cols)
        given = {"x": normal(rows, inner), "gate": normal(*shape) / inner ** 0.5, "up": normal(*shape) / inner ** 0.5}
    if case["op"] == "dropout" or case["train"]:
        given["error"] = 0.1 * normal(rows, cols)
    return given


def prepare(case, seed):
    given = _inputs(case, seed)
    state = {"case": case, "seed": 0x9E3779B97F4A7C15 ^ seed, "offset": seed % 1000 + (1 << 33)}
    if not own:
        return {**state, **given}
    from neureka_amd import HipDevice, Tensor
    state["device"] = HipDevice.get(0)
    held = {k: _given(v) for k, v in given.items()}
    if case["op"] == "gated" and case["transposed"]:
        held["gate"], held["up"] = held["gate"].T(), held["up"].T()
    if "error" in held:
        for k, t in held.items():
            t.setRqsGradient(k != "error")
    else:                                        # a serving program keeps its output buffer
        x = held["x"]
        state["y"] = Tensor.of(x.dtype, (case["rows"], case["cols"]), 0.0).to(state["device"]).setIsVirtual(False)
        state["y_seen"] = _seen(state["y"])
    torch.cuda.synchronize()
    return {**state, **held}


# ---- one pass --------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _trained_by_library(state) if "error" in state else _served_by_library(state)
    return {"norm": _plain_norm, "dropout": _plain_dropout, "gated": _plain_gated}[op](state)


def _served_by_library(s):
    if s["case"]["op"] == "norm":
        s["device"].launch_layer_norm(s["y"], s["x"], s["gain"], s["bias"], EPSILON)
    else:
        s["device"].launch_gated_matmul(s["case"]["act"], s["y"], s["x"], s["gate"], s["up"])
    return {"y": s["y_seen"]}


def _trained_by_library(s):
    c = s["case"]
    x = s["x"]
    x.gradient = None
    if c["op"] == "norm":
        s["gain"].gradient = s["bias"].gradient = None
        y = x.layerNorm(s["gain"], s["bias"], EPSILON)
        y.backward(s["error"])
        return {"y": _seen(y), "dx": _seen(x.gradient), "dgain": _seen(s["gain"].gradient), "dbias": _seen(s["bias"].gradient)}
    if c["op"] == "dropout":
        y = x.dropout(c["p"], s["seed"], s["offset"])
        y.backward(s["error"])
        return {"y": _seen(y), "dx": _seen(x.gradient)}
    s["gate"].gradient = s["up"].gradient = None
    y = x.gatedMatMul(s["gate"], s["up"], c["act"])
    y.backward(s["error"])
    return {"y": _seen(y), "dx": _seen(x.gradient), "dgate": _seen(s["gate"].gradient), "dup": _seen(s["up"].gradient)}


def _plain_norm(s):
    x, gain = s["x"], s["gain"]
    mean = x.mean(dim=1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(dim=1, keepdim=True) + EPSILON)
    hat = centred * rstd
    y = hat * gain + s["bias"]
    if "error" not in s:
        return {"y": y}
    e = s["error"]
    eg = e * gain
    dx = rstd * (eg - eg.mean(dim=1, keepdim=True) - hat * (eg * hat).mean(dim=1, keepdim=True))
    return {"y": y, "dx": dx, "dgain": (e * hat).sum(dim=0), "dbias": e.sum(dim=0)}


_M0, _M1, _W0, _W1, _LOW = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85, 0xFFFFFFFF


def _plain_words(n, seed, offset):
    """n words of Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): key = seed, counter =
    (index / 4, offset), word index % 4 of each block.  32-bit words in 64-bit integers, whose products wrap as unsigned ones."""
    block = torch.arange((n + 3) // 4, device="cuda", dtype=torch.int64)
    c0, c1 = block & _LOW, block >> 32
    c2 = torch.full_like(block, offset & _LOW)
    c3 = torch.full_like(block, (offset >> 32) & _LOW)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        p0, p1 = c0 * _M0, c2 * _M1
        c0, c1, c2, c3 = ((p1 >> 32) & _LOW) ^ c1 ^ k0, p1 & _LOW, ((p0 >> 32) & _LOW) ^ c3 ^ k1, p0 & _LOW
        k0, k1 = (k0 + _W0) & _LOW, (k1 + _W1) & _LOW
    return torch.stack((c0, c1, c2, c3), dim=1).reshape(-1)[:n]


def _plain_dropout(s):
    x, p = s["x"], s["case"]["p"]
    keep = (_plain_words(x.numel(), s["seed"], s["offset"]) >= int(p * 4294967296.0)).reshape(x.shape)
    scale = 1.0 / (1.0 - p)
    zero = torch.zeros((), device="cuda", dtype=x.dtype)
    return {"y": torch.where(keep, x * scale, zero), "dx": torch.where(keep, s["error"] * scale, zero)}


def _plain_act(name, g):
    """act(g) and its derivative, as this library defines its activations (relu keeps a hundredth of a negative value, gelu is
    the logistic approximation)."""
    if name == "idy":
        return g, torch.ones_like(g)
    if name == "relu":
        slope = torch.where(g >= 0, 1.0, 0.01).to(g.dtype)
        return g * slope, slope
    if name == "tanh":
        t = torch.tanh(g)
        return t, 1 - t * t
    k = 1.702 if name == "gelu" else 1.0
    s = 1 / (1 + torch.exp(-k * g))
    if name == "sig":
        return s, s * (1 - s)
    return g * s, s + k * g * s * (1 - s)


def _plain_gated(s):
    c, x = s["case"], s["x"]
    gate, up = (s["gate"].t(), s["up"].t()) if c["transposed"] else (s["gate"], s["up"])
    g, u = x @ gate, x @ up
    a, slope = _plain_act(c["act"], g)
    y = a * u
    if "error" not in s:
        return {"y": y}
    e = s["error"]
    dg, du = e * u * slope, e * a
    return {"y": y, "dx": dg @ gate.t() + du @ up.t(), "dgate": x.t() @ dg, "dup": x.t() @ du}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    given = {k: v.double() for k, v in _inputs(case, seed).items()}
    x = given["x"]
    if case["op"] == "dropout":
        keep = torch.from_numpy(_exact_keep(x.numel(), 0x9E3779B97F4A7C15 ^ seed, seed % 1000 + (1 << 33), case["p"])).reshape(x.shape).cuda()
        factor = keep.double() / (1.0 - case["p"])
        return {"y": x * factor, "dx": given["error"] * factor}
    leaves = {k: v.requires_grad_() for k, v in given.items() if k != "error"}
    with torch.enable_grad():
        if case["op"] == "norm":
            var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
            y = (x - mean) * torch.rsqrt(var + EPSILON) * leaves["gain"] + leaves["bias"]
        else:
            g, u = (torch.einsum("mk,nk->mn" if case["transposed"] else "mk,kn->mn", x, leaves[k]) for k in ("gate", "up"))
            act = {"idy": lambda v: v, "relu": lambda v: torch.maximum(v, 0.01 * v), "tanh": lambda v: 2 * torch.sigmoid(2 * v) - 1,
                   "sig": torch.sigmoid, "silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.sigmoid(1.702 * v)}[case["act"]]
            y = act(g) * u
        out = {"y": y.detach()}
        if case["train"]:
            for k, d in zip(leaves, torch.autograd.grad(y, list(leaves.values()), given["error"])):
                out["d" + k] = d.t().contiguous() if case["op"] == "gated" and case["transposed"] and k != "x" else d
    return out


def _exact_keep(n, seed, offset, p):
    """The same generator on the host, in unsigned 64-bit arithmetic."""
    u = np.uint64
    low, half = u(_LOW), u(32)
    block = np.arange((n + 3) // 4, dtype=u)
    c = [block & low, block >> half, np.full_like(block, offset & _LOW), np.full_like(block, offset >> 32 & _LOW)]
    key = [seed & _LOW, seed >> 32 & _LOW]
    for r in range(10):
        a, b = c[0] * u(_M0), c[2] * u(_M1)
        c = [(b >> half) ^ c[1] ^ u(key[0]), b & low, (a >> half) ^ c[3] ^ u(key[1]), a & low]
        key = [(key[0] + _W0) & _LOW, (key[1] + _W1) & _LOW]
    return (np.stack(c, axis=1).reshape(-1)[:n] >= u(int(p * 4294967296.0)))
