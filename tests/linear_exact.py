"""Inputs of the linear layer whose sums are whole numbers below 2^24, so exact
in 32 bits in any order: outputs have to be equal to these, rounded once to
their type, and a row, tile or part that is left out or counted twice shows."""
import numpy as np

from linear_cases import decode, encode


def _whole(rng, shape, most):
    return rng.integers(-most, most + 1, shape).astype(np.float64)


def inputs(n, i, o, seed, most=2, wide=8):
    """Factors of at most `most`, addends of at most `wide`; pre is never 0, where a
    relu has no derivative."""
    rng = np.random.default_rng(seed)
    longest = max(n, i, o)
    assert most * most * longest + 2 * wide < 1 << 24
    pre = _whole(rng, (n, i), 3)
    return {"x": _whole(rng, (n, i), most), "w": _whole(rng, (o, i), most), "bias": _whole(rng, (o,), wide), "residual": _whole(rng, (n, o), wide), "delta": _whole(rng, (n, o), most), "pre": np.where(pre == 0.0, 1.0, pre),
            "add": _whole(rng, (n, i), wide)}


def _product(a, b):
    """Exact: the sums are whole numbers below 2^24 in any order."""
    return (a.astype(np.float32) @ b.astype(np.float32)).astype(np.float64)


def _stored(values, kind):
    return decode(encode(values, kind), kind)


def forward(v, act, kind, y_kind, bias=True, residual=True):
    z = _product(v["x"], v["w"].T)
    if bias:
        z += v["bias"]
    y = np.maximum(z, 0.0) if act == "relu" else z
    return _stored(y + v["residual"] if residual else y, y_kind), _stored(z, kind)


def backward(v, act, kind, add=True):
    g = _product(v["delta"], v["w"])
    if add:
        g = g + v["add"]
    return {"dx": _stored(g, kind), "dpre": _stored(g * (v["pre"] > 0.0) if act == "relu" else g, kind), "dw": _product(v["delta"].T, v["x"]), "db": v["delta"].sum(0)}


def equal(got, want, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = got != want
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} differ, first at {np.argwhere(bad)[0]}: got {got[bad][0]!r} want {want[bad][0]!r}"
