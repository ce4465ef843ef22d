"""64-bit definitions of the linear layer, its gradients and the optimiser
operators, 16-bit conversions, and error bounds of the kernels' arithmetic,
shared by their tests."""
import numpy as np

from nerf_amd import _lib as L

ACTS = {"none": L.NERF_EXT_ACT_NONE, "relu": L.NERF_EXT_ACT_RELU, "softplus": L.NERF_EXT_ACT_SOFTPLUS, "sigmoid": L.NERF_EXT_ACT_SIGMOID, "silu": L.NERF_EXT_ACT_SILU, "gelu": L.NERF_EXT_ACT_GELU}
CODES = {"f16": L.NERF_EXT_F16, "bf16": L.NERF_EXT_BF16, "f32": L.NERF_EXT_F32}
# Half the distance between neighbours, relative to the value; the smallest
# normal number; the largest finite one.
UNIT = {"f16": 2.0**-11, "bf16": 2.0**-8, "f32": 2.0**-24}
TINY = {"f16": 2.0**-14, "bf16": 2.0**-126, "f32": 2.0**-126}
EPS = 2.0**-23


def encode(values, kind):
    """Values rounded to nearest even, as the bits the device stores."""
    v = np.ascontiguousarray(values, np.float32)
    if kind == "f32":
        return v
    if kind == "f16":
        return v.astype(np.float16).view(np.uint16)
    u = v.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(v), np.uint16(0x7FC0), r)


def decode(bits, kind):
    if kind == "f32":
        return np.asarray(bits, np.float64)
    if kind == "f16":
        return np.asarray(bits, np.uint16).view(np.float16).astype(np.float64)
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def sigma(t):
    e = np.exp(-np.abs(t))
    return np.where(t >= 0, 1.0 / (1.0 + e), e / (1.0 + e))


def act(z, name):
    if name == "relu":
        return np.where(z < 0, 0.0, z)
    if name == "softplus":
        return np.logaddexp(z, 0.0)
    if name == "sigmoid":
        return sigma(z)
    if name == "silu":
        return z * sigma(z)
    if name == "gelu":
        return 0.5 * z * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (z + 0.044715 * z**3)))
    return z


def slope(z, name):
    if name == "none":
        return np.ones_like(z)
    if name == "relu":
        return (z > 0).astype(np.float64)
    s = sigma(z)
    if name == "softplus":
        return s
    if name == "sigmoid":
        return s * sigma(-z)
    if name == "silu":
        return s + z * s * sigma(-z)
    a, b = np.sqrt(2.0 / np.pi), 0.044715
    t = 2.0 * a * (z + b * z**3)
    return sigma(t) + z * sigma(t) * sigma(-t) * 2.0 * a * (1.0 + 3.0 * b * z**2)


def rounding(y, kind):
    """Error of rounding y to a type: relative above its normal range, absolute below."""
    return UNIT[kind] * np.maximum(np.abs(y), TINY[kind])


def act_error(z, name):
    """Error of a 32-bit activation or derivative, its argument exact: the
    hardware's exp, log and reciprocal are within 2 units each, exp's argument is
    scaled by log2(e) with one rounding, which |t| multiplies, and a handful of
    roundings follow; |t| is at most 1.6 |z| (1 + 0.045 z^2) where the value has
    not reached its limit, 16 there at most.  32 covers the sum; the derivative
    of gelu multiplies it by its inner slope, at most 16."""
    if name in ("none", "relu"):
        return np.zeros_like(z)
    return 32.0 * EPS * np.maximum(1.0, np.minimum(np.abs(z), 128.0))


def forward(x, w, bias, residual, name, kind, y_kind):
    """(y, pre) in 64 bits and their error bounds.  A sum of k products in 32
    bits in any order is within (k + 2) EPS of the sum of their magnitudes; the
    activations' slopes are at most 1.13."""
    z = x @ w.T + (0.0 if bias is None else bias)
    size = np.abs(x) @ np.abs(w).T + (0.0 if bias is None else np.abs(bias))
    dz = (x.shape[1] + 2) * EPS * size
    y = act(z, name)
    dy = 1.13 * dz + act_error(z, name)
    if residual is not None:
        y = y + residual
        dy = dy + EPS * np.abs(y)
    return y, z, dy + rounding(np.abs(y) + dy, y_kind), dz + rounding(np.abs(z) + dz, kind)


def backward(x, w, delta, pre, add, name, kind):
    """{output: (value, bound)} in 64 bits."""
    g = delta @ w + (0.0 if add is None else add)
    dg = (w.shape[0] + 2) * EPS * (np.abs(delta) @ np.abs(w) + (0.0 if add is None else np.abs(add)))
    s = slope(pre, name)
    p = g * s
    dp = dg * np.abs(s) + (np.abs(g) + dg) * 16.0 * act_error(pre, name) + EPS * np.abs(p)
    n = x.shape[0] + 2
    return {"dx": (g, dg + rounding(np.abs(g) + dg, kind)), "dpre": (p, dp + rounding(np.abs(p) + dp, kind)), "dw": (delta.T @ x, n * EPS * (np.abs(delta).T @ np.abs(x)) + 2.0**-140),
            "db": (delta.sum(0), n * EPS * np.abs(delta).sum(0) + 2.0**-140)}


def within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not got.size:
        return
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} beyond the bound, first at {np.argwhere(bad)[0]}: got {got[bad][0]!r} want {want[bad][0]!r} bound {np.broadcast_to(bound, got.shape)[bad][0]!r}"
