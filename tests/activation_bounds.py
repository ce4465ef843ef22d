"""Activations and their derivatives in 64 bits without cancellation, and bounds
on their 32-bit evaluation that are relative, also where the values are small.

Units of 2^-23, relative: the hardware's exp, log and reciprocal are taken to be
within 2 each, a rounding within 1/2.  exp(x) takes x log2(e), a constant and a
product rounded, so it is within |x| + 2.  Results below 2^-126 may be flushed."""
import numpy as np

from linear_cases import EPS, sigma

FLUSHED = 2.0**-126
A, B = np.sqrt(2.0 / np.pi), 0.044715


def gelu_argument(z):
    return 2.0 * A * z * (1.0 + B * z * z)


def value(z, name):
    """(act(z), bound)."""
    a = np.abs(z)
    if name == "sigmoid":  # exp, a sum, a reciprocal
        y, units = sigma(z), a + 6.0
    elif name == "silu":
        y, units = z * sigma(z), a + 7.0
    elif name == "gelu":  # the argument: seven roundings, 3.5 units of it in the exponent
        s = gelu_argument(z)
        y, units = z * sigma(s), 4.5 * np.abs(s) + 8.0
    elif name == "softplus":
        # e log(u) / (u - 1): exp, log and its constant, reciprocal, three products,
        # and 2.5 for the quotient's own error; then the sum.
        l = np.log1p(np.exp(-a))
        y = np.maximum(z, 0.0) + l
        return y, EPS * ((a + 16.0) * l + y) + FLUSHED
    else:
        y, units = np.where(z < 0, 0.0, z) if name == "relu" else z, np.zeros_like(z)
    return y, EPS * units * np.abs(y) + FLUSHED * (units > 0) * (1.0 if name == "sigmoid" else 1.0 + a)


def derivative(z, name):
    """(act'(z), bound)."""
    a = np.abs(z)
    if name in ("none", "relu"):
        return (z > 0).astype(np.float64) if name == "relu" else np.ones_like(z), np.zeros_like(z)
    if name == "softplus":
        return sigma(z), EPS * (a + 6.0) * sigma(z) + FLUSHED
    slope = sigma(z) * sigma(-z)
    if name == "sigmoid":  # exp, a sum, the reciprocal twice, two products
        return slope, EPS * (a + 10.0) * slope + FLUSHED
    if name == "silu":
        first, second = sigma(z), z * slope
        return first + second, EPS * ((a + 6.0) * first + (a + 12.0) * np.abs(second) + np.abs(first + second)) + FLUSHED * (1.0 + a)
    t = gelu_argument(z)
    first, second = sigma(t), z * sigma(t) * sigma(-t) * 2.0 * A * (1.0 + 3.0 * B * z * z)
    return first + second, EPS * ((4.5 * np.abs(t) + 6.0) * first + (4.5 * np.abs(t) + 18.0) * np.abs(second) + np.abs(first + second)) + FLUSHED * (1.0 + a * (2.0 + a * a))


def arguments(name):
    """Of both signs, from small to where the exponent reaches 80."""
    most = 9.5 if name == "gelu" else 78.0
    a = np.concatenate([np.geomspace(2.0**-10, most, 64), np.linspace(0.05, min(most, 24.0), 64)])
    return np.concatenate([a, -a])
