"""The relative bounds on activations and derivatives: 32-bit evaluations that
keep their accuracy in the tails are within them, ones that lose it or leave a
tail out are not."""
import numpy as np
import pytest

from activation_bounds import A, B, arguments, derivative, value
from linear_cases import ACTS, act, slope

F = np.float32
ONE = F(1.0)


def _sigmoid(t):
    return ONE / (ONE + np.exp(-t))


def _slope(t):
    e = np.exp(-np.abs(t))
    r = ONE / (ONE + e)
    return e * r * r


def _softplus(z):
    e = np.exp(-np.abs(z))
    u = ONE + e
    d = u - ONE
    with np.errstate(invalid="ignore", divide="ignore"):
        return np.maximum(z, F(0)) + np.where(d == 0, e, e * np.log(u) / d)


def _inner(z):
    return F(2.0 * A) * z * (ONE + F(B) * z * z)


VALUES = {"sigmoid": _sigmoid, "silu": lambda z: z * _sigmoid(z), "softplus": _softplus, "gelu": lambda z: z * _sigmoid(_inner(z))}
DERIVATIVES = {"sigmoid": _slope, "softplus": _sigmoid, "silu": lambda z: _sigmoid(z) + z * _slope(z), "gelu": lambda z: _sigmoid(_inner(z)) + z * _slope(_inner(z)) * F(2.0 * A) * (ONE + F(3.0 * B) * z * z)}
# Formulas that cancel.
LOSSY_VALUES = {"softplus": lambda z: np.maximum(z, F(0)) + np.log(ONE + np.exp(-np.abs(z))), "gelu": lambda z: F(0.5) * z * (ONE + np.tanh(F(0.5) * _inner(z))), "sigmoid": lambda z: F(0.5) * (ONE + np.tanh(F(0.5) * z)),
                "silu": lambda z: z * F(0.5) * (ONE + np.tanh(F(0.5) * z))}
LOSSY_DERIVATIVES = {"sigmoid": lambda z: _sigmoid(z) * (ONE - _sigmoid(z)), "silu": lambda z: _sigmoid(z) + z * F(0.5) * (ONE + np.tanh(F(0.5) * z)) * (ONE - _sigmoid(z)), "softplus": LOSSY_VALUES["sigmoid"],
                     "gelu": lambda z: F(0.5) * (ONE + np.tanh(F(0.5) * _inner(z))) + z * _sigmoid(_inner(z)) * (ONE - _sigmoid(_inner(z))) * F(2.0 * A) * (ONE + F(3.0 * B) * z * z)}


@pytest.mark.parametrize("name", ["sigmoid", "silu", "softplus", "gelu"])
def test_bounds_accept_and_refuse(name):
    z = arguments(name).astype(F)
    for exact, good, bad in ((value, VALUES, LOSSY_VALUES), (derivative, DERIVATIVES, LOSSY_DERIVATIVES)):
        want, bound = exact(z.astype(np.float64), name)
        assert (np.abs(good[name](z) - want) <= bound).all()
        assert (np.abs(bad[name](z) - want) > 10.0 * bound).any()
        # Nothing where the tail is: every argument from -6 down and, for sigmoid', up.
        tail = (z < -6.0) | ((z > 6.0) & (exact is derivative) & (name == "sigmoid"))
        assert (np.abs(want[tail]) > 1e3 * bound[tail]).all()


@pytest.mark.parametrize("name", list(ACTS))
def test_definitions_agree(name):
    z = np.linspace(-4.0, 4.0, 200)
    assert np.abs(value(z, name)[0] - act(z, name)).max() < 1e-13
    assert np.abs(derivative(z, name)[0] - slope(z, name)).max() < 1e-13
