"""The linear layer's activations and their derivatives with errors relative to
their values, from small arguments to where they have all but vanished."""
import numpy as np
import pytest

from activation_bounds import arguments, derivative, value
from linear_cases import ACTS, decode, encode, rounding, within
from test_gpu_linear import run_backward, run_forward

pytestmark = pytest.mark.gpu

# One row; some; enough for the kernels that are not for few.
ROWS = (1, 40, 16600)
# Exponents of delta: what a 16-bit number holds.
EXPONENTS = {"f16": (-14, 15), "bf16": (-120, 120)}


def _inputs(name, kind, rows):
    z = decode(encode(np.resize(arguments(name), (rows, 256)), kind), kind)
    i = z.shape[1]
    return {"x": z, "w": np.eye(i), "bias": np.zeros(i), "residual": np.zeros(z.shape), "delta": np.ones(z.shape), "pre": z, "add": np.zeros(z.shape)}


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("act", list(ACTS))
def test_values(act, kind, rows):
    v = _inputs(act, kind, rows)
    want, bound = value(v["x"], act)
    y, pre = run_forward(v, kind, "f32", act, residual=False, bias=False)
    assert np.array_equal(pre, v["x"])
    within(y, want, bound, act)
    # Rounded once to 16 bits.
    y, _ = run_forward(v, kind, kind, act, residual=False, pre=False)
    within(y, want, bound + rounding(np.abs(want) + bound, kind), act)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("act", list(ACTS))
def test_derivatives(act, kind, rows):
    """delta is the power of two that brings the product near 1, so that no tail is
    lost below the range of 16 bits."""
    v = _inputs(act, kind, rows)
    want, bound = derivative(v["pre"], act)
    v["delta"] = np.ldexp(1.0, np.clip(np.ceil(-np.log2(np.maximum(np.abs(want), 2.0**-200))), *EXPONENTS[kind]).astype(int))
    got = run_backward(v, kind, act, dw=False, db=False)
    assert np.array_equal(got["dx"], v["delta"])
    want, bound = want * v["delta"], bound * v["delta"]
    within(got["dpre"], want, bound + rounding(np.abs(want) + bound, kind), act)
