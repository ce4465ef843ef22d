"""Derivatives of the activations where the pre-activation is an infinity or a
NaN: a NaN stays one, and an infinity (which a finite value beyond the range of
16 bits is stored as) gives the derivative's limit."""
import numpy as np
import pytest

from test_gpu_linear import run_backward, run_forward

pytestmark = pytest.mark.gpu

# act'(-inf), act'(+inf), act'(NaN).  The relu's is (z > 0), which a NaN is not.
LIMITS = {"none": (1.0, 1.0, 1.0), "relu": (0.0, 1.0, 0.0), "softplus": (0.0, 1.0, np.nan), "sigmoid": (0.0, 0.0, np.nan), "silu": (0.0, 1.0, np.nan), "gelu": (0.0, 1.0, np.nan)}


def _values(pre):
    n, i = pre.shape
    return {"x": np.ones((n, i)), "w": np.eye(i), "bias": np.zeros(i), "residual": np.zeros((n, i)), "delta": np.full((n, i), 0.5), "pre": pre, "add": np.zeros((n, i))}


# One row, some rows, and enough rows for the kernels that are not for few.
@pytest.mark.parametrize("rows", [1, 70, 16500])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("act", list(LIMITS))
def test_derivatives_of_infinities_and_nan(act, kind, rows):
    pre = np.tile([-np.inf, np.inf, np.nan, -np.inf, np.nan, np.inf, 0.25, np.inf], (rows, 3))
    got = run_backward(_values(pre), kind, act, dx=False, dw=False, db=False)["dpre"]
    low, high, nan = LIMITS[act]
    for value, want in ((-np.inf, low), (np.inf, high), (np.nan, nan)):
        at = np.isnan(pre) if np.isnan(value) else pre == value
        assert np.array_equal(got[at], np.full(at.sum(), 0.5 * want), equal_nan=True), (value, np.unique(got[at]))
    assert np.isfinite(got[pre == 0.25]).all()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_a_finite_layer_has_finite_gradients(act):
    """z = -90000 is finite in 32 bits and y is 0; its copy in fp16 is -inf."""
    v = _values(np.zeros((5, 8)))
    v["x"], v["w"] = np.full((5, 8), -300.0), np.eye(8) * 300.0
    y, pre = run_forward(v, "f16", "f16", act, residual=False)
    assert not y.any() and np.array_equal(pre, np.full((5, 8), -np.inf))
    assert not run_backward(_values(pre), "f16", act, dx=False, dw=False, db=False)["dpre"].any()
