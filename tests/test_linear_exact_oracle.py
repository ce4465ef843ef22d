"""The whole-number inputs of the linear layer's tests: they are what they claim
to be, and a product that leaves something out or counts it twice differs."""
import numpy as np
import pytest

import linear_exact
from linear_cases import decode, encode


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_inputs_are_exact(kind):
    v = linear_exact.inputs(501, 40, 24, 1)
    for a in v.values():
        assert np.array_equal(decode(encode(a, kind), kind), a)
    got = linear_exact.backward(v, "relu", kind)
    assert np.array_equal(got["dw"], v["delta"].astype(np.int64).T @ v["x"].astype(np.int64))
    assert np.array_equal(got["db"], v["delta"].astype(np.int64).sum(0))
    y, z = linear_exact.forward(v, "none", kind, "f32")
    want = v["x"].astype(np.int64) @ v["w"].astype(np.int64).T + v["bias"].astype(np.int64)
    assert np.array_equal(y, want + v["residual"].astype(np.int64)) and np.array_equal(z, decode(encode(want, kind), kind))


# Rows left out or doubled: a tile of 64, of 128, the tail, one part of a split, one row.
@pytest.mark.parametrize("first,last", [(0, 64), (6400, 6528), (20011 // 64 * 64, 20011), (4096, 4096 + 640), (20010, 20011)])
def test_rows_left_out_show(first, last):
    v = linear_exact.inputs(20011, 40, 24, 2)
    want = linear_exact.backward(v, "none", "f16")
    for factor in (0.0, 2.0):
        planted = dict(v, delta=v["delta"].copy())
        planted["delta"][first:last] *= factor
        got = linear_exact.backward(planted, "none", "f16")
        for k in ("dw", "db"):
            with pytest.raises(AssertionError):
                linear_exact.equal(got[k], want[k], k)


# The same along the inner dimension of y, by steps of 8, 32 and 64 and the tail.
@pytest.mark.parametrize("first,last", [(0, 64), (32, 64), (8, 16), (1096, 1101), (1100, 1101)])
def test_terms_left_out_show(first, last):
    v = linear_exact.inputs(70, 1101, 24, 3)
    want, _ = linear_exact.forward(v, "none", "bf16", "f32")
    for factor in (0.0, 2.0):
        planted = dict(v, x=v["x"].copy())
        planted["x"][:, first:last] *= factor
        got, _ = linear_exact.forward(planted, "none", "bf16", "f32")
        with pytest.raises(AssertionError):
            linear_exact.equal(got, want, "y")
