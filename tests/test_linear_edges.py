"""Calls at the edges of what nerf_ext_linear_* accept, decided on the host: no
GPU work is started."""
import ctypes as C

import pytest

from nerf_amd import _lib as L

A = 1 << 20  # an address that is never followed


def _desc(**kw):
    d = L.NerfExtLinearDesc(4, 8, 16, L.NERF_EXT_F16, L.NERF_EXT_F16, L.NERF_EXT_ACT_RELU, 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("change", [dict(out_dtype=L.NERF_EXT_F32), dict(y_stride=24), dict(residual_stride=24), dict(y_stride=32, residual_stride=24), dict(rows=1, out_dtype=L.NERF_EXT_F32)])
def test_outputs_over_residuals_that_lie_otherwise(lib, change):
    """y over residual with another type or row stride: a row of y would lie over
    residuals that another workgroup has yet to read."""
    status = L.status_of("nerf_ext_linear_forward", C.byref(_desc(**change)), A, A, None, A, A, None, None, 0, None)
    assert status == L.NERF_STATUS_INVALID_USAGE
    assert "nerf_ext_linear_forward" in L.last_error() and "residual" in L.last_error()


@pytest.mark.parametrize("dx,dpre", [(A, None), (None, A), (A, A)])
def test_no_rows_and_no_weight_gradient(lib, dx, dpre):
    """Nothing to compute: nothing is launched, and arrays need not be there."""
    for arrays in ((None, None, None, None, None), (A, A, A, A, A)):
        x, w, delta, pre, add = arrays
        status = L.status_of("nerf_ext_linear_backward", C.byref(_desc(rows=0)), x, w, delta, pre, add, dx, dpre, None, None, None, 0, None)
        assert status == L.NERF_STATUS_OK, L.last_error()
