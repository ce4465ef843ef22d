"""The optimiser's calls with nothing to update: what they report is written all
the same."""
import ctypes as C

import numpy as np
import pytest

from nerf_amd import _lib as L
from nerf_amd.device import DeviceArray, synchronize

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [0, 1, 70])
@pytest.mark.parametrize("norm,guard,want", [(3.0, 1e30, 0), (np.inf, 1e30, 1), (np.nan, 1e30, 1), (300.0, 2.0, 1)])
def test_skipped_of_empty_lists(count, norm, guard, want):
    """No tensor, and tensors of no elements."""
    hyper = L.NerfHyperParams(1e-2, 0.9, 0.99, 1e-8, 1e30, guard, 128.0, 0)
    tensors = (L.NerfExtAdamTensor * max(count, 1))(*[L.NerfExtAdamTensor(None, None, None, None, None, 0, 0, 0)] * max(count, 1))
    n, skipped = DeviceArray.from_numpy(np.array([norm], np.float32)), DeviceArray.from_numpy(np.array([7, 7], np.uint32))
    L.call("nerf_ext_adam_step", tensors, count, C.byref(hyper), 3, n.ptr, skipped.ptr, None)
    L.call("nerf_ext_adam_step", tensors, count, C.byref(hyper), 3, n.ptr, None, None)
    synchronize()
    assert skipped.numpy().tolist() == [want, 7]
