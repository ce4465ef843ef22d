"""The widest rows that a layer with adapters may have, without an index: fp32 outputs
more than 2^19 values apart, so that 1024 rows are beyond 32-bit offsets."""
import ctypes as C

import numpy as np
import pytest

import grouped_cases as G
from conftest import announce
from linear_exact import equal
from nerf_amd import _lib as L, ext
from nerf_amd.device import DeviceArray, synchronize
from nerf_amd.network import adapter_linear_forward

pytestmark = pytest.mark.gpu


def test_widest_rows_of_many(lib):
    announce("fp32 outputs 2^19 + 8 values apart")
    n, i, o, rank, stride = 65536, 32, 64, 16, (1 << 19) + 8
    free, total = C.c_size_t(), C.c_size_t()
    assert C.CDLL("libamdhip64.so").hipMemGetInfo(C.byref(free), C.byref(total)) == 0
    if free.value < 4 * n * stride + (8 << 30):
        pytest.skip("needs 146 GB of device memory")
    c = G.Case(n, 3, i, o, "bf16", seed=5, rank=rank, whole=True)
    d, mid, y = G.Device(c), G.Out((n, rank), "f32"), DeviceArray((n, stride), np.float32)
    desc = L.NerfExtLinearDesc(n, i, o, L.NERF_EXT_BF16, L.NERF_EXT_F32, L.NERF_EXT_ACT_NONE, 0, stride, 0, 0)
    rows = np.concatenate([np.arange(k, k + 8) for k in (0, 504, 1016, 1024, 2040, 30000, n - 8)])
    for row in rows:
        ext.write_device(y.ptr + 4 * stride * int(row), np.full(2 * o, G.OLD, np.float32))
    adapter_linear_forward(desc, d.groups, d.adapters, d.x, d.w, y.ptr, mid.ptr, bias=d.bias)
    synchronize()
    want = G.forward(c, "none", "f32", residual=False)
    equal(mid.values(), want["mid"][0], "mid")
    for row in rows:
        got = ext.read_device(y.ptr + 4 * stride * int(row), (2 * o,), np.float32).astype(np.float64)
        equal(got[:o], want["y"][0][row], f"row {row}")
        assert (got[o:] == G.OLD).all(), f"written behind row {row}"
