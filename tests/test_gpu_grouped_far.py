"""Grouped layers and adapters on arrays of more than 2^31 bytes that an index names
rows of, at sizes that take tiles and the sums over rows: kernels with 32-bit offsets
must not be taken.  And grouping around the sizes where one workgroup ends."""
import numpy as np
import pytest

import grouped_cases as G
from conftest import announce
from linear_cases import decode, encode
from linear_exact import equal
from nerf_amd import _lib as L, ext
from nerf_amd.device import DeviceArray, synchronize
from nerf_amd.network import adapter_linear_backward, adapter_linear_forward, grouped_linear_backward, grouped_linear_forward
from test_gpu_grouped import stored
from test_gpu_groups import check

pytestmark = pytest.mark.gpu

STRIDE, COUNT = 1 << 14, 140000  # rows of 32 KB, 4.6 GB of them
NAN = 0x7FFF


@pytest.fixture(scope="module")
def workspace():
    return DeviceArray((L.NERF_EXT_LINEAR_WORKSPACE,), np.uint8)


@pytest.fixture(scope="module")
def arrays():
    made = [DeviceArray((COUNT, STRIDE), np.uint16) for _ in range(4)]
    assert made[0].nbytes > 1 << 32
    return made


def far_row(row, n):
    """Row of the far array for row `row` of n: half of them at each end."""
    return np.where(row < n // 2, row, COUNT - n + row)


def put(array, values, n):
    """The n rows' values at the far array's ends, NaN behind each row's."""
    for rows in (slice(0, n // 2), slice(n // 2, n)):
        host = np.full((rows.stop - rows.start, STRIDE), NAN, np.uint16)
        host[:, : values.shape[1]] = encode(values[rows], "f16")
        ext.write_device(array.ptr + 2 * STRIDE * int(far_row(rows.start, n)), host)


def get(array, n, width):
    """The n rows, whose other values must be what put() left there."""
    out = []
    for rows in (slice(0, n // 2), slice(n // 2, n)):
        host = ext.read_device(array.ptr + 2 * STRIDE * int(far_row(rows.start, n)), (rows.stop - rows.start, STRIDE), np.uint16)
        assert (host[:, width:] == NAN).all(), "written between rows"
        out.append(decode(host[:, :width], "f16"))
    return np.concatenate(out)


@pytest.mark.parametrize("rank", [0, 12])
@pytest.mark.parametrize("i,o", [(64, 136), (72, 648), (648, 72)])
def test_tiles_and_sums_of_far_rows(workspace, arrays, i, o, rank):
    announce(f"far rows, {i} -> {o}, rank {rank}")
    n, (x, delta, y, dx) = 6000, arrays
    c = G.Case(n, 3, i, o, "f16", seed=i + rank, rank=rank, whole=True, gather=True, scatter=True)
    put(x, c.x, n)
    put(delta, c.delta, n)
    put(y, np.full((n, o), G.OLD), n)
    put(dx, np.full((n, i), G.OLD), n)
    d = G.Device(c)
    index = [DeviceArray.from_numpy(np.asarray(a, np.uint32)) for a in (c.offsets, far_row(c.x_rows, n), far_row(c.y_rows, n))]
    groups = L.NerfExtRowGroups(*[a.ptr for a in index], 3, COUNT, COUNT, 0)
    desc = L.NerfExtLinearDesc(n, i, o, L.NERF_EXT_F16, L.NERF_EXT_F16, L.NERF_EXT_ACT_NONE, STRIDE, STRIDE, 0, 0)
    want = G.forward(c, "none", "f16", residual=False)
    ref = G.backward(c, "none", add=False, mid=want["mid"][0] if rank else None)
    if rank:
        outs = {"mid": G.Out((n, rank), "f32"), "dmid": G.Out((n, rank), "f32"), "ddown": G.Out((3, rank, i), "f32"), "dup": G.Out((3, o, rank), "f32")}
        adapter_linear_forward(desc, groups, d.adapters, x.ptr, d.w, y.ptr, outs["mid"].ptr, bias=d.bias, workspace=workspace)
        adapter_linear_backward(desc, groups, d.adapters, x.ptr, d.w, delta.ptr, mid=outs["mid"].ptr, dx=dx.ptr, dmid=outs["dmid"].ptr, ddown=outs["ddown"].ptr, dup=outs["dup"].ptr, workspace=workspace)
    else:
        outs = {"dw": G.Out((3, o, i), "f32"), "db": G.Out((3, o), "f32")}
        grouped_linear_forward(desc, groups, x.ptr, d.w, y.ptr, bias=d.bias, workspace=workspace)
        grouped_linear_backward(desc, groups, x.ptr, d.w, delta.ptr, dx=dx.ptr, dweight=outs["dw"].ptr, dbias=outs["db"].ptr, workspace=workspace)
    synchronize()
    equal(get(y, n, o), stored(want["y"][0], "f16"), "y")
    equal(get(dx, n, i), stored(ref["dx"][0], "f16"), "dx")
    for k, out in outs.items():
        equal(out.values(), (want if k == "mid" else ref)[k][0], k)


def test_outputs_too_far_for_streamed_rows(workspace, arrays):
    """Rows and weights of the kernel that streams them, and outputs by an index beyond
    its 32-bit offsets: more than 2^31 bytes of an array of which each row is named."""
    announce("outputs too far for streamed rows")
    n, i, o, rank, y = 66000, 64, 64, 16, arrays[2]
    assert 2 * n * STRIDE > 1 << 31
    c = G.Case(n, 3, i, o, "f16", seed=5, rank=rank, whole=True, gather=True, scatter=True)
    d, mid = G.Device(c), G.Out((n, rank), "f32")
    desc = L.NerfExtLinearDesc(n, i, o, L.NERF_EXT_F16, L.NERF_EXT_F16, L.NERF_EXT_ACT_RELU, 0, STRIDE, 0, 0)
    y.fill_bytes(0xFF)
    adapter_linear_forward(desc, d.groups, d.adapters, d.x, d.w, y.ptr, mid.ptr, bias=d.bias, workspace=workspace)
    synchronize()
    want = G.forward(c, "relu", "f16", residual=False)
    equal(mid.values(), want["mid"][0], "mid")
    for first in range(0, n, 8250):
        host = ext.read_device(y.ptr + 2 * STRIDE * first, (8250, STRIDE), np.uint16)
        assert (host[:, o:] == 0xFFFF).all(), "written between rows"
        equal(decode(host[:, :o], "f16"), stored(want["y"][0][first : first + 8250], "f16"), f"y from row {first}")
    assert (ext.read_device(y.ptr + 2 * STRIDE * n, (64, STRIDE), np.uint16) == 0xFFFF).all(), "written behind the rows"


@pytest.mark.parametrize("n", [8191, 8192, 8193])
@pytest.mark.parametrize("groups", [1, 64, 4096])
def test_grouping_where_one_workgroup_ends(n, groups):
    announce(f"group_rows {n} rows, {groups} groups")
    check(np.random.default_rng(n).integers(0, groups + 1, n), groups)
    check(np.arange(n)[::-1] * groups // n, groups, place=False)
