"""Rows put in groups by an id: equal to a stable sort, at sizes around the
kernels' turns and chunks, with ids in no group, of one group, with and without
a workspace and place."""
import numpy as np
import pytest

import grouped_cases as G
from conftest import announce
from nerf_amd import _lib as L
from nerf_amd.device import DeviceArray, Stream, synchronize
from nerf_amd.network import group_rows

pytestmark = pytest.mark.gpu


def run(ids, groups, workspace=L.NERF_EXT_GROUP_WORKSPACE, place=True, stream=None):
    n = len(ids)
    d = DeviceArray.from_numpy(np.asarray(ids, np.uint32) if n else np.zeros(1, np.uint32))
    outs = [DeviceArray.from_numpy(np.full(k + 8, 0xABCDEF01, np.uint32)) for k in (groups + 1, n, n)]
    ws = DeviceArray((workspace,), np.uint8) if workspace else None
    group_rows(d.ptr, n, groups, outs[0].ptr, outs[1].ptr, place=outs[2].ptr if place else None, workspace=ws, stream=stream)
    (stream.synchronize if stream else synchronize)()
    got = [o.numpy() for o in outs]
    for o, k in zip(got, (groups + 1, n, n if place else 0)):
        assert (o[k:] == 0xABCDEF01).all()
    return got[0][: groups + 1], got[1][:n], got[2][:n]


def check(ids, groups, **kw):
    got, want = run(ids, groups, **kw), G.group_rows(ids, groups)
    assert np.array_equal(got[0], want[0])
    assert np.array_equal(got[1], want[1])
    if kw.get("place", True):
        assert np.array_equal(got[2], want[2])


SIZES = [(0, 1), (1, 1), (1, 4096), (63, 3), (64, 64), (65, 127), (100, 128), (1023, 1), (1024, 1023), (4095, 1024), (4097, 64), (16384, 4096), (16385, 4096), (16385, 1), (40000, 127), (70001, 1000), (262147, 64), (1048577, 4095)]


@pytest.mark.parametrize("n,groups", SIZES)
def test_sizes(n, groups):
    announce(f"group_rows {n} rows, {groups} groups")
    rng = np.random.default_rng(n + groups)
    check(rng.integers(0, groups + max(1, groups // 20), n), groups)


@pytest.mark.parametrize("n,groups", [(5000, 50), (50001, 700)])
def test_contents(n, groups):
    rng = np.random.default_rng(1)
    announce(f"contents of {n} rows, {groups} groups")
    check(np.zeros(n, np.int64), groups)
    check(np.full(n, groups - 1), groups)
    check(np.full(n, 0xFFFFFFFF), groups)
    check(np.arange(n) % groups, groups)
    check(np.arange(n)[::-1] * groups // n, groups)
    check(np.where(rng.random(n) < 0.99, 7, rng.integers(0, groups, n)), groups, place=False)


@pytest.mark.parametrize("workspace", [0, 64, 16 * 1024, 200 * 1024])
def test_small_workspaces(workspace):
    announce(f"workspace of {workspace} bytes")
    check(np.random.default_rng(2).integers(0, 4096, 60001), 4095, workspace=workspace)
    check(np.random.default_rng(3).integers(0, 90, 60001), 80, workspace=workspace)


def test_same_every_time_on_streams():
    rng = np.random.default_rng(4)
    ids = [rng.integers(0, 300, 100003) for _ in range(2)]
    streams = [Stream(), Stream()]
    for _ in range(3):
        for i, s in zip(ids, streams):
            check(i, 290, stream=s)
