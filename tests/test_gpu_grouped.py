"""Grouped linear layers and adapters, forward and backward: on whole numbers,
whose sums are exact in 32 bits, for equality; on random values against 64-bit
definitions within bounds of the arithmetic."""
import numpy as np
import pytest

import grouped_cases as G
from conftest import announce
from linear_cases import decode, encode, within
from linear_exact import equal
from nerf_amd import _lib as L
from nerf_amd.device import DeviceArray, synchronize
from nerf_amd.network import adapter_linear_backward, adapter_linear_forward, grouped_linear_backward, grouped_linear_forward

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def workspace():
    return DeviceArray((L.NERF_EXT_LINEAR_WORKSPACE,), np.uint8)


def run_forward(c, name, y_kind, ws, bias=True, residual=True, pre=True, **device):
    d = G.Device(c, **device)
    outs = {"y": G.Out((c.y_count, c.o), y_kind, d.y_pad, d.lead), "pre": G.Out((c.y_count, c.o), c.kind, 0, d.lead), "mid": G.Out((c.n, max(c.rank, 1)), "f32")}
    kw = dict(bias=d.bias if bias else None, residual=d.residual if residual else None, pre=outs["pre"].ptr if pre else None, workspace=ws)
    if c.rank:
        adapter_linear_forward(d.desc(name, y_kind), d.groups, d.adapters, d.x, d.w, outs["y"].ptr, outs["mid"].ptr, **kw)
    else:
        grouped_linear_forward(d.desc(name, y_kind), d.groups, d.x, d.w, outs["y"].ptr, **kw)
    synchronize()
    return {k: o.values() for k, o in outs.items() if (k != "pre" or pre) and (k != "mid" or c.rank)}


def run_backward(c, name, ws, mid=None, add=True, dx=True, dpre=True, sums=True, **device):
    d = G.Device(c, **device)
    outs = {"dx": G.Out((c.x_count, c.i), c.kind, d.x_pad, d.lead), "dpre": G.Out((c.x_count, c.i), c.kind, 0, d.lead)}
    kw = dict(pre=d.pre, add=d.add if add else None, dx=outs["dx"].ptr if dx else None, dpre=outs["dpre"].ptr if dpre else None, workspace=ws)
    if c.rank:
        outs |= {"dmid": G.Out((c.n, c.rank), "f32"), "ddown": G.Out((c.groups, c.rank, c.i), "f32"), "dup": G.Out((c.groups, c.o, c.rank), "f32")}
        m = DeviceArray.from_numpy(mid.astype(np.float32))
        adapter_linear_backward(d.desc(name), d.groups, d.adapters, d.x, d.w, d.delta, mid=m.ptr, dmid=outs["dmid"].ptr, ddown=outs["ddown"].ptr if sums else None, dup=outs["dup"].ptr if sums else None, **kw)
    else:
        outs |= {"dw": G.Out((c.groups, c.o, c.i), "f32"), "db": G.Out((c.groups, c.o), "f32")}
        grouped_linear_backward(d.desc(name), d.groups, d.x, d.w, d.delta, dweight=outs["dw"].ptr if sums else None, dbias=outs["db"].ptr if sums else None, **kw)
    synchronize()
    skipped = {"dx": not dx, "dpre": not dpre, "dw": not sums, "db": not sums, "ddown": not sums, "dup": not sums}
    return {k: o.values() for k, o in outs.items() if not skipped.get(k)}


def stored(values, kind):
    return decode(encode(values, kind), kind)


def forward_equal(c, name, y_kind, ws, **kw):
    want = G.forward(c, name, y_kind)
    got = run_forward(c, name, y_kind, ws, **kw)
    equal(got["y"], stored(want["y"][0], y_kind), "y")
    equal(got["pre"], stored(want["pre"][0], c.kind), "pre")
    if c.rank:
        equal(got["mid"], want["mid"][0], "mid")


def backward_equal(c, name, ws, **kw):
    mid = G.forward(c, name, c.kind)["mid"][0] if c.rank else None
    want = G.backward(c, name, mid=mid)
    got = run_backward(c, name, ws, mid=mid, **kw)
    for k in got:
        equal(got[k], stored(want[k][0], c.kind) if k in ("dx", "dpre") else want[k][0], k)


# rows, groups, in, out: whole chunks and odd widths, one to many tiles, more groups
# than rows, single values.
SHAPES = [(1, 1, 8, 8), (1, 4096, 16, 16), (3, 2, 1, 1), (40, 3, 1, 1), (40, 3, 2, 3), (5, 1, 1, 3), (37, 5, 7, 9), (64, 4, 64, 64), (129, 7, 63, 65), (200, 9, 96, 72), (300, 2, 256, 40), (500, 40, 33, 130), (700, 3, 8, 264), (1000, 300, 24, 16), (2000, 6, 128, 136), (3001, 5, 200, 100)]
INDEXES = [dict(), dict(gather=True, scatter=True, extra=11), dict(gather=True), dict(scatter=True, extra=3)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n,groups,i,o", SHAPES)
def test_grouped_whole_numbers(workspace, n, groups, i, o, kind):
    at = SHAPES.index((n, groups, i, o)) + (kind == "bf16")
    announce(f"grouped {n} x {i} -> {o}, {groups} groups, {kind}, {INDEXES[at % 4]}")
    c = G.Case(n, groups, i, o, kind, seed=at, whole=True, **INDEXES[at % 4])
    forward_equal(c, "relu", "f32" if at % 3 == 0 else kind, workspace)
    backward_equal(c, "relu", workspace)


@pytest.mark.parametrize("index", range(4))
@pytest.mark.parametrize("sizes", ["uneven", "one", "each", "none"])
def test_grouped_sizes(workspace, sizes, index):
    announce(f"grouped sizes {sizes}, {INDEXES[index]}")
    for n, i, o in ((77, 40, 48), (1500, 72, 33)):
        c = G.Case(n, 50, i, o, "bf16", seed=9, whole=True, sizes=sizes, **INDEXES[index])
        forward_equal(c, "none", "bf16", workspace)
        backward_equal(c, "none", workspace)


@pytest.mark.parametrize("n,groups,i,o,rank", [(1, 1, 8, 8, 1), (3, 2, 1, 1, 1), (40, 3, 1, 3, 2), (1, 40, 16, 16, 8), (33, 33, 64, 48, 16), (64, 5, 31, 65, 3), (150, 4, 128, 72, 16), (300, 90, 40, 24, 9), (500, 3, 65, 130, 33), (2000, 6, 96, 104, 64), (700, 2, 24, 264, 130),
                                               (260, 7, 200, 8, 256)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_adapter_whole_numbers(workspace, n, groups, i, o, rank, kind):
    at = n + (kind == "bf16")
    announce(f"adapter {n} x {i} -> {o}, {groups} groups, rank {rank}, {kind}")
    # Ranks and inputs are such that mid and its products stay whole and in the type's
    # two pieces (16 bits): mid is at most 2 in, its products 2 in out.
    c = G.Case(n, groups, i, o, kind, seed=at, rank=rank, whole=True, **INDEXES[at % 4])
    forward_equal(c, "relu", "f32" if at % 3 == 0 else kind, workspace)
    backward_equal(c, "relu", workspace)


@pytest.mark.parametrize("index", range(4))
@pytest.mark.parametrize("sizes", ["one", "each", "none"])
def test_adapter_sizes(workspace, sizes, index):
    announce(f"adapter sizes {sizes}, {INDEXES[index]}")
    for n, i, o in ((77, 40, 48), (1500, 72, 33)):
        c = G.Case(n, 50, i, o, "f16", seed=9, rank=12, whole=True, sizes=sizes, **INDEXES[index])
        forward_equal(c, "none", "f16", workspace)
        backward_equal(c, "none", workspace)


@pytest.mark.parametrize("rank", [0, 5])
@pytest.mark.parametrize("device", [dict(x_pad=3), dict(y_pad=5, lead=1), dict(x_pad=8, y_pad=16, lead=8), dict(lead=4)])
def test_strides_and_alignment(workspace, device, rank):
    announce(f"strides {device}, rank {rank}")
    for n, i, o in ((90, 40, 48), (600, 129, 64)):
        c = G.Case(n, 6, i, o, "f16", seed=3, rank=rank, whole=True, gather=True, scatter=True, extra=2)
        forward_equal(c, "relu", "f16", workspace, **device)
        backward_equal(c, "relu", workspace, **device)


@pytest.mark.parametrize("rank", [0, 17])
def test_without_workspace_and_optional_arrays(rank):
    announce(f"no workspace, rank {rank}")
    c = G.Case(5000, 3, 48, 40, "bf16", seed=4, rank=rank, whole=True)
    forward_equal(c, "relu", "bf16", None)
    backward_equal(c, "relu", None)
    small = DeviceArray((40 * 1024,), np.uint8)
    backward_equal(c, "relu", small)
    want = G.forward(c, "relu", "bf16", bias=False, residual=False)
    got = run_forward(c, "relu", "bf16", None, bias=False, residual=False, pre=False)
    equal(got["y"], stored(want["y"][0], "bf16"), "y")
    mid = want["mid"][0] if rank else None
    ref = G.backward(c, "relu", add=False, mid=mid)
    for kw in (dict(dpre=False, sums=False), dict(dx=False), dict(dx=False, dpre=False)):
        got = run_backward(c, "relu", None, mid=mid, add=False, **kw)
        for k in got:
            equal(got[k], stored(ref[k][0], "bf16") if k in ("dx", "dpre") else ref[k][0], k)


@pytest.mark.parametrize("name", ["none", "relu", "softplus", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("kind,y_kind", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("rank", [0, 16])
def test_random_values(workspace, name, kind, y_kind, rank):
    announce(f"random values {name}, {kind} -> {y_kind}, rank {rank}")
    c = G.Case(700, 6, 120, 88, kind, seed=5, rank=rank, gather=True, scatter=True)
    want, got = G.forward(c, name, y_kind), run_forward(c, name, y_kind, workspace)
    for k in got:
        within(got[k], *want[k], k)
    mid = want["mid"][0].astype(np.float32).astype(np.float64) if rank else None
    want, got = G.backward(c, name, mid=mid), run_backward(c, name, workspace, mid=mid)
    for k in got:
        within(got[k], *want[k], k)


# Enough rows for the kernels that stream them, and for tiles of every size.
LARGE = [(40001, 7, 256, 256), (70000, 300, 32, 64), (33000, 5, 128, 264), (33001, 3, 63, 64), (40000, 9, 64, 31), (36000, 11, 96, 32), (33000, 2, 256, 520), (20000, 3, 520, 264), (9000, 2, 1032, 1024), (5000, 20, 600, 300)]


@pytest.mark.parametrize("n,groups,i,o", LARGE)
@pytest.mark.parametrize("kind,index", [("f16", 1), ("bf16", 0)])
def test_grouped_many_rows(workspace, n, groups, i, o, kind, index):
    announce(f"grouped {n} x {i} -> {o}, {groups} groups, {kind}, {INDEXES[index]}")
    c = G.Case(n, groups, i, o, kind, seed=n, whole=True, **INDEXES[index])
    forward_equal(c, "relu", "f32" if kind == "bf16" else kind, workspace)
    backward_equal(c, "relu", workspace)


@pytest.mark.parametrize("n,groups,i,o,rank", [(66001, 7, 256, 256, 16), (66000, 300, 64, 64, 12), (65536, 5, 128, 264, 20), (66000, 3, 96, 72, 64), (66000, 4, 256, 512, 9), (33000, 2, 63, 64, 16), (20000, 3, 520, 264, 48), (9000, 2, 1032, 1024, 128), (5000, 20, 600, 300, 7)])
@pytest.mark.parametrize("kind,index", [("f16", 1), ("bf16", 0)])
def test_adapter_many_rows(workspace, n, groups, i, o, rank, kind, index):
    announce(f"adapter {n} x {i} -> {o}, {groups} groups, rank {rank}, {kind}, {INDEXES[index]}")
    c = G.Case(n, groups, i, o, kind, seed=n, rank=rank, whole=True, **INDEXES[index])
    forward_equal(c, "relu", "f32" if kind == "bf16" else kind, workspace)
    backward_equal(c, "relu", workspace)


@pytest.mark.parametrize("kind,y_kind", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
def test_adapter_many_random_rows(workspace, kind, y_kind):
    announce(f"adapter, many random rows, {kind} -> {y_kind}")
    c = G.Case(65600, 6, 128, 96, kind, seed=6, rank=16)
    want, got = G.forward(c, "silu", y_kind), run_forward(c, "silu", y_kind, workspace)
    for k in got:
        within(got[k], *want[k], k)
    mid = want["mid"][0].astype(np.float32).astype(np.float64)
    want, got = G.backward(c, "silu", mid=mid), run_backward(c, "silu", workspace, mid=mid)
    for k in got:
        within(got[k], *want[k], k)
