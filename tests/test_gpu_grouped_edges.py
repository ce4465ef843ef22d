"""Grouped layers and adapters at their edges: infinities and NaN that must not
reach other groups' rows or sums, index entries that are no rows, offsets beyond
the rows, values beyond fp16's range between the low-rank products, arrays
beyond 32-bit offsets, and the same bits every time."""
import numpy as np
import pytest

import grouped_cases as G
from conftest import announce
from linear_cases import decode, encode, within
from linear_exact import equal
from nerf_amd import _lib as L, ext
from nerf_amd.device import DeviceArray, synchronize
from nerf_amd.network import grouped_linear_backward, grouped_linear_forward
from test_gpu_grouped import run_backward, run_forward, stored

pytestmark = pytest.mark.gpu

SHAPES = [(60, 40, 24, 7), (900, 72, 136, 16), (3000, 33, 65, 5), (70000, 64, 64, 16)]


@pytest.fixture(scope="module")
def workspace():
    return DeviceArray((L.NERF_EXT_LINEAR_WORKSPACE,), np.uint8)


def outside_group(c, g):
    keep = np.ones(c.n, bool)
    keep[c.offsets[g] : c.offsets[g + 1]] = False
    return keep


@pytest.mark.parametrize("rank", [False, True])
@pytest.mark.parametrize("n,i,o,r", SHAPES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_one_group_does_not_reach_others(workspace, n, i, o, r, rank, bad):
    """A group whose weights or adapter, rows and deltas are NaN or infinite, and rows
    in no group with NaN: all others' outputs and sums are what they are without."""
    announce(f"non-finite group, {n} x {i} -> {o}, rank {r if rank else 0}")
    c = G.Case(n, 6, i, o, "bf16", seed=1, rank=r if rank else 0, whole=True, gather=True, scatter=True)
    g = int(np.argmax(np.diff(c.offsets)))
    want, mid = G.forward(c, "relu", "bf16"), None
    if rank:
        mid = want["mid"][0]
    ref = G.backward(c, "relu", mid=mid)
    keep, groups = outside_group(c, g), np.arange(6) != g
    xr, yr, rows = c.xr(), c.yr(), np.arange(c.n)
    loose = (rows < c.offsets[0]) | (rows >= c.offsets[-1])
    spoilt = ~keep | loose
    c.x[xr[spoilt]] = bad
    c.delta[yr[spoilt]] = bad
    if rank:
        c.down[g], c.up[g] = bad, bad
        mid = mid.copy()
        mid[spoilt] = bad
    else:
        c.w[g], c.bias[g] = bad, bad
    clean = ~spoilt
    got = run_forward(c, "relu", "bf16", workspace)
    equal(got["y"][yr[clean]], stored(want["y"][0], "bf16")[yr[clean]], "y")
    equal(got["pre"][yr[clean]], stored(want["pre"][0], "bf16")[yr[clean]], "pre")
    # (The relu takes a negative infinity to 0.)
    assert not np.isfinite(got["pre"][yr[~keep]]).any()
    if rank:
        equal(got["mid"][clean], want["mid"][0][clean], "mid")
    got = run_backward(c, "none", workspace, mid=mid, add=False)
    ref = G.backward(clean_case(c, spoilt, g), "none", add=False, mid=None if mid is None else np.where(spoilt[:, None], 0.0, mid))
    equal(got["dx"][xr[clean]], stored(ref["dx"][0], "bf16")[xr[clean]], "dx")
    for k in ("dw", "db", "ddown", "dup"):
        if k in got:
            equal(got[k][groups], ref[k][0][groups], k)


def clean_case(c, spoilt, g):
    """The case with zeros for what was spoilt."""
    out = G.Case.__new__(G.Case)
    out.__dict__.update(c.__dict__)
    out.x, out.delta = c.x.copy(), c.delta.copy()
    out.x[c.xr()[spoilt]], out.delta[c.yr()[spoilt]] = 0.0, 0.0
    for k in ("down", "up") if c.rank else ("w", "bias"):
        v = getattr(c, k).copy()
        v[g] = 0.0
        setattr(out, k, v)
    return out


@pytest.mark.parametrize("rank", [0, 9])
@pytest.mark.parametrize("n,i,o", [(50, 40, 24), (900, 72, 136), (1200, 33, 65)])
def test_index_entries_that_are_no_rows(workspace, n, i, o, rank):
    """An x_rows entry beyond the array reads as zeros, a y_rows entry beyond it is not
    written (and its delta reads as zeros)."""
    announce(f"entries that are no rows, {n} x {i} -> {o}, rank {rank}")
    c = G.Case(n, 5, i, o, "f16", seed=2, rank=rank, whole=True, gather=True, scatter=True, extra=9)
    rng = np.random.default_rng(3)
    no_x, no_y = rng.choice(n, n // 5, replace=False), rng.choice(n, n // 5, replace=False)
    x_rows, y_rows = c.x_rows.copy(), c.y_rows.copy()
    # The definition on rows of zeros behind the arrays; nothing there is compared.
    d = G.Case.__new__(G.Case)
    d.__dict__.update(c.__dict__)
    for name in ("x", "add", "pre"):
        setattr(d, name, np.concatenate([getattr(c, name), np.zeros((n, i))]))
    for name in ("residual", "delta"):
        setattr(d, name, np.concatenate([getattr(c, name), np.zeros((n, o))]))
    d.x_rows, d.y_rows = x_rows.copy(), y_rows.copy()
    d.x_rows[no_x], d.y_rows[no_y] = c.x_count + no_x, c.y_count + no_y
    d.x_count, d.y_count = c.x_count + n, c.y_count + n
    c.x_rows, c.y_rows = x_rows.astype(np.int64), y_rows.astype(np.int64)
    c.x_rows[no_x[::2]], c.x_rows[no_x[1::2]] = 0xFFFFFFFF, c.x_count
    c.y_rows[no_y[::2]], c.y_rows[no_y[1::2]] = 0xFFFFFFFF, c.y_count
    want, got = G.forward(d, "relu", "f16"), run_forward(c, "relu", "f16", workspace)
    for k in ("y", "pre"):
        equal(got[k], stored(want[k][0][: c.y_count], "f16"), k)
    if rank:
        equal(got["mid"], want["mid"][0], "mid")
    mid = want["mid"][0] if rank else None
    want, got = G.backward(d, "none", mid=mid), run_backward(c, "none", workspace, mid=mid)
    for k in got:
        equal(got[k], stored(want[k][0][: c.x_count], "f16") if k in ("dx", "dpre") else want[k][0], k)


@pytest.mark.parametrize("rank", [0, 8])
def test_offsets_beyond_the_rows(workspace, rank):
    announce(f"offsets beyond the rows, rank {rank}")
    for n in (70, 2000):
        c = G.Case(n, 6, 40, 48, "f16", seed=4, rank=rank, whole=True)
        c.offsets[3:] = [n, n, n, n]
        want = G.forward(c, "relu", "f16")
        mid = want["mid"][0] if rank else None
        ref = G.backward(c, "relu", mid=mid)
        c.offsets[4:] = [n + 5, n + 100000, 0xFFFFFFFF]
        got = run_forward(c, "relu", "f16", workspace)
        equal(got["y"], stored(want["y"][0], "f16"), "y")
        got = run_backward(c, "relu", workspace, mid=mid)
        for k in got:
            equal(got[k], stored(ref[k][0], "f16") if k in ("dx", "dpre") else ref[k][0], k)


@pytest.mark.parametrize("n", [300, 66000])
def test_low_rank_values_beyond_fp16(workspace, n):
    """mid and dmid far beyond 65504, and far below fp16's normal numbers."""
    announce(f"low-rank values beyond fp16, {n} rows")
    c = G.Case(n, 4, 64, 64, "f16", seed=5, rank=16)
    rows = np.arange(n) % 3
    c.x = stored(c.x * np.where(rows == 0, 6e3, np.where(rows == 1, 1.0, 2e-4))[:, None], "f16")
    c.down, c.up = stored(c.down * 200.0, "f16"), stored(c.up * 2e-3, "f16")
    want = G.forward(c, "none", "f32", residual=False)
    assert np.abs(want["mid"][0]).max() > 1e6
    got = run_forward(c, "none", "f32", workspace, residual=False, pre=False)
    within(got["y"], *want["y"], "y")
    within(got["mid"], *want["mid"], "mid")
    c.delta = stored(c.delta * np.where(rows == 0, 3e4, 1e-2)[:, None], "f16")
    c.up, c.down = stored(c.up * 3e4, "f16"), stored(c.down * 1e-5, "f16")
    mid = G.forward(c, "none", "f32")["mid"][0].astype(np.float32).astype(np.float64)
    want, got = G.backward(c, "none", add=False, mid=mid), run_backward(c, "none", workspace, mid=mid, add=False)
    assert np.abs(want["dmid"][0]).max() > 1e5
    for k in got:
        within(got[k], *want[k], k)


def test_arrays_beyond_32_bit_offsets(workspace):
    """Rows that an index names at both ends of arrays of more than 2^32 bytes."""
    announce("arrays of more than 4 GiB by an index")
    n, i, o, stride, count = 300, 64, 72, 1 << 14, 140000
    c = G.Case(n, 3, i, o, "f16", seed=6, whole=True, gather=True, scatter=True)
    x, y, delta, dx = (DeviceArray((count, stride), np.uint16) for _ in range(4))
    assert x.nbytes > 1 << 32
    rng = np.random.default_rng(7)
    rows = np.concatenate([np.arange(100), count - 1 - np.arange(200)])
    x_rows, y_rows = rng.permutation(rows), rng.permutation(rows)
    for p in range(n):
        ext.write_device(x.ptr + 2 * stride * int(x_rows[p]), encode(c.x[c.x_rows[p]], "f16"))
        ext.write_device(delta.ptr + 2 * stride * int(y_rows[p]), encode(c.delta[c.y_rows[p]], "f16"))
    w, bias = DeviceArray.from_numpy(encode(c.w, "f16")), DeviceArray.from_numpy(c.bias.astype(np.float32))
    index = [DeviceArray.from_numpy(np.asarray(v, np.uint32)) for v in (c.offsets, x_rows, y_rows)]
    groups = L.NerfExtRowGroups(*[a.ptr for a in index], 3, count, count, 0)
    desc = L.NerfExtLinearDesc(n, i, o, L.NERF_EXT_F16, L.NERF_EXT_F16, L.NERF_EXT_ACT_NONE, stride, stride, 0, 0)
    dw = DeviceArray((3, o, i), np.float32)
    grouped_linear_forward(desc, groups, x.ptr, w.ptr, y.ptr, bias=bias.ptr)
    grouped_linear_backward(desc, groups, x.ptr, w.ptr, delta.ptr, dx=dx.ptr, dweight=dw.ptr, workspace=workspace)
    synchronize()
    want, ref = G.forward(c, "none", "f16", residual=False), G.backward(c, "none", add=False)
    for p in range(int(c.offsets[0]), int(c.offsets[-1])):
        equal(decode(ext.read_device(y.ptr + 2 * stride * int(y_rows[p]), (o,), np.uint16), "f16"), stored(want["y"][0][c.y_rows[p]], "f16"), f"y of position {p}")
        equal(decode(ext.read_device(dx.ptr + 2 * stride * int(x_rows[p]), (i,), np.uint16), "f16"), stored(ref["dx"][0][c.x_rows[p]], "f16"), f"dx of position {p}")
    equal(dw.numpy().astype(np.float64), ref["dw"][0], "dw")


@pytest.mark.parametrize("rank", [0, 16])
def test_same_bits_every_time(workspace, rank):
    announce(f"same bits, rank {rank}")
    for n, i, o in ((500, 200, 96), (66000, 128, 64)):
        c = G.Case(n, 20, i, o, "f16", seed=8, rank=rank, gather=True, scatter=True)
        first = run_forward(c, "gelu", "f32", workspace)
        mid = first.get("mid")
        back = run_backward(c, "gelu", workspace, mid=mid)
        for _ in range(3):
            again = run_forward(c, "gelu", "f32", workspace), run_backward(c, "gelu", workspace, mid=mid)
            for a, b in ((first, again[0]), (back, again[1])):
                for k in a:
                    assert np.array_equal(a[k], b[k], equal_nan=True), k


def test_rows_read_twice(workspace):
    """An index may name a row more than once where it is read: x in the forward pass
    and in the sums."""
    announce("rows read twice")
    c = G.Case(400, 5, 48, 40, "f16", seed=9, whole=True, gather=True)
    c.x_rows = np.random.default_rng(1).integers(0, 50, c.n)
    want, got = G.forward(c, "relu", "f16"), run_forward(c, "relu", "f16", workspace)
    equal(got["y"], stored(want["y"][0], "f16"), "y")
    want, got = G.backward(c, "relu"), run_backward(c, "relu", workspace, dx=False, dpre=False)
    for k in ("dw", "db"):
        equal(got[k], want[k][0], k)
