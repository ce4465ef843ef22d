"""What nerf_ext_group_rows, nerf_ext_grouped_linear_* and
nerf_ext_adapter_linear_* refuse, decided on the host before any GPU work; and
the 64-bit definitions that the GPU tests compare with, checked against each
other and against finite differences."""
import ctypes as C

import numpy as np
import pytest

import grouped_cases as G
from nerf_amd import _lib as L

BAD = L.NERF_STATUS_INVALID_USAGE
A = 1 << 20  # an address that is never followed


def desc(**kw):
    d = L.NerfExtLinearDesc(4, 8, 16, L.NERF_EXT_F16, L.NERF_EXT_F16, L.NERF_EXT_ACT_RELU, 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def groups(**kw):
    g = L.NerfExtRowGroups(A, None, None, 3, 0, 0, 0)
    for k, v in kw.items():
        setattr(g, k, v)
    return g


def adapters(**kw):
    a = L.NerfExtAdapters(A, A, A, 4, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def ref(s):
    return C.byref(s) if s is not None else None


GFWD = dict(x=A, w=A, b=A, r=A, y=A, z=A, ws=A, nb=1 << 20)
GBWD = dict(x=A, w=A, delta=A, z=A, a=A, dx=A, dz=A, dw=A, db=A, ws=A, nb=1 << 20)
AFWD = dict(x=A, w=A, b=A, r=A, y=A, z=A, mid=A, ws=A, nb=1 << 20)
ABWD = dict(x=A, w=A, delta=A, mid=A, z=A, a=A, dx=A, dz=A, dmid=A, ddown=A, dup=A, ws=A, nb=1 << 20)


def gfwd(d=desc(), g=groups(), **kw):
    return L.status_of("nerf_ext_grouped_linear_forward", ref(d), ref(g), *(GFWD | kw).values(), None)


def gbwd(d=desc(), g=groups(), **kw):
    return L.status_of("nerf_ext_grouped_linear_backward", ref(d), ref(g), *(GBWD | kw).values(), None)


def afwd(d=desc(), g=groups(), ad=adapters(), **kw):
    return L.status_of("nerf_ext_adapter_linear_forward", ref(d), ref(g), ref(ad), *(AFWD | kw).values(), None)


def abwd(d=desc(), g=groups(), ad=adapters(), **kw):
    return L.status_of("nerf_ext_adapter_linear_backward", ref(d), ref(g), ref(ad), *(ABWD | kw).values(), None)


CALLS = {"nerf_ext_grouped_linear_forward": gfwd, "nerf_ext_grouped_linear_backward": gbwd, "nerf_ext_adapter_linear_forward": afwd, "nerf_ext_adapter_linear_backward": abwd}


@pytest.mark.parametrize("name", CALLS)
def test_descriptors(lib, name):
    call = CALLS[name]
    for d, word in ((None, "null"), (desc(in_features=0), "features"), (desc(rows=(1 << 30) + 1), "rows"), (desc(dtype=L.NERF_EXT_F32), "dtype"), (desc(out_dtype=L.NERF_EXT_BF16), "out_dtype"), (desc(activation=6), "activation"),
                    (desc(x_stride=7), "stride"), (desc(reserved=1), "reserved"), (desc(rows=1 << 30, in_features=65536), "tiles")):
        assert call(d) == BAD and word in L.last_error() and name in L.last_error(), (word, L.last_error())
    for g, word in ((None, "null"), (groups(groups=0), "groups"), (groups(groups=4097), "groups"), (groups(offsets=None), "offsets"), (groups(offsets=A + 2), "aligned"), (groups(x_rows=A + 1), "aligned"), (groups(y_rows=A + 2), "aligned"),
                    (groups(reserved=1), "reserved"), (groups(x_count=5), "x_count"), (groups(y_count=3), "y_count"), (groups(x_rows=A, x_count=(1 << 30) + 1), "2^30")):
        assert call(g=g) == BAD and word in L.last_error() and name in L.last_error(), (word, L.last_error())


@pytest.mark.parametrize("name", ["nerf_ext_adapter_linear_forward", "nerf_ext_adapter_linear_backward"])
def test_adapters(lib, name):
    for a, word in ((None, "null"), (adapters(rank=0), "rank"), (adapters(rank=257), "rank"), (adapters(reserved=1), "reserved"), (adapters(down=A + 1), "aligned"), (adapters(up=A + 1), "aligned"), (adapters(scales=A + 2), "aligned")):
        assert CALLS[name](ad=a) == BAD and word in L.last_error() and name in L.last_error(), word


def test_arrays(lib):
    odd = [dict(x=A + 1), dict(w=A + 1), dict(z=A + 1), dict(ws=A + 8)]
    for kw in odd + [dict(x=None), dict(w=None), dict(y=None), dict(b=A + 2), dict(r=A + 1), dict(y=A + 1)]:
        assert gfwd(**kw) == BAD and afwd(**kw) == BAD, kw
    for kw in (dict(mid=None), dict(mid=A + 2)):
        assert afwd(**kw) == BAD, kw
    assert afwd(ad=adapters(down=None)) == BAD and afwd(ad=adapters(up=None)) == BAD
    # y over residual of another type or row stride.
    assert gfwd(desc(out_dtype=L.NERF_EXT_F32)) == BAD and afwd(desc(y_stride=24)) == BAD
    for kw in odd + [dict(x=None), dict(w=None), dict(delta=None), dict(z=None), dict(dx=None, dz=None, dw=None, db=None), dict(dw=None), dict(delta=A + 1), dict(dw=A + 2), dict(db=A + 2), dict(dx=A + 1), dict(a=A + 1), dict(dz=A + 1)]:
        assert gbwd(**kw) == BAD, kw
    for kw in odd + [dict(x=None), dict(w=None), dict(delta=None), dict(z=None), dict(mid=None), dict(dmid=None), dict(dx=None, dz=None, dmid=None, ddown=None, dup=None), dict(mid=A + 2), dict(dmid=A + 2), dict(ddown=A + 2), dict(dup=A + 2), dict(dx=A + 1)]:
        assert abwd(**kw) == BAD, kw
    assert abwd(ad=adapters(down=None)) == BAD and abwd(ad=adapters(up=None)) == BAD


def test_no_rows_need_no_arrays(lib):
    none = {k: None for k in ("x", "w", "b", "r", "y", "z", "ws")} | {"nb": 0}
    assert gfwd(desc(rows=0), **none) == L.NERF_STATUS_OK
    assert afwd(desc(rows=0), ad=adapters(down=None, up=None, scales=None), mid=None, **none) == L.NERF_STATUS_OK
    assert gbwd(desc(rows=0), x=None, w=None, delta=None, z=None, a=None, dw=None, db=None) == L.NERF_STATUS_OK
    assert abwd(desc(rows=0), x=None, w=None, delta=None, z=None, a=None, mid=None, ddown=None, dup=None) == L.NERF_STATUS_OK


def test_group_rows(lib):
    def call(ids=A, rows=10, n=3, offsets=A, order=A, place=A, ws=A, nb=1 << 20):
        return L.status_of("nerf_ext_group_rows", ids, rows, n, offsets, order, place, ws, nb, None)

    for kw in (dict(n=0), dict(n=4097), dict(rows=(1 << 30) + 1), dict(ids=None), dict(offsets=None), dict(order=None), dict(ids=A + 1), dict(offsets=A + 2), dict(order=A + 2), dict(place=A + 1), dict(ws=A + 8), dict(rows=0, offsets=None)):
        assert call(**kw) == BAD and "nerf_ext_group_rows" in L.last_error(), kw


def test_structures():
    assert C.sizeof(L.NerfExtRowGroups) == 40 and L.NerfExtRowGroups.groups.offset == 24
    assert C.sizeof(L.NerfExtAdapters) == 32 and L.NerfExtAdapters.rank.offset == 24


@pytest.mark.parametrize("rank", [0, 3])
def test_definitions_against_differences(rank):
    """The definitions' gradients of sum(y * delta) for a smooth activation, against
    central differences in every operand."""
    c = G.Case(12, 3, 5, 4, "f16", seed=1, rank=rank, gather=True, scatter=True, extra=3)
    c.residual = np.zeros_like(c.residual)

    def loss():
        out = G.forward(c, "none", "f32")
        return (out["y"][0] * c.delta).sum()  # rows outside keep a constant

    mid = G.forward(c, "none", "f32")["mid"][0] if rank else None
    c.pre[:] = 1.0
    got = G.backward(c, "none", add=False, mid=mid)
    rows = c.xr() if rank else c.xr()[c.offsets[0] : c.offsets[-1]]
    checks = [("dx", c.x, rows)] + ([("ddown", c.down, None), ("dup", c.up, None)] if rank else [("dw", c.w, None), ("db", c.bias, None)])
    rng, h = np.random.default_rng(2), 2.0**-6
    for name, array, only in checks:
        flat, want = array.reshape(-1), got[name][0].reshape(-1)
        places = np.arange(array.size) if only is None else (only[:, None] * array.shape[1] + np.arange(array.shape[1])).reshape(-1)
        for at in rng.choice(places, min(20, len(places)), replace=False):
            old = flat[at]
            flat[at] = old + h
            up = loss()
            flat[at] = old - h
            down = loss()
            flat[at] = old
            assert abs((up - down) / (2 * h) - want[at]) <= 1e-8 * (1 + abs(want[at])), (name, at)


def test_group_definition():
    offsets, order, place = G.group_rows([2, 0, 7, 2, 1, 0], 3)
    assert offsets.tolist() == [0, 2, 3, 5] and order.tolist() == [1, 5, 4, 0, 3, 2] and place.tolist() == [3, 0, 5, 4, 2, 1]
