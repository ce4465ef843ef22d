"""The linear layer and its gradients (nerf_ext_linear_*) against their
definitions in 64 bits, at the sizes, strides, alignments, types and values
where a tiled product can go wrong."""
import ctypes as C

import numpy as np
import pytest

from conftest import announce
from linear_cases import ACTS, CODES, backward, decode, encode, forward, within
from nerf_amd import _lib as L, ext
from nerf_amd.device import DeviceArray, Stream, synchronize

pytestmark = pytest.mark.gpu


class Guarded:
    """A device array of rows with a stride, inside a larger allocation whose
    other bytes are checked to stay as they were; shift: elements by which its
    start misses a 256-byte boundary."""

    def __init__(self, rows, cols, kind, stride=0, shift=0, values=None):
        self.rows, self.cols, self.kind, self.stride = rows, cols, kind, stride or cols
        self.shift = shift
        dtype = np.float32 if kind == "f32" else np.uint16
        self.lead = 128 + shift
        self.host = np.full(self.lead + max(rows, 1) * self.stride + 128, 0x5A5A if dtype == np.uint16 else 1234.5, dtype)
        if values is not None:
            self.view(self.host)[:] = encode(values, kind)
        self.dev = DeviceArray.from_numpy(self.host)

    def view(self, flat):
        return np.lib.stride_tricks.as_strided(flat[self.lead :], (self.rows, self.cols), (self.stride * flat.itemsize, flat.itemsize))

    @property
    def ptr(self):
        return self.dev.ptr + self.lead * self.host.itemsize

    def read(self):
        now = self.dev.numpy()
        got = self.view(now).copy()
        rest = now.copy()
        self.view(rest)[:] = self.view(self.host)
        assert np.array_equal(rest.view(np.uint8), self.host.view(np.uint8)), "bytes outside the array changed"
        return got

    def values(self):
        return decode(self.read(), self.kind)


def _ptr(a):
    return None if a is None else a.ptr


def _inputs(n, i, o, kind, seed):
    rng = np.random.default_rng(seed)
    make = lambda shape, scale: decode(encode(rng.normal(0, scale, shape), kind), kind)  # noqa: E731
    return {"x": make((n, i), 1.0), "w": make((o, i), (2.0 / (i + o)) ** 0.5), "bias": rng.normal(0, 0.5, o).astype(np.float32).astype(np.float64), "residual": make((n, o), 1.0), "delta": make((n, o), 0.1),
            "pre": make((n, i), 1.5), "add": make((n, i), 0.1)}


def run_forward(v, kind, y_kind, act, *, bias=True, residual=True, pre=True, strides=(0, 0, 0), shift=0, workspace=L.NERF_EXT_LINEAR_WORKSPACE, stream=None):
    n, i = v["x"].shape
    o = v["w"].shape[0]
    d = L.NerfExtLinearDesc(n, i, o, CODES[kind], CODES[y_kind], ACTS[act], *strides, 0)
    x, w = Guarded(n, i, kind, strides[0], shift, v["x"]), Guarded(o, i, kind, 0, shift, v["w"])
    b = Guarded(1, o, "f32", 0, shift, v["bias"]) if bias else None
    r = Guarded(n, o, kind, strides[2], shift, v["residual"]) if residual else None
    y = Guarded(n, o, y_kind, strides[1], shift)
    z = Guarded(n, o, kind, 0, shift) if pre else None
    ws = DeviceArray((max(workspace, 1),), np.uint8)
    L.call("nerf_ext_linear_forward", C.byref(d), x.ptr, w.ptr, _ptr(b), _ptr(r), y.ptr, _ptr(z), ws.ptr if workspace else None, workspace, stream.handle if stream else None)
    synchronize()
    for a in (x, w, b, r):
        if a is not None:
            assert np.array_equal(a.read(), a.view(a.host)), "an input changed"
    return y.values(), z.values() if pre else None


def check_forward(n, i, o, kind, y_kind, act, seed=0, **kw):
    announce(f"forward n={n} in={i} out={o} {kind}->{y_kind} {act} {kw}")
    v = _inputs(n, i, o, kind, seed)
    y, z = run_forward(v, kind, y_kind, act, **kw)
    wy, wz, by, bz = forward(v["x"], v["w"], v["bias"] if kw.get("bias", True) else None, v["residual"] if kw.get("residual", True) else None, act, kind, y_kind)
    within(y, wy, by, "y")
    if z is not None:
        within(z, wz, bz, "pre")


def run_backward(v, kind, act, *, add=True, dx=True, dpre=True, dw=True, db=True, strides=(0, 0), shift=0, workspace=L.NERF_EXT_LINEAR_WORKSPACE):
    n, i = v["x"].shape
    o = v["w"].shape[0]
    d = L.NerfExtLinearDesc(n, i, o, CODES[kind], CODES[kind], ACTS[act], strides[0], strides[1], 0, 0)
    x, w = Guarded(n, i, kind, strides[0], shift, v["x"]), Guarded(o, i, kind, 0, shift, v["w"])
    g, z = Guarded(n, o, kind, strides[1], shift, v["delta"]), Guarded(n, i, kind, 0, shift, v["pre"])
    a = Guarded(n, i, kind, strides[0], shift, v["add"]) if add else None
    out = {"dx": Guarded(n, i, kind, strides[0], shift) if dx else None, "dpre": Guarded(n, i, kind, 0, shift) if dpre else None, "dw": Guarded(o, i, "f32", 0, shift) if dw else None,
           "db": Guarded(1, o, "f32", 0, shift) if db else None}
    ws = DeviceArray((max(workspace, 1),), np.uint8)
    L.call("nerf_ext_linear_backward", C.byref(d), x.ptr if dw else None, w.ptr if dx or dpre else None, g.ptr, z.ptr if dpre else None, _ptr(a), _ptr(out["dx"]), _ptr(out["dpre"]), _ptr(out["dw"]), _ptr(out["db"]),
           ws.ptr if workspace else None, workspace, None)
    synchronize()
    for b in (x, w, g, z, a):
        if b is not None:
            assert np.array_equal(b.read(), b.view(b.host)), "an input changed"
    return {k: b.values() for k, b in out.items() if b is not None}


def check_backward(n, i, o, kind, act, seed=0, **kw):
    announce(f"backward n={n} in={i} out={o} {kind} {act} {kw}")
    v = _inputs(n, i, o, kind, seed)
    got = run_backward(v, kind, act, **kw)
    want = backward(v["x"], v["w"], v["delta"], v["pre"], v["add"] if kw.get("add", True) else None, act, kind)
    for k, value in got.items():
        ref, bound = want[k]
        within(value.reshape(ref.shape), ref, bound, k)


# Lengths of one, odd ones, ones around the tiles' edges, wide and narrow.
SHAPES = [(1, 1, 1), (1, 256, 256), (1, 63, 5), (2, 7, 3), (3, 8, 1000), (4, 1000, 8), (5, 640, 520), (15, 64, 64), (16, 65, 63), (17, 33, 31), (31, 1, 129), (33, 129, 1), (63, 64, 128), (64, 128, 64), (65, 127, 130), (128, 128, 128),
          (129, 136, 264), (200, 256, 256), (255, 257, 259), (257, 512, 72), (300, 72, 512), (1000, 63, 256), (1025, 320, 96)]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_shapes(shape, kind):
    check_forward(*shape, kind, kind, "relu")


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_backward_shapes(shape, kind):
    check_backward(*shape, kind, "relu")


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("y_kind", ["f16", "f32"])
def test_forward_activations(act, y_kind):
    check_forward(70, 48, 96, "f16", y_kind, act)


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_backward_activations(act, kind):
    check_backward(70, 96, 48, kind, act)


@pytest.mark.parametrize("bias,residual,pre", [(False, False, False), (True, False, False), (False, True, False), (False, False, True)])
def test_forward_optional_arrays(bias, residual, pre):
    check_forward(77, 72, 88, "bf16", "f32", "silu", bias=bias, residual=residual, pre=pre)


@pytest.mark.parametrize("which", ["dx", "dpre", "dw"])
@pytest.mark.parametrize("add", [False, True])
def test_backward_single_outputs(which, add):
    check_backward(130, 72, 88, "f16", "gelu", add=add, db=which == "dw", **{k: k == which for k in ("dx", "dpre", "dw")})


def test_backward_weight_gradient_without_bias():
    check_backward(130, 72, 88, "f16", "none", dx=False, dpre=False, db=False)


# Strides and starts: multiples of 8, of 4 only, odd; columns of a wider array.
@pytest.mark.parametrize("strides,shift", [((80, 96, 104), 0), ((76, 92, 100), 4), ((75, 91, 99), 0), ((72, 88, 88), 1), ((73, 88, 89), 3), ((200, 88, 88), 8)])
@pytest.mark.parametrize("n", [5, 150])
def test_strides_and_alignment(n, strides, shift):
    check_forward(n, 72, 88, "f16", "f16", "relu", strides=strides, shift=shift)
    check_forward(n, 72, 88, "bf16", "f32", "none", strides=strides, shift=shift)
    check_backward(n, 72, 88, "f16", "relu", strides=strides[:2], shift=shift)


# Sums split over workgroups: few outputs, many terms; none, too little and
# enough workspace for the parts.
@pytest.mark.parametrize("workspace", [0, 4096, 100000, L.NERF_EXT_LINEAR_WORKSPACE])
def test_split_sums(workspace):
    check_forward(3, 4096, 24, "f16", "f16", "sigmoid", workspace=workspace)
    check_forward(70, 2501, 24, "bf16", "f32", "none", workspace=workspace)
    check_backward(20011, 40, 24, "f16", "relu", workspace=workspace)
    check_backward(40, 31, 3001, "bf16", "silu", workspace=workspace)


def test_rows_over_many_tiles():
    check_forward(40003, 24, 40, "f16", "f16", "relu")
    check_forward(40003, 64, 256, "f16", "f16", "relu")
    check_backward(40003, 64, 32, "f16", "relu")
    check_backward(33001, 256, 256, "f16", "relu")


# Many rows and few k: every step of 32 k, whole and cut rows, narrow and wide
# outputs, a last tile of rows that is not whole.
@pytest.mark.parametrize("n,k,p", [(16384, 1, 3), (16385, 7, 40), (16400, 8, 33), (20011, 31, 64), (20011, 33, 200), (16397, 63, 256), (17001, 96, 129), (16999, 130, 70), (16384, 255, 300), (20000, 256, 16), (16401, 250, 257), (16411, 200, 96)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_many_rows(n, k, p, kind):
    check_forward(n, k, p, kind, kind if p % 2 else "f32", "relu")
    check_backward(n, p, k, kind, "relu", dw=False, db=False)


def test_many_rows_with_strides():
    for strides, shift in (((272, 136, 144), 0), ((257, 131, 133), 1)):
        check_forward(17003, 256, 130, "f16", "f16", "silu", strides=strides, shift=shift)
        check_backward(17003, 256, 130, "f16", "silu", strides=strides[:2], shift=shift, dw=False, db=False)


# So many rows that a CU keeps its weights for all 64, 128 and 256 k, and sums in
# whole tiles beside them.
@pytest.mark.parametrize("n,k,p", [(32800, 64, 40), (32771, 57, 24), (65541, 128, 72), (65536, 96, 32), (131077, 256, 136), (131072, 224, 24), (131073, 160, 300), (131075, 250, 24)])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_very_many_rows(n, k, p, kind):
    check_forward(n, k, p, kind, kind, "relu")
    check_backward(n, p, k, kind, "relu", dw=False, db=False)


# Around the sizes at which sums are split and tiles change.
@pytest.mark.parametrize("n,i,o", [(16, 8192, 96), (70, 1088, 520), (500, 1100, 1032), (1500, 1048, 1160), (2050, 264, 256), (4096, 64, 1040), (4100, 1024, 1032)])
def test_split_and_tile_choices(n, i, o):
    check_forward(n, i, o, "f16", "f16", "silu")
    check_backward(n, i, o, "f16", "silu")


def test_more_rows_than_one_launch():
    check_forward(65535 * 64 + 100, 9, 2, "f16", "f16", "relu")
    check_backward(65535 * 64 + 100, 2, 9, "bf16", "relu")


def test_offsets_beyond_32_bits():
    """Rows 2^20 elements apart: offsets up to 2^36 bytes."""
    n, i, o, stride = 16400, 64, 40, 1 << 20
    v = _inputs(n, i, o, "f16", 9)
    x, y = DeviceArray((n, stride), np.uint16), DeviceArray((n, stride // 4), np.float32)
    bits = encode(v["x"], "f16")
    for r in range(n):
        ext.write_device(x.ptr + 2 * stride * r, bits[r])
    w, b, d = Guarded(o, i, "f16", values=v["w"]), Guarded(1, o, "f32", values=v["bias"]), Guarded(n, o, "f16", values=v["delta"])
    desc = L.NerfExtLinearDesc(n, i, o, CODES["f16"], CODES["f32"], ACTS["relu"], stride, stride // 4, 0, 0)
    L.call("nerf_ext_linear_forward", C.byref(desc), x.ptr, w.ptr, b.ptr, None, y.ptr, None, None, 0, None)
    synchronize()
    got = np.stack([ext.read_device(y.ptr + stride * r, (o,), np.float32) for r in range(n)]).astype(np.float64)
    want, _, bound, _ = forward(v["x"], v["w"], v["bias"], None, "relu", "f16", "f32")
    within(got, want, bound, "y")
    desc.y_stride = 0
    dw, db = Guarded(o, i, "f32"), Guarded(1, o, "f32")
    ws = DeviceArray((L.NERF_EXT_LINEAR_WORKSPACE,), np.uint8)
    L.call("nerf_ext_linear_backward", C.byref(desc), x.ptr, None, d.ptr, None, None, None, None, dw.ptr, db.ptr, ws.ptr, ws.nbytes, None)
    synchronize()
    ref = backward(v["x"], v["w"], v["delta"], v["pre"], None, "relu", "f16")
    within(dw.values(), *ref["dw"], "dw")
    within(db.values()[0], *ref["db"], "db")


def test_wide_layers():
    check_forward(700, 1024, 2056, "bf16", "bf16", "gelu")
    check_backward(700, 1032, 1024, "bf16", "gelu")


def test_no_rows():
    v = _inputs(0, 24, 40, "f16", 0)
    y, z = run_forward(v, "f16", "f16", "relu")
    assert y.shape == (0, 40) and z.shape == (0, 40)
    got = run_backward(v, "f16", "relu")
    assert not got["dw"].any() and not got["db"].any() and got["dx"].shape == (0, 24)


@pytest.mark.parametrize("act", list(ACTS))
def test_activation_ends(act):
    """Large arguments of both signs reach the activations' and derivatives'
    limits without a NaN."""
    z = np.array([[0.0, -0.0, 1e-4, -1e-4, 5.0, -5.0, 9.0, -9.0, 15.0, -15.0, 30.0, -30.0, 200.0, -200.0, 6e4, -6e4]])
    n = z.shape[1]
    eye = np.eye(n)
    z = decode(encode(z, "f16"), "f16")
    v = {"x": z, "w": eye, "bias": np.zeros(n), "residual": z * 0, "delta": np.full((1, n), 0.5), "pre": z, "add": z * 0}
    y, _ = run_forward(v, "f16", "f32", act)
    wy, _, by, _ = forward(z, eye, None, None, act, "f16", "f32")
    within(y, wy, by, act)
    got = run_backward(v, "f16", act)
    ref, bound = backward(z, eye, v["delta"], z, None, act, "f16")["dpre"]
    within(got["dpre"], ref, bound, act + " derivative")


def test_infinities_and_nan_stay_in_their_rows():
    """A row that holds an infinity or a NaN spoils its own outputs only: the
    tiles' padding never meets it."""
    v = _inputs(37, 45, 51, "f16", 3)
    for row, value in ((0, np.inf), (17, -np.inf), (36, np.nan)):
        v["x"][row, 44] = value
        v["delta"][row, 50] = value
    y, _ = run_forward(v, "f16", "f16", "relu")
    good = [r for r in range(37) if r not in (0, 17, 36)]
    clean = {k: a.copy() for k, a in v.items()}
    for row in (0, 17, 36):
        clean["x"][row] = clean["delta"][row] = 0.0
    wy, _, by, _ = forward(clean["x"], v["w"], v["bias"], v["residual"], "relu", "f16", "f16")
    within(y[good], wy[good], by[good], "y")
    assert np.isnan(y[36]).all() and not np.isfinite(y[0]).all()
    got = run_backward(v, "f16", "relu")
    ref, bound = backward(clean["x"], v["w"], clean["delta"], v["pre"], v["add"], "relu", "f16")["dx"]
    within(got["dx"][good], ref[good], bound[good], "dx")
    assert np.isnan(got["dx"][36]).all()
    assert np.isnan(got["db"].ravel()[50]) and np.isfinite(got["db"].ravel()[:50]).all()
    assert np.isfinite(got["dw"][:50, :44]).all()


def test_outputs_over_their_inputs():
    """y over residual, dx over add, dpre over pre."""
    v = _inputs(133, 72, 88, "f16", 5)
    want = forward(v["x"], v["w"], v["bias"], v["residual"], "relu", "f16", "f16")
    d = L.NerfExtLinearDesc(133, 72, 88, CODES["f16"], CODES["f16"], ACTS["relu"], 0, 0, 0, 0)
    x, w, b, r = Guarded(133, 72, "f16", values=v["x"]), Guarded(88, 72, "f16", values=v["w"]), Guarded(1, 88, "f32", values=v["bias"]), Guarded(133, 88, "f16", values=v["residual"])
    L.call("nerf_ext_linear_forward", C.byref(d), x.ptr, w.ptr, b.ptr, r.ptr, r.ptr, None, None, 0, None)
    synchronize()
    within(r.values(), want[0], want[2], "y")
    g, a, p = Guarded(133, 88, "f16", values=v["delta"]), Guarded(133, 72, "f16", values=v["add"]), Guarded(133, 72, "f16", values=v["pre"])
    L.call("nerf_ext_linear_backward", C.byref(d), None, w.ptr, g.ptr, p.ptr, a.ptr, a.ptr, p.ptr, None, None, None, 0, None)
    synchronize()
    ref = backward(v["x"], v["w"], v["delta"], v["pre"], v["add"], "relu", "f16")
    within(a.values(), *ref["dx"], "dx")
    within(p.values(), *ref["dpre"], "dpre")


def test_same_bits_every_time():
    v = _inputs(5000, 96, 72, "f16", 6)
    first = run_backward(v, "f16", "relu")
    second = run_backward(v, "f16", "relu")
    assert all(np.array_equal(first[k], second[k]) for k in first)


def test_other_stream():
    v = _inputs(300, 96, 72, "bf16", 7)
    y, _ = run_forward(v, "bf16", "bf16", "relu", stream=Stream())
    here, _ = run_forward(v, "bf16", "bf16", "relu")
    assert np.array_equal(y, here)


def test_gradients_against_differences():
    """loss = sum c y, y = sigmoid(x W^T + b) from the forward pass itself in 32
    bits: its change along a direction of W and of b is the backward's gradient."""
    n, i, o = 96, 40, 24
    rng = np.random.default_rng(8)
    v = _inputs(n, i, o, "f16", 8)
    c = rng.normal(0, 1, (n, o))
    h = 2.0**-5
    dw, db = rng.integers(-2, 3, (o, i)) * 2.0**-3, rng.integers(-2, 3, o) * 2.0**-3
    v["w"] = np.round(v["w"] * 2.0**9) / 2.0**9  # w +- h dw are fp16 numbers

    def loss(t):
        u = dict(v, w=v["w"] + t * dw, bias=v["bias"] + t * db)
        return float((c * run_forward(u, "f16", "f32", "sigmoid", residual=False, pre=False)[0]).sum())

    # Central differences of steps h and h / 2, extrapolated: error O(h^4).
    numeric = (4.0 * (loss(h / 2) - loss(-h / 2)) / h - (loss(h) - loss(-h)) / (2.0 * h)) / 3.0
    z = v["x"] @ v["w"].T + v["bias"]
    exact_delta = c * 0.25 / np.cosh(z / 2.0) ** 2
    v["delta"] = decode(encode(exact_delta, "f16"), "f16")
    got = run_backward(v, "f16", "none", dx=False, dpre=False)
    analytic = float((got["dw"] * dw).sum() + (got["db"] * db).sum())
    # |analytic - numeric|: the fp16 deltas (2^-11 of each, through the direction's
    # move of z), 32-bit losses (2^-21 of their size over the step), and the h^4
    # term with the fifth derivative of sigmoid (at most 1/4 here) along t.
    move = np.abs(v["x"] @ dw.T + db)
    bound = (2.0**-11 * np.abs(exact_delta) * move).sum() + 2.0**-21 * np.abs(c).sum() * 4.0 / h + (np.abs(c) * move**5).sum() * h**4 / 4.0
    print(f"analytic {analytic} numeric {numeric} bound {bound}")
    assert abs(analytic - numeric) <= bound
