"""Adapters where an operand is infinite, or 32-bit values lie at the ends of what
their pieces in 16 bits can hold: the definition's infinity, NaN or number in
every output, whichever kernel a call takes."""
import numpy as np
import pytest

import grouped_cases as G
from conftest import announce
from linear_cases import EPS, encode, decode, rounding
from nerf_amd import _lib as L
from nerf_amd.device import DeviceArray
from test_gpu_grouped import run_backward, run_forward

pytestmark = pytest.mark.gpu

# rows, in, out, rank: few outputs, tiles of 64, 128 and 256, rows streamed past the
# weights, with ranks that are whole multiples of 16 and others.
SHAPES = [(60, 40, 24, 7), (900, 72, 136, 16), (3000, 33, 65, 5), (9000, 264, 520, 20), (16500, 1024, 1024, 8), (66000, 64, 64, 9), (66000, 96, 72, 16), (65700, 64, 128, 40)]
TYPES = [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")]


@pytest.fixture(scope="module")
def workspace():
    return DeviceArray((L.NERF_EXT_LINEAR_WORKSPACE,), np.uint8)


def case(n, i, o, r, kind):
    c = G.Case(n, 3, i, o, kind, seed=n + i, rank=r, gather=True, scatter=True)
    g = int(np.argmax(np.diff(c.offsets)))
    c.scales = np.abs(c.scales) + 0.5
    some = 12 if i * o > 1 << 18 else 40
    at = np.unique(np.linspace(c.offsets[g], c.offsets[g + 1] - 1, some).astype(int))
    return c, g, at


def settle(c):
    """Inputs as the device has them."""
    for name in ("x", "w", "down", "up", "delta"):
        setattr(c, name, decode(encode(getattr(c, name), c.kind), c.kind))
    c.scales = c.scales.astype(np.float32).astype(np.float64)


def products(a, b):
    """sum_k a[n][k] b[m][k], term by term (a library's product may pad its sums), and the
    sums of the finite terms' magnitudes."""
    with np.errstate(invalid="ignore"):
        t = a[:, None, :] * b[None]
        return t.sum(-1), np.where(np.isfinite(t), np.abs(t), 0.0).sum(-1)


def same(got, want, bound, what):
    """NaN where the definition has one, its infinities, its numbers within the bound."""
    nan, inf = np.isnan(want), np.isinf(want)
    assert (np.isnan(got) == nan).all(), f"{what}: {np.isnan(got).sum()} NaN, {nan.sum()} expected"
    assert (got[inf] == want[inf]).all(), what
    rest = ~(nan | inf)
    assert (np.abs(got - want)[rest] <= bound[rest]).all(), what


def forward_is(c, g, at, y_kind, ws):
    settle(c)
    got = run_forward(c, "none", y_kind, ws, residual=False)
    x, s = c.x[c.xr()[at]], c.scales[g]
    mid, size = products(x, c.down[g])
    same(got["mid"][at], mid, (c.i + 2) * EPS * size, "mid")
    z, terms = products(x, c.w)
    # m is off by its own sum's error, which is relative to size, and by its pieces',
    # 2^-16 of it (bf16, two pieces; three for fp32 outputs: 2^-24) or 2^-22 of the row's
    # largest (fp16).
    finite = np.where(np.isfinite(mid), np.abs(mid), 0.0)
    off = (c.i + 2) * EPS * size + ((2.0**-24 if y_kind == "f32" else 2.0**-16) * finite if c.kind == "bf16" else 2.0**-22 * finite.max(1, keepdims=True))
    up = np.where(np.isfinite(c.up[g]), np.abs(c.up[g]), 0.0)
    low, low_terms = products(mid, c.up[g])
    bound = (c.i + 4) * EPS * terms + s * (off @ up.T) + (3 * c.rank + 8) * EPS * (s * low_terms + np.abs(c.bias))
    with np.errstate(invalid="ignore"):
        z = z + s * low + c.bias
    same(got["y"][c.yr()[at]], z, bound + rounding(np.where(np.isfinite(z), np.abs(z) + bound, 0.0), y_kind), "y")
    return z


def backward_is(c, g, at, mid, ws, x_columns=(), d_columns=()):
    settle(c)
    got = run_backward(c, "none", ws, mid=mid, add=False, dpre=False)
    d, s, rows = c.delta[c.yr()], c.scales[g], slice(int(c.offsets[g]), int(c.offsets[g + 1]))
    low, size = products(d[at], c.up[g].T)
    low, size = s * low, s * size
    same(got["dmid"][at], low, (c.o + 4) * EPS * size, "dmid")
    z, terms = products(d[at], c.w.T)
    finite = np.where(np.isfinite(low), np.abs(low), 0.0)
    off = (c.o + 4) * EPS * size + (2.0**-16 * finite if c.kind == "bf16" else 2.0**-22 * finite.max(1, keepdims=True))
    down = np.where(np.isfinite(c.down[g]), np.abs(c.down[g]), 0.0)
    part, part_terms = products(low, c.down[g].T)
    bound = (c.o + 4) * EPS * terms + off @ down + (3 * c.rank + 8) * EPS * part_terms
    with np.errstate(invalid="ignore"):
        z = z + part
    same(got["dx"][c.xr()[at]], z, bound + rounding(np.where(np.isfinite(z), np.abs(z) + bound, 0.0), c.kind), "dx")
    # Sums over the group's rows, of the columns asked for: dmid as the kernel has it.
    n, x, k = rows.stop - rows.start, c.x[c.xr()], (rows.stop - rows.start + 8) * EPS
    for col in x_columns:
        want, terms = products(got["dmid"][rows].T, x[rows, col][None])
        same(got["ddown"][g][:, col], want[:, 0], k * terms[:, 0] + 2.0**-140, f"ddown of column {col}")
    for col in d_columns:
        want, terms = products(mid[rows].T, d[rows, col][None])
        same(got["dup"][g][col], s * want[:, 0], s * k * terms[:, 0] + 2.0**-140, f"dup of column {col}")
    return got


@pytest.mark.parametrize("kind,y_kind", TYPES)
@pytest.mark.parametrize("n,i,o,r", SHAPES)
def test_infinite_up(workspace, n, i, o, r, kind, y_kind):
    announce(f"infinite up, {n} x {i} -> {o}, rank {r}, {kind} -> {y_kind}")
    c, g, at = case(n, i, o, r, kind)
    c.up[g][3, 0], c.up[g][5, r - 1], c.up[g][o - 1, r // 2] = np.inf, -np.inf, np.inf
    c.x[c.xr()[at[1]]] = 0.0  # m of zeros, whose products with infinities are NaN
    z = forward_is(c, g, at, y_kind, workspace)
    assert np.isposinf(z).any() and np.isneginf(z).any() and np.isnan(z[1, 3])


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n,i,o,r", SHAPES)
def test_infinite_down(workspace, n, i, o, r, kind):
    """In the forward pass m of that rank is infinite, in the backward pass an input's
    gradient."""
    announce(f"infinite down, {n} x {i} -> {o}, rank {r}, {kind}")
    c, g, at = case(n, i, o, r, kind)
    c.down[g][0, 3], c.down[g][r - 1, 5] = np.inf, -np.inf
    forward_is(c, g, at, "f32", workspace)
    mid = np.random.default_rng(1).normal(0, 1, (n, r)).astype(np.float32).astype(np.float64)
    backward_is(c, g, at, mid, workspace)


@pytest.mark.parametrize("kind,y_kind", TYPES)
@pytest.mark.parametrize("n,i,o,r", SHAPES)
def test_infinite_inputs(workspace, n, i, o, r, kind, y_kind):
    """An infinite input whose products all have the same sign: outputs of that row are
    infinite, at ranks that are no whole multiples of a tile's too."""
    announce(f"infinite inputs, {n} x {i} -> {o}, rank {r}, {kind} -> {y_kind}")
    c, g, at = case(n, i, o, r, kind)
    for a in (c.w[:, 7], c.down[g][:, 7]):
        a[:] = np.abs(a) + 0.125
    c.up[g] = np.abs(c.up[g]) + 0.125
    row = c.xr()[at[2]]
    c.x[row, 7] = np.inf
    z = forward_is(c, g, at, y_kind, workspace)
    assert np.isposinf(z[2]).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n,i,o,r", SHAPES)
def test_infinite_deltas(workspace, n, i, o, r, kind):
    """The same of a row's gradient."""
    announce(f"infinite deltas, {n} x {i} -> {o}, rank {r}, {kind}")
    c, g, at = case(n, i, o, r, kind)
    for a in (c.w[7], c.up[g][7]):
        a[:] = np.abs(a) + 0.125
    c.down[g] = np.abs(c.down[g]) + 0.125
    c.delta[c.yr()[at[2]], 7] = -np.inf
    mid = np.random.default_rng(1).normal(0, 1, (n, r)).astype(np.float32).astype(np.float64)
    got = backward_is(c, g, at, mid, workspace)
    assert np.isneginf(got["dx"][c.xr()[at[2]]]).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("n,i,o,r", SHAPES)
def test_infinite_rows_of_sums(workspace, n, i, o, r, kind):
    """An infinite input and an infinite delta in the sums over a group's rows: an
    infinity of the other factor's sign."""
    announce(f"infinite rows of sums, {n} x {i} -> {o}, rank {r}, {kind}")
    c, g, at = case(n, i, o, r, kind)
    mid = np.random.default_rng(1).normal(0, 1, (n, r)).astype(np.float32).astype(np.float64)
    c.x[c.xr()[at[2]], 7] = np.inf
    got = backward_is(c, g, at, mid, workspace, x_columns=(6, 7))
    assert np.isposinf(got["ddown"][g][:, 7]).any() and np.isinf(got["ddown"][g][:, 7]).all()
    c.delta[c.yr()[at[3]], 7] = -np.inf
    got = backward_is(c, g, at, mid, workspace, d_columns=(6, 7))
    assert np.isposinf(got["dup"][g][7]).any() and np.isinf(got["dup"][g][7]).all()


@pytest.mark.parametrize("n,i,o,r", SHAPES)
def test_large_values_beside_an_infinity(workspace, n, i, o, r):
    """fp16: an infinite m, and others of the row beyond 65504 with factors of the other
    sign, do not cancel."""
    announce(f"large m beside an infinite one, {n} x {i} -> {o}, rank {r}")
    c, g, at = case(n, i, o, r, "f16")
    c.x = decode(encode(np.abs(c.x) * 3e3 + 1e3, "f16"), "f16")
    c.down[g] = decode(encode(np.abs(c.down[g]) * 200.0 + 1.0, "f16"), "f16")
    c.down[g][1, 3] = np.inf
    c.up[g] = -np.abs(c.up[g]) - 0.125
    c.up[g][:, 1] = 1.0
    z = forward_is(c, g, at, "f32", workspace)
    assert np.isposinf(z).all()


@pytest.mark.parametrize("n,i,o,r", SHAPES)
def test_small_values_beside_large_ones(workspace, n, i, o, r):
    """fp16: an m far below the row's largest is still not zero where up is infinite."""
    announce(f"small m beside large ones, {n} x {i} -> {o}, rank {r}")
    c, g, at = case(n, i, o, r, "f16")
    c.x = decode(encode(np.abs(c.x) * 3e3 + 1e3, "f16"), "f16")
    c.down[g] = decode(encode(np.abs(c.down[g]) * 200.0 + 1.0, "f16"), "f16")
    c.down[g][1], c.down[g][1, 3] = 0.0, 2.0**-24
    c.up[g][4, 1], c.up[g][6, 1] = np.inf, -np.inf
    z = forward_is(c, g, at, "f32", workspace)
    assert np.isposinf(z[:, 4]).all() and np.isneginf(z[:, 6]).all()


@pytest.mark.parametrize("y_kind", ["bf16", "f32"])
@pytest.mark.parametrize("n,i,o,r", SHAPES)
def test_values_beyond_the_largest_of_bf16(workspace, n, i, o, r, y_kind):
    """m between bf16's largest number and 32 bits': finite, and so are its products."""
    announce(f"m beyond bf16's largest, {n} x {i} -> {o}, rank {r}, {y_kind}")
    c, g, at = case(n, i, o, r, "bf16")
    largest = 255.0 * 2.0**120
    rows = c.xr()[at]
    c.x[rows] = 0.0
    c.x[rows, 2], c.x[rows, 3] = largest, 2.0**119
    c.w[:, 2:4] = 0.0
    c.down[g][:, 2:4] = 1.0  # m = (255 + 1/2) 2^120, which rounds to an infinity
    c.up[g] = decode(encode(c.up[g] * 2.0**-30, "bf16"), "bf16")
    z = forward_is(c, g, at, y_kind, workspace)
    assert np.isfinite(z).all()
    mid = np.where(np.arange(n)[:, None] % 50 == 0, 255.5 * 2.0**120, np.ones((n, r)))
    c.delta = decode(encode(c.delta * 2.0**-60, "bf16"), "bf16")
    c.up[g] = decode(encode(c.up[g] * 2.0**30, "bf16"), "bf16")
    got = backward_is(c, g, at, mid, workspace, d_columns=(0, o - 1))
    assert np.isfinite(got["dup"][g]).all()
