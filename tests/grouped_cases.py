"""Rows in groups, grouped linear layers and adapters: 64-bit definitions, group
by group, and bounds of the kernels' arithmetic; calls on the device."""
import numpy as np

from linear_cases import CODES, EPS, act, act_error, decode, encode, rounding, slope
from nerf_amd import _lib as L

OLD = 0.5  # what outputs hold before a call


def group_rows(ids, groups):
    ids = np.minimum(np.asarray(ids, np.int64), groups)
    order = np.argsort(ids, kind="stable")
    place = np.empty(len(ids), np.int64)
    place[order] = np.arange(len(ids))
    return np.searchsorted(ids[order], np.arange(groups + 1)), order, place


def sizes_of(n, groups, rng, kind="uneven"):
    """Offsets of groups of n positions: uneven with some empty and some rows in none;
    everything in one; one row each; nothing in any."""
    if kind == "one":
        g = int(rng.integers(groups))
        return np.where(np.arange(groups + 1) > g, n, 0)
    if kind == "each":
        return np.minimum(np.arange(groups + 1), n)
    if kind == "none":
        return np.full(groups + 1, n // 2)
    share = rng.random(groups) ** 2 * (rng.random(groups) > 0.25) + 1e-9
    ends = np.cumsum(share) / share.sum() * (n - n // 9)
    return np.concatenate([[0], np.floor(ends + 1e-6).astype(np.int64)]) + n // 18


class Case:
    """Inputs of one call on the host, whole numbers or not, with the rows' indexes."""

    def __init__(self, n, groups, i, o, kind, seed, rank=0, gather=False, scatter=False, sizes="uneven", whole=False, extra=0):
        rng = np.random.default_rng(seed)
        self.n, self.groups, self.i, self.o, self.rank, self.kind, self.whole = n, groups, i, o, rank, kind, whole
        self.offsets = sizes_of(n, groups, rng, sizes)
        # Indexes into arrays that have more rows than there are positions.
        self.x_count, self.y_count = n + (extra if gather else 0), n + (extra if scatter else 0)
        self.x_rows = rng.permutation(self.x_count)[:n] if gather else None
        self.y_rows = rng.permutation(self.y_count)[:n] if scatter else None

        def values(shape, scale, most=2):
            v = rng.integers(-most, most + 1, shape).astype(np.float64) if whole else rng.normal(0, scale, shape)
            return decode(encode(v, kind), kind)

        def f32(shape, scale, most=8):
            return rng.integers(-most, most + 1, shape).astype(np.float64) if whole else rng.normal(0, scale, shape).astype(np.float32).astype(np.float64)

        shared = rank > 0
        self.x = values((self.x_count, i), 1.0)
        self.w = values((o, i) if shared else (groups, o, i), i**-0.5)
        self.bias = f32((o,) if shared else (groups, o), 0.1)
        self.residual, self.delta = values((self.y_count, o), 1.0, 8), values((self.y_count, o), 0.1)
        self.add, self.pre = values((self.x_count, i), 0.1, 8), values((self.x_count, i), 1.0, 3)
        self.pre = np.where(self.pre == 0.0, 1.0, self.pre)
        if shared:
            self.down, self.up = values((groups, rank, i), i**-0.5, 1), values((groups, o, rank), rank**-0.5, 1)
            self.scales = rng.choice([0.5, 1.0, 2.0], groups) if whole else f32((groups,), 1.0)

    def xr(self):
        return np.arange(self.n) if self.x_rows is None else self.x_rows

    def yr(self):
        return np.arange(self.n) if self.y_rows is None else self.y_rows

    def spans(self):
        return [(g, int(a), int(b)) for g, (a, b) in enumerate(zip(self.offsets, self.offsets[1:])) if b > a]


def _spread(values, bound, rows, written, count):
    """Outputs by position into an array's rows; the others keep OLD."""
    full, off = np.full((count, values.shape[1]), OLD), np.zeros((count, values.shape[1]))
    full[rows[written]], off[rows[written]] = values[written], bound[written]
    return full, off


def forward(c, name, y_kind, bias=True, residual=True):
    """{output: (value, bound)}: a sum of k products in 32 bits in any order is within
    (k + 2) EPS of the sum of their magnitudes; the activations' slopes are at most 1.13.
    An adapter's part: mid by its own sum, its split into two pieces of the type (three
    for fp32 outputs of bf16) leaves 2^-16 of bf16 values (2^-24), 2^-22 of the row's
    largest fp16 value; twice the sum's length, one product and one sum more."""
    x, xr, yr = c.x[c.xr()], c.xr(), c.yr()
    z, dz = np.zeros((c.n, c.o)), np.zeros((c.n, c.o))
    written = np.zeros(c.n, bool)
    out = {}
    if c.rank:
        z, dz = x @ c.w.T, (c.i + 2) * EPS * (np.abs(x) @ np.abs(c.w).T)
        mid, dmid = np.full((c.n, c.rank), OLD), np.zeros((c.n, c.rank))
        split = 2.0**-22 if c.kind == "f16" else 2.0**-24 if y_kind == "f32" else 2.0**-16
        for g, a, b in c.spans():
            mid[a:b], dmid[a:b] = x[a:b] @ c.down[g].T, (c.i + 2) * EPS * (np.abs(x[a:b]) @ np.abs(c.down[g]).T)
            size = np.abs(mid[a:b]) + dmid[a:b]
            rest = split * (size.max(1, keepdims=True) if c.kind == "f16" else size)
            z[a:b] += c.scales[g] * (mid[a:b] @ c.up[g].T)
            dz[a:b] += np.abs(c.scales[g]) * ((dmid[a:b] + rest + (3 * c.rank + 4) * EPS * size) @ np.abs(c.up[g]).T) + 2 * EPS * np.abs(z[a:b])
        out["mid"] = (mid, dmid)
        written[:] = True
    else:
        for g, a, b in c.spans():
            z[a:b], dz[a:b] = x[a:b] @ c.w[g].T, (c.i + 2) * EPS * (np.abs(x[a:b]) @ np.abs(c.w[g]).T)
            written[a:b] = True
    if bias:
        for g, a, b in [(0, 0, c.n)] if c.rank else c.spans():
            each = c.bias if c.rank else c.bias[g]
            z[a:b], dz[a:b] = z[a:b] + each, dz[a:b] + 2 * EPS * (np.abs(each) + np.abs(z[a:b]))
    y, dy = act(z, name), 1.13 * dz + act_error(z, name)
    if residual:
        y = y + c.residual[yr]
        dy = dy + EPS * np.abs(y)
    out["y"] = _spread(y, dy + rounding(np.abs(y) + dy, y_kind), yr, written, c.y_count)
    out["pre"] = _spread(z, dz + rounding(np.abs(z) + dz, c.kind), yr, written, c.y_count)
    return out


def backward(c, name, add=True, mid=None):
    d, x, xr = c.delta[c.yr()], c.x[c.xr()], c.xr()
    g_, dg, written = np.zeros((c.n, c.i)), np.zeros((c.n, c.i)), np.zeros(c.n, bool)
    out = {}
    if c.rank:
        g_, dg = d @ c.w, (c.o + 2) * EPS * (np.abs(d) @ np.abs(c.w))
        written[:] = True
        dmid, ddmid = np.full((c.n, c.rank), OLD), np.zeros((c.n, c.rank))
        ddown, eddown = np.zeros((c.groups, c.rank, c.i)), np.zeros((c.groups, c.rank, c.i))
        dup, edup = np.zeros((c.groups, c.o, c.rank)), np.zeros((c.groups, c.o, c.rank))
        split = 2.0**-22 if c.kind == "f16" else 2.0**-16
        for g, a, b in c.spans():
            s, k = c.scales[g], (b - a + 4) * EPS
            dmid[a:b], ddmid[a:b] = s * (d[a:b] @ c.up[g]), (c.o + 4) * EPS * np.abs(s) * (np.abs(d[a:b]) @ np.abs(c.up[g]))
            size = np.abs(dmid[a:b]) + ddmid[a:b]
            rest = split * (size.max(1, keepdims=True) if c.kind == "f16" else size)
            g_[a:b] += dmid[a:b] @ c.down[g]
            dg[a:b] += (ddmid[a:b] + rest + (3 * c.rank + 4) * EPS * size) @ np.abs(c.down[g]) + 2 * EPS * np.abs(g_[a:b])
            ddown[g], eddown[g] = dmid[a:b].T @ x[a:b], (ddmid[a:b] + k * size).T @ np.abs(x[a:b])
            dup[g], edup[g] = s * (d[a:b].T @ mid[a:b]), k * np.abs(s) * (np.abs(d[a:b]).T @ np.abs(mid[a:b]))
        out = {"dmid": (dmid, ddmid), "ddown": (ddown, eddown + 2.0**-140), "dup": (dup, edup + 2.0**-140)}
    else:
        dw, edw, db, edb = np.zeros(c.w.shape), np.zeros(c.w.shape), np.zeros(c.bias.shape), np.zeros(c.bias.shape)
        for g, a, b in c.spans():
            k = (b - a + 2) * EPS
            g_[a:b], dg[a:b] = d[a:b] @ c.w[g], (c.o + 2) * EPS * (np.abs(d[a:b]) @ np.abs(c.w[g]))
            written[a:b] = True
            dw[g], edw[g] = d[a:b].T @ x[a:b], k * (np.abs(d[a:b]).T @ np.abs(x[a:b]))
            db[g], edb[g] = d[a:b].sum(0), k * np.abs(d[a:b]).sum(0)
        out = {"dw": (dw, edw + 2.0**-140), "db": (db, edb + 2.0**-140)}
    if add:
        g_ = g_ + c.add[xr]
        dg = dg + 2 * EPS * (np.abs(c.add[xr]) + np.abs(g_))
    s = slope(c.pre[xr], name)
    p = g_ * s
    dp = dg * np.abs(s) + (np.abs(g_) + dg) * 16.0 * act_error(c.pre[xr], name) + EPS * np.abs(p)
    out["dx"] = _spread(g_, dg + rounding(np.abs(g_) + dg, c.kind), xr, written, c.x_count)
    out["dpre"] = _spread(p, dp + rounding(np.abs(p) + dp, c.kind), xr, written, c.x_count)
    return out


# -------------------------------------------------------------------- device
def upload(values, kind, pad=0, lead=0):
    """A device array of `lead` values and then rows of one more than `pad` unused
    values each; (array, address of the first row)."""
    from nerf_amd.device import DeviceArray

    bits = encode(values, kind)
    flat = bits.reshape(-1, bits.shape[-1])
    host = np.full((flat.shape[0], flat.shape[1] + pad), 0x7FFF if kind != "f32" else np.nan, bits.dtype)  # NaN between the rows
    host[:, : flat.shape[1]] = flat
    a = DeviceArray.from_numpy(np.concatenate([np.zeros(lead, bits.dtype), host.reshape(-1)]))
    return a, a.ptr + lead * bits.itemsize


class Out:
    """A device array of outputs that hold OLD, with guards before and behind."""

    GUARD = 64

    def __init__(self, shape, kind, pad=0, lead=0):
        from nerf_amd.device import DeviceArray

        self.shape, self.kind, self.pad, self.lead = shape, kind, pad, self.GUARD + lead
        width = shape[-1] + pad
        self.rows, self.width = int(np.prod(shape[:-1], dtype=np.int64)), width
        self.host = encode(np.full(self.lead + self.rows * width + self.GUARD, OLD), kind)
        self.array = DeviceArray.from_numpy(self.host)
        self.ptr = self.array.ptr + self.lead * self.host.itemsize

    def values(self):
        """The outputs; nothing around them may have changed."""
        got = self.array.numpy()
        old = self.host[0]
        assert (got[: self.lead] == old).all() and (got[self.lead + self.rows * self.width :] == old).all(), "written around the array"
        rows = got[self.lead : self.lead + self.rows * self.width].reshape(self.rows, self.width)
        assert (rows[:, self.shape[-1] :] == old).all(), "written between rows"
        return decode(rows[:, : self.shape[-1]], self.kind).reshape(self.shape)


class Device:
    """A case's inputs on the device; pads: unused values behind rows of x, y."""

    def __init__(self, c, x_pad=0, y_pad=0, lead=0):
        from nerf_amd.device import DeviceArray

        self.c, self.keep = c, []
        self.x_pad, self.y_pad, self.lead = x_pad, y_pad, lead

        def put(values, kind, pad=0):
            a, at = upload(values, kind, pad, lead if kind != "f32" else 0)
            self.keep.append(a)
            return at

        self.x, self.w, self.bias = put(c.x, c.kind, x_pad), put(c.w, c.kind), put(c.bias, "f32")
        self.residual, self.delta = put(c.residual, c.kind, y_pad), put(c.delta, c.kind, y_pad)
        self.add, self.pre = put(c.add, c.kind, x_pad), put(c.pre, c.kind)
        index = [DeviceArray.from_numpy(np.asarray(v, np.uint32)) if v is not None else None for v in (c.offsets, c.x_rows, c.y_rows)]
        self.keep += index
        self.groups = L.NerfExtRowGroups(index[0].ptr, index[1].ptr if index[1] else None, index[2].ptr if index[2] else None, c.groups, c.x_count if index[1] else 0, c.y_count if index[2] else 0, 0)
        if c.rank:
            self.adapters = L.NerfExtAdapters(put(c.down, c.kind), put(c.up, c.kind), put(c.scales, "f32"), c.rank, 0)

    def desc(self, name, y_kind=None):
        from linear_cases import ACTS

        c = self.c
        return L.NerfExtLinearDesc(c.n, c.i, c.o, CODES[c.kind], CODES[y_kind or c.kind], ACTS[name], c.i + self.x_pad, c.o + self.y_pad, c.o + self.y_pad, 0)
