"""The work of a user's networks for many regions or scenes at once, as
measurable cases: rows put in groups by an id, a linear layer with weights of
its own for every group, and low-rank adapters of every group beside a shared
linear layer, the layers with their gradients.

Twelve listed cases; draw() gives further cases of the same ranges.  Where
`own` is false, run() computes an operator by elementary torch operations in 32
bits, rounded once at the end (groups as a batch of products, each padded to the
longest); where it is true, it calls the framework through nerf_amd on device
memory that torch allocated (torch's default stream is the library's null
stream).  Group sizes are uneven, some groups are empty, and the rows that are
in no group keep what their outputs held.
"""
import ctypes as C
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
ACTIVATIONS = ("none", "relu", "softplus", "sigmoid", "silu", "gelu")
GELU_A, GELU_B = math.sqrt(2.0 / math.pi), 0.044715
WORKSPACE, GROUP_WORKSPACE = 64 << 20, 16 << 20
OLD = 0.5  # what outputs hold before the call


def listed():
    return [
        # The samples of some rays by the region that they fall into.
        {"name": "group_rays", "kind": "group", "n": 4099, "groups": 64},
        # The samples of a large training batch by 16^3 regions.
        {"name": "group_batch", "kind": "group", "n": 1 << 20, "groups": 4096},
        # Eight samples of a query stepped by hand, through the regions' networks:
        # latency alone.
        {"name": "forward_few", "kind": "forward", "n": 8, "groups": 64, "in": 256, "out": 256, "type": "f16", "y": "f16", "act": "relu", "residual": False, "pre": False, "gather": True, "scatter": True},
        # The first layer of 512 small region networks on a frequency encoding of 63
        # features, in the samples' order: rows of odd length, gathered.
        {"name": "forward_encoded", "kind": "forward", "n": 1 << 18, "groups": 512, "in": 63, "out": 64, "type": "f16", "y": "f16", "act": "relu", "residual": False, "pre": True, "gather": True, "scatter": False},
        # A residual hidden layer of 64 region networks on a training batch.
        {"name": "forward_regions", "kind": "forward", "n": 1 << 18, "groups": 64, "in": 256, "out": 256, "type": "f16", "y": "f16", "act": "relu", "residual": True, "pre": True, "gather": False, "scatter": False},
        # The wide layers of eight large scene representations.
        {"name": "forward_wide", "kind": "forward", "n": 16384, "groups": 8, "in": 4096, "out": 4096, "type": "bf16", "y": "bf16", "act": "gelu", "residual": False, "pre": False, "gather": True, "scatter": True},
        # Gradients of the hidden layer of the region networks.
        {"name": "backward_regions", "kind": "backward", "n": 1 << 18, "groups": 64, "in": 256, "out": 256, "type": "f16", "act": "relu", "add": False, "dx": False, "gather": False, "scatter": False},
        # Gradients of the wide layers.
        {"name": "backward_wide", "kind": "backward", "n": 16384, "groups": 8, "in": 2048, "out": 4096, "type": "bf16", "act": "gelu", "add": False, "dx": False, "gather": False, "scatter": True},
        # One row each of 32 requests, every one with an adapter of its own.
        {"name": "adapter_requests", "kind": "adapter", "n": 32, "groups": 32, "rank": 16, "in": 4096, "out": 4096, "type": "bf16", "y": "bf16", "act": "silu", "residual": False, "pre": False, "gather": True, "scatter": True},
        # A hidden layer shared by 16 scenes, a training batch of all of them.
        {"name": "adapter_scenes", "kind": "adapter", "n": 1 << 18, "groups": 16, "rank": 16, "in": 256, "out": 256, "type": "f16", "y": "f16", "act": "relu", "residual": True, "pre": True, "gather": False, "scatter": False},
        # Its gradients, the shared weights held.
        {"name": "adapter_backward_scenes", "kind": "adapter_backward", "n": 1 << 18, "groups": 16, "rank": 16, "in": 256, "out": 256, "type": "f16", "act": "relu", "add": True, "dx": True, "gather": False, "scatter": False},
        # Gradients of adapters of a higher rank on a wide layer.
        {"name": "adapter_backward_wide", "kind": "adapter_backward", "n": 8192, "groups": 8, "rank": 64, "in": 4096, "out": 2048, "type": "bf16", "act": "gelu", "add": False, "dx": False, "gather": True, "scatter": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["group", "forward", "forward", "backward", "adapter", "adapter", "adapter_backward"])
    if kind == "group":
        return {"kind": kind, "n": _log(rng, 1, 1 << 20), "groups": _log(rng, 1, 4096)}
    # Widths from a few features to thousands, as often odd as whole multiples of
    # 32; rows from one sample to a training batch, within the listed work.
    width = [_log(rng, 1, 2047) | 1 if rng.random() < 0.5 else 32 * _log(rng, 1, 63) for _ in range(2)]
    groups = min(_log(rng, 1, 512), max(1, (1 << 25) // (width[0] * width[1])))
    most = min(1 << 18, (1 << 26) // max(width), (1 << 37) // (width[0] * width[1]))
    case = {"kind": kind, "n": _log(rng, 1, most), "groups": groups, "in": width[0], "out": width[1], "type": rng.choice(["f16", "bf16"]), "act": rng.choice(ACTIVATIONS), "gather": rng.random() < 0.5, "scatter": rng.random() < 0.5}
    if kind.startswith("adapter"):
        case["rank"] = rng.choice([_log(rng, 1, 64), 8, 16, 32])
        case["scatter"] = case["gather"]
    if kind in ("forward", "adapter"):
        return case | {"y": rng.choice([case["type"], case["type"], "f32"]), "residual": rng.random() < 0.5, "pre": rng.random() < 0.5}
    return case | {"add": rng.random() < 0.5, "dx": rng.random() < 0.5}


# ----------------------------------------------------------------- inputs
def _normal(g, shape, scale, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _old(shape, dtype):
    return torch.full(shape, OLD, dtype=dtype, device=DEV)


def _pointer(t):
    return None if t is None else t.data_ptr()


def _ids(g, n, groups):
    """A group for every row, in no order: of uneven sizes, with one group in eight
    left empty and one row in 64 in none (where there are several)."""
    share = torch.rand((groups,), generator=g, device=DEV, dtype=torch.float64).square() + 0.1
    if groups > 1:
        share = share * (torch.rand((groups,), generator=g, device=DEV) > 0.125)
        share[int(torch.randint(groups, (1,), generator=g, device=DEV))] += 0.5
    bounds = torch.cumsum(share, 0)
    ids = torch.searchsorted(bounds, torch.rand((n,), generator=g, device=DEV, dtype=torch.float64) * bounds[-1], right=True)
    return torch.where(torch.rand((n,), generator=g, device=DEV) < 1.0 / 64.0, groups, ids.clamp(max=groups)).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + 29)
    n, groups = case["n"], case["groups"]
    ids = _ids(g, n, groups)
    s = {"case": case}
    if case["kind"] == "group":
        s["ids"] = ids
        s["offsets"] = torch.empty((groups + 1,), dtype=torch.int32, device=DEV)
        s["order"] = torch.empty((n,), dtype=torch.int32, device=DEV)
        s["place"] = torch.empty((n,), dtype=torch.int32, device=DEV)
        s["workspace"] = torch.empty(GROUP_WORKSPACE, dtype=torch.uint8, device=DEV)
        return s
    i, o, t = case["in"], case["out"], TYPES[case["type"]]
    ranked, order = torch.sort(ids, stable=True)
    s["offsets"] = torch.searchsorted(ranked, torch.arange(groups + 1, dtype=torch.int32, device=DEV)).to(torch.int32)
    s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # rows of the largest group
    s["order"] = order.to(torch.int32)
    s["x_rows"] = s["order"] if case["gather"] else None
    s["y_rows"] = s["order"] if case["scatter"] else None
    s["x"] = _normal(g, (n, i), 1.0, t)
    adapter = case["kind"].startswith("adapter")
    s["w"] = ((torch.rand((o, i) if adapter else (groups, o, i), generator=g, device=DEV) * 2.0 - 1.0) * math.sqrt(6.0 / (i + o))).to(t)
    s["workspace"] = torch.empty(WORKSPACE, dtype=torch.uint8, device=DEV)
    if adapter:
        r = case["rank"]
        s["down"] = _normal(g, (groups, r, i), 1.0 / math.sqrt(i), t)
        s["up"] = _normal(g, (groups, o, r), 0.5 / math.sqrt(r), t)
        s["scales"] = torch.rand((groups,), generator=g, device=DEV) + 0.5
        s["mid"] = _old((n, r), torch.float32)
    if case["kind"] in ("forward", "adapter"):
        s["bias"] = _normal(g, (o,) if adapter else (groups, o), 0.1)
        s["residual"] = _normal(g, (n, o), 1.0, t) if case["residual"] else None
        s["y"] = _old((n, o), TYPES[case["y"]])
        s["pre"] = _old((n, o), t) if case["pre"] else None
        return s
    s["delta"] = _normal(g, (n, o), 0.05, t)
    s["prior"] = _normal(g, (n, i), 1.0, t)
    s["add"] = _normal(g, (n, i), 0.05, t) if case["add"] else None
    s["dx"] = _old((n, i), t) if case["dx"] else None
    s["dpre"] = _old((n, i), t)
    if adapter:
        _plain_mid(s)  # as the forward pass left it
        s["dmid"] = _old((n, r), torch.float32)
        s["ddown"] = torch.empty((groups, r, i), device=DEV)
        s["dup"] = torch.empty((groups, o, r), device=DEV)
    else:
        s["dw"] = torch.empty((groups, o, i), device=DEV)
        s["db"] = torch.empty((groups, o), device=DEV)
    return s


# ------------------------------------------------------------- plain forms
def _act(z, name):
    if name == "relu":
        return torch.clamp(z, min=0.0)
    if name == "softplus":
        return torch.clamp(z, min=0.0) + torch.log1p(torch.exp(-z.abs()))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(GELU_A * (z + GELU_B * z * z * z)))
    return z


def _derivative(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "none":
        return torch.ones_like(z)
    if name == "gelu":
        h = torch.tanh(GELU_A * (z + GELU_B * z * z * z))
        return 0.5 * (1.0 + h) + 0.5 * z * (1.0 - h * h) * GELU_A * (1.0 + 3.0 * GELU_B * z * z)
    q = 1.0 / (1.0 + torch.exp(-z))
    return q if name == "softplus" else q * (1.0 - q) if name == "sigmoid" else q * (1.0 + z * (1.0 - q))


def _places(s):
    """Positions of the padded batch [groups][most] and which of them are a group's;
    of every position its group (any, for those in none), place and whether it is in one."""
    n, groups, offsets = s["case"]["n"], s["case"]["groups"], s["offsets"].long()
    padded = offsets[:-1, None] + torch.arange(s["most"], device=DEV)
    inside = padded < offsets[1:, None]
    position = torch.arange(n, device=DEV)
    group = torch.searchsorted(offsets[1:], position, right=True)
    member = group < groups
    group = group.clamp(max=groups - 1)
    return padded.clamp(max=n - 1), inside, group, torch.where(member, position - offsets[group], 0), member


def _rows(s, t, index):
    """The rows of t at every position, in 32 bits."""
    return t.float() if index is None else t[index.long()].float()


def _batched(rows, places):
    return rows[places[0]] * places[1][:, :, None]


def _positions(batch, places):
    return batch[places[2], places[3]] if batch.shape[1] else batch.new_zeros((places[2].shape[0], batch.shape[2]))


def _put(out, index, values, member):
    """Rows of `out` at the member positions become `values`; the others stay."""
    if index is None:
        out.copy_(torch.where(member[:, None], values.to(out.dtype), out))
    else:
        out[index.long()] = torch.where(member[:, None], values.to(out.dtype), out[index.long()])


def _plain_group(s):
    ranked, order = torch.sort(s["ids"].clamp(max=s["case"]["groups"]), stable=True)
    s["offsets"].copy_(torch.searchsorted(ranked, torch.arange(s["case"]["groups"] + 1, dtype=torch.int32, device=DEV)))
    s["order"].copy_(order)
    s["place"][order] = torch.arange(s["case"]["n"], dtype=torch.int32, device=DEV)
    return {k: s[k] for k in ("offsets", "order", "place")}


def _finish(s, z, member):
    """What becomes of the sums z at every position."""
    case = s["case"]
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + _rows(s, s["residual"], s["y_rows"])
    _put(s["y"], s["y_rows"], y, member)
    if case["pre"]:
        _put(s["pre"], s["y_rows"], z, member)
    return {k: s[k] for k in ("y",) + (("pre",) if case["pre"] else ())}


def _plain_forward(s):
    places = _places(s)
    x = _batched(_rows(s, s["x"], s["x_rows"]), places)
    z = torch.bmm(x, s["w"].float().transpose(1, 2).contiguous()) + s["bias"][:, None, :]
    return _finish(s, _positions(z, places), places[4])


def _finish_gradient(s, g, member):
    case = s["case"]
    if s["add"] is not None:
        g = g + _rows(s, s["add"], s["x_rows"])
    _put(s["dpre"], s["x_rows"], g * _derivative(_rows(s, s["prior"], s["x_rows"]), case["act"]), member)
    if case["dx"]:
        _put(s["dx"], s["x_rows"], g, member)
    return {k: s[k] for k in ("dpre",) + (("dx",) if case["dx"] else ())}


def _plain_backward(s):
    places = _places(s)
    d, x = _batched(_rows(s, s["delta"], s["y_rows"]), places), _batched(_rows(s, s["x"], s["x_rows"]), places)
    s["dw"].copy_(torch.bmm(d.transpose(1, 2).contiguous(), x))
    s["db"].copy_(d.sum(1))
    return _finish_gradient(s, _positions(torch.bmm(d, s["w"].float()), places), places[4]) | {"dw": s["dw"], "db": s["db"]}


def _plain_mid(s):
    places = _places(s)
    x = _batched(_rows(s, s["x"], s["x_rows"]), places)
    _put(s["mid"], None, _positions(torch.bmm(x, s["down"].float().transpose(1, 2).contiguous()), places), places[4])
    return places


def _plain_adapter(s):
    places = _plain_mid(s)
    low = torch.bmm(_batched(s["mid"], places), s["up"].float().transpose(1, 2).contiguous()) * s["scales"][:, None, None]
    z = _rows(s, s["x"], s["x_rows"]) @ s["w"].float().t() + s["bias"]
    z = z + torch.where(places[4][:, None], _positions(low, places), 0.0)
    return _finish(s, z, torch.ones_like(places[4])) | {"mid": s["mid"]}


def _plain_adapter_backward(s):
    places = _places(s)
    rows = _rows(s, s["delta"], s["y_rows"])
    d, x, mid = _batched(rows, places), _batched(_rows(s, s["x"], s["x_rows"]), places), _batched(s["mid"], places)
    dmid = torch.bmm(d, s["up"].float()) * s["scales"][:, None, None]
    _put(s["dmid"], None, _positions(dmid, places), places[4])
    s["ddown"].copy_(torch.bmm(dmid.transpose(1, 2).contiguous(), x))
    s["dup"].copy_(torch.bmm(d.transpose(1, 2).contiguous(), mid) * s["scales"][:, None, None])
    g = rows @ s["w"].float() + torch.where(places[4][:, None], _positions(torch.bmm(dmid, s["down"].float()), places), 0.0)
    return _finish_gradient(s, g, torch.ones_like(places[4])) | {k: s[k] for k in ("dmid", "ddown", "dup")}


# ----------------------------------------------------- the framework's calls
def _own_group(s):
    from nerf_amd import _lib as L

    c = s["case"]
    L.call("nerf_ext_group_rows", s["ids"].data_ptr(), c["n"], c["groups"], *[s[k].data_ptr() for k in ("offsets", "order", "place", "workspace")], GROUP_WORKSPACE, None)
    return {k: s[k] for k in ("offsets", "order", "place")}


def _arguments(s, names):
    """The layer's call on the case's arrays, made once as a program keeps it."""
    from nerf_amd import _lib as L

    if "args" not in s:
        c = s["case"]
        s["desc"] = L.NerfExtLinearDesc(c["n"], c["in"], c["out"], CODES[c["type"]], CODES[c.get("y", c["type"])], ACTIVATIONS.index(c["act"]), 0, 0, 0, 0)
        s["rows"] = L.NerfExtRowGroups(s["offsets"].data_ptr(), _pointer(s["x_rows"]), _pointer(s["y_rows"]), c["groups"], 0, 0, 0)
        s["args"] = [C.byref(s["desc"]), C.byref(s["rows"])]
        if c["kind"].startswith("adapter"):
            s["adapters"] = L.NerfExtAdapters(s["down"].data_ptr(), s["up"].data_ptr(), s["scales"].data_ptr(), c["rank"], 0)
            s["args"].append(C.byref(s["adapters"]))
        s["args"] += [_pointer(s[k]) for k in names] + [s["workspace"].data_ptr(), WORKSPACE, None]
    return s["args"]


def _own_forward(s):
    from nerf_amd import _lib as L

    L.call("nerf_ext_grouped_linear_forward", *_arguments(s, ("x", "w", "bias", "residual", "y", "pre")))
    return {k: s[k] for k in ("y",) + (("pre",) if s["case"]["pre"] else ())}


def _own_backward(s):
    from nerf_amd import _lib as L

    L.call("nerf_ext_grouped_linear_backward", *_arguments(s, ("x", "w", "delta", "prior", "add", "dx", "dpre", "dw", "db")))
    return {k: s[k] for k in ("dpre", "dw", "db") + (("dx",) if s["case"]["dx"] else ())}


def _own_adapter(s):
    from nerf_amd import _lib as L

    L.call("nerf_ext_adapter_linear_forward", *_arguments(s, ("x", "w", "bias", "residual", "y", "pre", "mid")))
    return {k: s[k] for k in ("y", "mid") + (("pre",) if s["case"]["pre"] else ())}


def _own_adapter_backward(s):
    from nerf_amd import _lib as L

    L.call("nerf_ext_adapter_linear_backward", *_arguments(s, ("x", "w", "delta", "mid", "prior", "add", "dx", "dpre", "dmid", "ddown", "dup")))
    return {k: s[k] for k in ("dpre", "dmid", "ddown", "dup") + (("dx",) if s["case"]["dx"] else ())}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"group": _own_group, "forward": _own_forward, "backward": _own_backward, "adapter": _own_adapter, "adapter_backward": _own_adapter_backward}[kind](state)
    return {"group": _plain_group, "forward": _plain_forward, "backward": _plain_backward, "adapter": _plain_adapter, "adapter_backward": _plain_adapter_backward}[kind](state)


def work(case):
    n, groups = case["n"], case["groups"]
    if case["kind"] == "group":
        return {"bytes": 12 * n + 4 * groups + 4, "flops": n}
    i, o, used = case["in"], case["out"], min(n, groups)  # groups that can have rows
    index = 4 * groups + 4 + 4 * n * (case["gather"] or case["scatter"])
    if case["kind"] == "forward":
        wide = 4 if case["y"] == "f32" else 2
        return {"bytes": index + 2 * (n * i + used * o * i + n * o * (case["residual"] + case["pre"])) + wide * n * o + 4 * used * o, "flops": 2 * n * i * o}
    if case["kind"] == "backward":
        return {"bytes": index + 2 * (n * o + used * o * i + n * i * (3 + case["add"] + case["dx"])) + 4 * groups * (o * i + o), "flops": 4 * n * i * o}
    r = case["rank"]
    if case["kind"] == "adapter":
        wide = 4 if case["y"] == "f32" else 2
        return {"bytes": index + 2 * (n * i + o * i + used * r * (i + o) + n * o * (case["residual"] + case["pre"])) + wide * n * o + 4 * (o + used + n * r), "flops": 2 * n * (i * o + r * (i + o))}
    return {"bytes": index + 2 * (n * o + o * i + used * r * (i + o) + n * i * (3 + case["add"] + case["dx"])) + 4 * (2 * n * r + used + groups * r * (i + o)), "flops": 2 * n * (i * o + 2 * r * (i + o))}


# ------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    """The operators' definitions in 64 bits on the same inputs, group by group."""
    s = prepare(case, seed)
    n, groups, kind = case["n"], case["groups"], case["kind"]
    if kind == "group":
        ids = s["ids"].tolist()
        lists = [[] for _ in range(groups + 1)]
        for row, g in enumerate(ids):
            lists[g].append(row)
        order = [row for rows in lists for row in rows]
        place = [0] * n
        for position, row in enumerate(order):
            place[row] = position
        ends = [0]
        for rows in lists[:groups]:
            ends.append(ends[-1] + len(rows))
        return {k: torch.tensor(v, dtype=torch.int32, device=DEV) for k, v in (("offsets", ends), ("order", order), ("place", place))}
    offsets = s["offsets"].tolist()
    adapter = kind.startswith("adapter")
    everywhere = torch.arange(n, device=DEV)
    xr = everywhere if s["x_rows"] is None else s["x_rows"].long()
    yr = everywhere if s["y_rows"] is None else s["y_rows"].long()
    spans = [(g, a, b) for g, (a, b) in enumerate(zip(offsets, offsets[1:]))]
    f = torch.nn.functional
    act = {"none": lambda z: z, "relu": torch.relu, "softplus": lambda z: torch.logaddexp(z, torch.zeros_like(z)), "sigmoid": torch.sigmoid, "silu": f.silu, "gelu": lambda z: f.gelu(z, approximate="tanh")}[case["act"]]
    # The rows that get outputs, by position: an adapter's call covers all.
    written = everywhere if adapter else torch.cat([everywhere[a:b] for _, a, b in spans])

    def old(t):
        return torch.full(t.shape, OLD, dtype=torch.float64, device=DEV)

    w = s["w"].double()
    if kind in ("forward", "adapter"):
        x = s["x"].double()[xr]
        z = f.linear(x, w) if adapter else torch.zeros((n, case["out"]), dtype=torch.float64, device=DEV)
        mid = old(s["mid"]) if adapter else None
        for g, a, b in spans:
            if adapter:
                mid[a:b] = f.linear(x[a:b], s["down"][g].double())
                z[a:b] += float(s["scales"][g]) * f.linear(mid[a:b], s["up"][g].double())
            else:
                z[a:b] = f.linear(x[a:b], w[g], s["bias"][g].double())
        if adapter:
            z += s["bias"].double()
        y = act(z)
        if s["residual"] is not None:
            y = y + s["residual"].double()[yr]
        out = {"y": old(s["y"])}
        out["y"][yr[written]] = y[written]
        if case["pre"]:
            out["pre"] = old(s["pre"])
            out["pre"][yr[written]] = z[written]
        return out | {"mid": mid} if adapter else out
    d, x = s["delta"].double()[yr], s["x"].double()[xr]
    gx = torch.mm(d, w) if adapter else torch.zeros((n, case["in"]), dtype=torch.float64, device=DEV)
    out = {}
    if adapter:
        out = {k: torch.zeros(s[k].shape, dtype=torch.float64, device=DEV) for k in ("ddown", "dup")} | {"dmid": old(s["dmid"])}
        for g, a, b in spans:
            scale, dg = float(s["scales"][g]), d[a:b]
            out["dmid"][a:b] = scale * torch.mm(dg, s["up"][g].double())
            out["ddown"][g] = torch.mm(out["dmid"][a:b].t().contiguous(), x[a:b])
            out["dup"][g] = scale * torch.mm(dg.t().contiguous(), s["mid"][a:b].double())
            gx[a:b] += torch.mm(out["dmid"][a:b], s["down"][g].double())
    else:
        out = {k: torch.zeros(s[k].shape, dtype=torch.float64, device=DEV) for k in ("dw", "db")}
        for g, a, b in spans:
            gx[a:b] = torch.mm(d[a:b], w[g])
            out["dw"][g] = torch.mm(d[a:b].t().contiguous(), x[a:b])
            out["db"][g] = d[a:b].sum(0)
    if s["add"] is not None:
        gx = gx + s["add"].double()[xr]
    prior = s["prior"].double()[xr].requires_grad_()
    (slope,) = torch.autograd.grad(act(prior).sum(), prior)
    out["dpre"] = old(s["dpre"])
    out["dpre"][xr[written]] = (gx * slope)[written]
    if case["dx"]:
        out["dx"] = old(s["dx"])
        out["dx"][xr[written]] = gx[written]
    return out
