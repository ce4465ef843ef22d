"""A host's own network next to the fields of the library: a stack of linear
layers with residual connections, its gradients and its Adam step, all on the
device through nerf_ext_linear_*, nerf_ext_grad_norm and nerf_ext_adam_step.

    net = Network([63, 256, 256, 256, 4], activation="relu")
    y = net.forward(features, rows)            # fp32 [rows][4]
    net.backward(delta, rows)                  # delta fp16 [rows][4] = loss_scale d loss / d y
    net.step(hyper)                            # clip, skip guard and Adam

GroupedNetwork is the same with weights of its own for every group of rows (the
regions of a scene), Adapters a low-rank correction of a Network for every group
(the scenes that share it), through nerf_ext_group_rows,
nerf_ext_grouped_linear_* and nerf_ext_adapter_linear_*.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib as L
from .device import DeviceArray, Stream

ACTIVATIONS = {"none": L.NERF_EXT_ACT_NONE, "relu": L.NERF_EXT_ACT_RELU, "softplus": L.NERF_EXT_ACT_SOFTPLUS, "sigmoid": L.NERF_EXT_ACT_SIGMOID, "silu": L.NERF_EXT_ACT_SILU, "gelu": L.NERF_EXT_ACT_GELU}
ALIGN = 64  # elements: every tensor starts at a multiple of 128 bytes in each array


def linear_forward(desc: L.NerfExtLinearDesc, x: int, weight: int, y: int, *, bias: int | None = None, residual: int | None = None, pre: int | None = None, workspace: DeviceArray | None = None, stream: Stream | None = None) -> None:
    """nerf_ext_linear_forward on device addresses."""
    L.call("nerf_ext_linear_forward", C.byref(desc), x, weight, bias, residual, y, pre, workspace.ptr if workspace else None, workspace.nbytes if workspace else 0, stream.handle if stream else None)


def linear_backward(desc: L.NerfExtLinearDesc, x: int | None, weight: int | None, delta: int, *, pre: int | None = None, add: int | None = None, dx: int | None = None, dpre: int | None = None, dweight: int | None = None, dbias: int | None = None,
                    workspace: DeviceArray | None = None, stream: Stream | None = None) -> None:
    """nerf_ext_linear_backward on device addresses."""
    L.call("nerf_ext_linear_backward", C.byref(desc), x, weight, delta, pre, add, dx, dpre, dweight, dbias, workspace.ptr if workspace else None, workspace.nbytes if workspace else 0, stream.handle if stream else None)


def group_rows(ids: int, rows: int, groups: int, offsets: int, order: int, *, place: int | None = None, workspace: DeviceArray | None = None, stream: Stream | None = None) -> None:
    """nerf_ext_group_rows on device addresses."""
    L.call("nerf_ext_group_rows", ids, rows, groups, offsets, order, place, workspace.ptr if workspace else None, workspace.nbytes if workspace else 0, stream.handle if stream else None)


def grouped_linear_forward(desc: L.NerfExtLinearDesc, groups: L.NerfExtRowGroups, x: int, weight: int, y: int, *, bias: int | None = None, residual: int | None = None, pre: int | None = None, workspace: DeviceArray | None = None,
                           stream: Stream | None = None) -> None:
    """nerf_ext_grouped_linear_forward on device addresses."""
    L.call("nerf_ext_grouped_linear_forward", C.byref(desc), C.byref(groups), x, weight, bias, residual, y, pre, workspace.ptr if workspace else None, workspace.nbytes if workspace else 0, stream.handle if stream else None)


def grouped_linear_backward(desc: L.NerfExtLinearDesc, groups: L.NerfExtRowGroups, x: int | None, weight: int | None, delta: int, *, pre: int | None = None, add: int | None = None, dx: int | None = None, dpre: int | None = None,
                            dweight: int | None = None, dbias: int | None = None, workspace: DeviceArray | None = None, stream: Stream | None = None) -> None:
    """nerf_ext_grouped_linear_backward on device addresses."""
    L.call("nerf_ext_grouped_linear_backward", C.byref(desc), C.byref(groups), x, weight, delta, pre, add, dx, dpre, dweight, dbias, workspace.ptr if workspace else None, workspace.nbytes if workspace else 0, stream.handle if stream else None)


def adapter_linear_forward(desc: L.NerfExtLinearDesc, groups: L.NerfExtRowGroups, adapters: L.NerfExtAdapters, x: int, weight: int, y: int, mid: int, *, bias: int | None = None, residual: int | None = None, pre: int | None = None,
                           workspace: DeviceArray | None = None, stream: Stream | None = None) -> None:
    """nerf_ext_adapter_linear_forward on device addresses."""
    L.call("nerf_ext_adapter_linear_forward", C.byref(desc), C.byref(groups), C.byref(adapters), x, weight, bias, residual, y, pre, mid, workspace.ptr if workspace else None, workspace.nbytes if workspace else 0, stream.handle if stream else None)


def adapter_linear_backward(desc: L.NerfExtLinearDesc, groups: L.NerfExtRowGroups, adapters: L.NerfExtAdapters, x: int | None, weight: int | None, delta: int, *, mid: int | None = None, pre: int | None = None, add: int | None = None,
                            dx: int | None = None, dpre: int | None = None, dmid: int | None = None, ddown: int | None = None, dup: int | None = None, workspace: DeviceArray | None = None, stream: Stream | None = None) -> None:
    """nerf_ext_adapter_linear_backward on device addresses."""
    L.call("nerf_ext_adapter_linear_backward", C.byref(desc), C.byref(groups), C.byref(adapters), x, weight, delta, mid, pre, add, dx, dpre, dmid, ddown, dup, workspace.ptr if workspace else None, workspace.nbytes if workspace else 0,
           stream.handle if stream else None)


def _check_rows(array: DeviceArray, rows: int, width: int, what: str) -> None:
    """Rows of `width` 16-bit values, `rows` of them at least: an array of rows of
    any inner shape, or a flat one."""
    if array.dtype not in (np.float16, np.uint16):
        raise ValueError(f"{what} is {array.dtype}: it must be float16, or its bits as uint16")
    size = int(np.prod(array.shape, dtype=np.int64))
    fits = size >= rows * width if len(array.shape) == 1 else array.shape[0] >= rows and size == array.shape[0] * width
    if not fits:
        raise ValueError(f"{what} has shape {array.shape}: {rows} rows of {width} values are needed")


class _Parameters:
    """fp32 masters with gradients, Adam state and fp16 working copies, one
    allocation a kind; each tensor starts at a multiple of ALIGN elements."""

    def _allocate(self, tensors: list[np.ndarray]) -> None:
        self._sizes, self._at, at = [t.size for t in tensors], [], 0
        for n in self._sizes:
            self._at.append(at)
            at += -(-n // ALIGN) * ALIGN
        host = np.zeros(at, np.float32)
        for a, t in zip(self._at, tensors):
            host[a : a + t.size] = t.reshape(-1)
        self._shapes = [t.shape for t in tensors]
        self.params = DeviceArray.from_numpy(host)
        self.copies = DeviceArray.from_numpy(host.astype(np.float16))
        self.grads, self.m, self.v = (DeviceArray.zeros((at,), np.float32) for _ in range(3))
        self.norm = DeviceArray.zeros((1,), np.float32)
        self.skipped = DeviceArray.zeros((1,), np.uint32)
        self.steps_done = 0
        n = len(tensors)
        self._grad_list = (L.NerfExtGradTensor * n)(*[L.NerfExtGradTensor(self.grads.ptr + 4 * a, None, s, L.NERF_EXT_F32, 0) for a, s in zip(self._at, self._sizes)])
        self._adam_list = (L.NerfExtAdamTensor * n)(
            *[L.NerfExtAdamTensor(self.params.ptr + 4 * a, self.grads.ptr + 4 * a, self.m.ptr + 4 * a, self.v.ptr + 4 * a, self.copies.ptr + 2 * a, s, L.NERF_EXT_F16, 0) for a, s in zip(self._at, self._sizes)])

    def tensor(self, index: int, array: str = "params") -> np.ndarray:
        """Host copy of a tensor (of params, copies, grads, m or v)."""
        return getattr(self, array).numpy()[self._at[index] :][: self._sizes[index]].reshape(self._shapes[index])

    def step(self, hyper: L.NerfHyperParams, stream: Stream | None = None) -> None:
        """Norm of all gradients, then the update of all parameters (clipping and
        skip guard included)."""
        handle = stream.handle if stream else None
        L.call("nerf_ext_grad_norm", self._grad_list, len(self._grad_list), self.norm.ptr, self.workspace.ptr, self.workspace.nbytes, handle)
        L.call("nerf_ext_adam_step", self._adam_list, len(self._adam_list), C.byref(hyper), self.steps_done + 1, self.norm.ptr, self.skipped.ptr, handle)
        self.steps_done += 1


class Network(_Parameters):
    """Layers widths[0] -> ... -> widths[-1]: hidden layers act(x W^T + b), plus
    x where a layer is as wide as its input, then a linear layer with fp32
    outputs.  fp32 masters, fp16 working copies of the weights."""

    def __init__(self, widths: list[int], activation: str = "relu", seed: int = 0, max_rows: int = 1 << 16):
        if len(widths) < 2 or min(widths) < 1:
            raise ValueError("a network has an input and an output width, all positive")
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}")
        self.widths, self.max_rows = list(widths), int(max_rows)
        self.act = ACTIVATIONS[activation]
        self._rows, self._input = None, None  # of the last forward pass
        self.layers = len(widths) - 1
        self.residual = [l < self.layers - 1 and widths[l] == widths[l + 1] for l in range(self.layers)]
        rng = np.random.default_rng(seed)
        tensors = []
        for i, o in zip(widths, widths[1:]):
            bound = np.sqrt(6.0 / (i + o))
            tensors += [rng.uniform(-bound, bound, (o, i)), np.zeros(o)]
        self._allocate(tensors)
        self.workspace = DeviceArray((L.NERF_EXT_LINEAR_WORKSPACE,), np.uint8)
        wide = max(widths[1:-1], default=0)
        # Inputs of every layer but the first, z of every hidden layer, and two deltas
        # and gradients in turn for the way back.
        self._x = [None] + [DeviceArray((self.max_rows, w), np.float16) for w in widths[1:-1]]
        self._z = [DeviceArray((self.max_rows, w), np.float16) for w in widths[1:-1]]
        self._delta, self._g = ([DeviceArray((self.max_rows, max(wide, 1)), np.float16) for _ in range(2)] for _ in range(2))
        self.y = DeviceArray((self.max_rows, widths[-1]), np.float32)

    def weight(self, layer: int, array: str = "params") -> np.ndarray:
        """Host copy of a layer's [out][in] weights (params, copies, grads, m or v)."""
        o, i = self.widths[layer + 1], self.widths[layer]
        return getattr(self, array).numpy()[self._at[2 * layer] :][: o * i].reshape(o, i)

    def bias(self, layer: int, array: str = "params") -> np.ndarray:
        o = self.widths[layer + 1]
        return getattr(self, array).numpy()[self._at[2 * layer + 1] :][:o]

    def _check(self, rows: int) -> None:
        if not 0 <= rows <= self.max_rows:
            raise ValueError(f"{rows} rows: the network was made for at most {self.max_rows}")

    def forward(self, x: DeviceArray, rows: int, stream: Stream | None = None) -> DeviceArray:
        """x: fp16 [rows][widths[0]].  Returns the fp32 outputs, the network's own
        array; keeps what backward() needs (x is read again there).  fp16 arrays may
        be flat, hold more rows, or hold the numbers' bits as uint16."""
        self._check(rows)
        _check_rows(x, rows, self.widths[0], "x")
        self._rows, self._input = None, x
        for l in range(self.layers):
            last = l == self.layers - 1
            i, o = self.widths[l], self.widths[l + 1]
            d = L.NerfExtLinearDesc(rows, i, o, L.NERF_EXT_F16, L.NERF_EXT_F32 if last else L.NERF_EXT_F16, L.NERF_EXT_ACT_NONE if last else self.act, 0, 0, 0, 0)
            src = (x if l == 0 else self._x[l]).ptr
            linear_forward(d, src, self.copies.ptr + 2 * self._at[2 * l], self.y.ptr if last else self._x[l + 1].ptr, bias=self.params.ptr + 4 * self._at[2 * l + 1], residual=src if self.residual[l] else None,
                           pre=None if last else self._z[l].ptr, workspace=self.workspace, stream=stream)
        self._rows = rows
        return self.y

    def backward(self, delta: DeviceArray, rows: int, stream: Stream | None = None) -> None:
        """delta: fp16 [rows][widths[-1]], the loss' derivative in the outputs of the
        last forward() times the loss scale; rows: that forward()'s.  Fills the
        gradients."""
        if rows != self._rows:
            raise ValueError(f"{rows} rows: " + ("no forward pass" if self._rows is None else f"the last forward pass had {self._rows}"))
        _check_rows(delta, rows, self.widths[-1], "delta")
        g = delta  # the gradient in the layer's output, where a residual passes it on
        for l in reversed(range(self.layers)):
            i, o = self.widths[l], self.widths[l + 1]
            d = L.NerfExtLinearDesc(rows, i, o, L.NERF_EXT_F16, L.NERF_EXT_F16, self.act, 0, 0, 0, 0)
            below = l > 0
            dx = self._g[l % 2] if below and self.residual[l - 1] else None
            dpre = self._delta[l % 2] if below else None
            linear_backward(d, (self._input if l == 0 else self._x[l]).ptr, self.copies.ptr + 2 * self._at[2 * l] if below else None, delta.ptr, pre=self._z[l - 1].ptr if below else None, add=g.ptr if below and self.residual[l] else None,
                            dx=dx.ptr if dx else None, dpre=dpre.ptr if dpre else None, dweight=self.grads.ptr + 4 * self._at[2 * l], dbias=self.grads.ptr + 4 * self._at[2 * l + 1], workspace=self.workspace, stream=stream)
            delta, g = dpre, dx


class _GroupedLayers(_Parameters):
    """What layers of rows in groups share: the rows' order, the arrays between the
    layers, in the groups' order, and the way through them.  The first layer reads
    its rows, and the last one writes them, by the order."""

    def __init__(self, widths: list[int], activation: str, groups: int, max_rows: int):
        if len(widths) < 2 or min(widths) < 1:
            raise ValueError("a network has an input and an output width, all positive")
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}")
        if not 1 <= groups <= L.NERF_EXT_MAX_GROUPS:
            raise ValueError(f"{groups} groups: 1 to {L.NERF_EXT_MAX_GROUPS} are possible")
        self.widths, self.groups, self.max_rows, self.layers, self.act = list(widths), int(groups), int(max_rows), len(widths) - 1, ACTIVATIONS[activation]
        self.residual = [0 < l < self.layers - 1 and widths[l] == widths[l + 1] for l in range(self.layers)]
        self._rows, self._input = None, None  # of the last forward pass
        self.workspace = DeviceArray((L.NERF_EXT_LINEAR_WORKSPACE,), np.uint8)
        self.offsets, self.order = DeviceArray.zeros((groups + 1,), np.uint32), DeviceArray.zeros((max(1, max_rows),), np.uint32)
        wide = max(widths[1:-1], default=1)
        self._x = [None] + [DeviceArray((self.max_rows, w), np.float16) for w in widths[1:-1]]
        self._z = [DeviceArray((self.max_rows, w), np.float16) for w in widths[1:-1]]
        self._delta, self._g = ([DeviceArray((self.max_rows, wide), np.float16) for _ in range(2)] for _ in range(2))
        self.y = DeviceArray.zeros((self.max_rows, widths[-1]), np.float32)

    def _groups_of(self, l: int) -> L.NerfExtRowGroups:
        return L.NerfExtRowGroups(self.offsets.ptr, self.order.ptr if l == 0 else None, self.order.ptr if l == self.layers - 1 else None, self.groups, 0, 0, 0)

    def forward(self, x: DeviceArray, ids: DeviceArray, rows: int, stream: Stream | None = None) -> DeviceArray:
        """x: fp16 [rows][widths[0]], ids: uint32 [rows], the group of each row.
        Returns the fp32 outputs, the network's own array; keeps what backward() needs
        (x is read again there)."""
        if not 0 <= rows <= self.max_rows:
            raise ValueError(f"{rows} rows: the network was made for at most {self.max_rows}")
        _check_rows(x, rows, self.widths[0], "x")
        if ids.dtype != np.uint32 or int(np.prod(ids.shape, dtype=np.int64)) < rows:
            raise ValueError(f"ids are {ids.dtype} {ids.shape}: {rows} uint32 are needed")
        self._rows, self._input = None, x
        group_rows(ids.ptr, rows, self.groups, self.offsets.ptr, self.order.ptr, workspace=self.workspace, stream=stream)
        for l in range(self.layers):
            last = l == self.layers - 1
            d = L.NerfExtLinearDesc(rows, self.widths[l], self.widths[l + 1], L.NERF_EXT_F16, L.NERF_EXT_F32 if last else L.NERF_EXT_F16, L.NERF_EXT_ACT_NONE if last else self.act, 0, 0, 0, 0)
            src = (x if l == 0 else self._x[l]).ptr
            self._layer_forward(l, d, src, self.y.ptr if last else self._x[l + 1].ptr, src if self.residual[l] else None, None if last else self._z[l].ptr, stream)
        self._rows = rows
        return self.y

    def backward(self, delta: DeviceArray, rows: int, stream: Stream | None = None) -> None:
        """delta: fp16 [rows][widths[-1]], the loss' derivative in the outputs of the
        last forward() times the loss scale; rows: that forward()'s.  Fills the
        gradients."""
        if rows != self._rows:
            raise ValueError(f"{rows} rows: " + ("no forward pass" if self._rows is None else f"the last forward pass had {self._rows}"))
        _check_rows(delta, rows, self.widths[-1], "delta")
        g = delta
        for l in reversed(range(self.layers)):
            d = L.NerfExtLinearDesc(rows, self.widths[l], self.widths[l + 1], L.NERF_EXT_F16, L.NERF_EXT_F16, self.act, 0, 0, 0, 0)
            below = l > 0
            dx = self._g[l % 2] if below and self.residual[l - 1] else None
            dpre = self._delta[l % 2] if below else None
            self._layer_backward(l, d, (self._input if l == 0 else self._x[l]).ptr, delta.ptr, self._z[l - 1].ptr if below else None, g.ptr if below and self.residual[l] else None, dx.ptr if dx else None, dpre.ptr if dpre else None, stream)
            delta, g = dpre, dx


class GroupedNetwork(_GroupedLayers):
    """A network of its own for every group of rows (a region of a scene), all of one
    shape: hidden layers act(x W_g^T + b_g), plus x where a hidden layer behind the
    first is as wide as its input, then a linear layer with fp32 outputs.  Rows whose
    id is no group's keep what y held for them."""

    def __init__(self, widths: list[int], groups: int, activation: str = "relu", seed: int = 0, max_rows: int = 1 << 16):
        super().__init__(widths, activation, groups, max_rows)
        rng = np.random.default_rng(seed)
        tensors = []
        for i, o in zip(widths, widths[1:]):
            bound = np.sqrt(6.0 / (i + o))
            tensors += [rng.uniform(-bound, bound, (groups, o, i)), np.zeros((groups, o))]
        self._allocate(tensors)

    def _layer_forward(self, l, desc, x, y, residual, pre, stream):
        grouped_linear_forward(desc, self._groups_of(l), x, self.copies.ptr + 2 * self._at[2 * l], y, bias=self.params.ptr + 4 * self._at[2 * l + 1], residual=residual, pre=pre, workspace=self.workspace, stream=stream)

    def _layer_backward(self, l, desc, x, delta, pre, add, dx, dpre, stream):
        grouped_linear_backward(desc, self._groups_of(l), x, self.copies.ptr + 2 * self._at[2 * l] if dpre else None, delta, pre=pre, add=add, dx=dx, dpre=dpre, dweight=self.grads.ptr + 4 * self._at[2 * l],
                                dbias=self.grads.ptr + 4 * self._at[2 * l + 1], workspace=self.workspace, stream=stream)


class Adapters(_GroupedLayers):
    """A low-rank correction of a Network's layers for every group of rows (a scene or
    view that shares the network): W + scale up_g down_g, up zero at first.  The
    network's weights are held; rows whose id is no group's go through them alone.
    All arrays are in the rows' own order."""

    def __init__(self, network: Network, groups: int, rank: int = 16, scale: float = 1.0, seed: int = 0, max_rows: int | None = None):
        names = {v: k for k, v in ACTIVATIONS.items()}
        super().__init__(network.widths, names[network.act], groups, network.max_rows if max_rows is None else max_rows)
        if not 1 <= rank <= L.NERF_EXT_MAX_RANK:
            raise ValueError(f"rank {rank}: 1 to {L.NERF_EXT_MAX_RANK} are possible")
        self.network, self.rank, self.residual = network, int(rank), network.residual
        rng = np.random.default_rng(seed)
        tensors = []
        for i, o in zip(self.widths, self.widths[1:]):
            tensors += [rng.normal(0, i**-0.5, (groups, rank, i)), np.zeros((groups, o, rank))]
        self._allocate(tensors)
        self.scales = DeviceArray.from_numpy(np.full(groups, scale, np.float32))
        self._mid = [DeviceArray.zeros((self.max_rows, rank), np.float32) for _ in range(self.layers)]
        self._dmid = DeviceArray.zeros((self.max_rows, rank), np.float32)

    def _groups_of(self, l: int) -> L.NerfExtRowGroups:
        return L.NerfExtRowGroups(self.offsets.ptr, self.order.ptr, self.order.ptr, self.groups, 0, 0, 0)

    def _of_layer(self, l):
        return L.NerfExtAdapters(self.copies.ptr + 2 * self._at[2 * l], self.copies.ptr + 2 * self._at[2 * l + 1], self.scales.ptr, self.rank, 0)

    def _layer_forward(self, l, desc, x, y, residual, pre, stream):
        n = self.network
        adapter_linear_forward(desc, self._groups_of(l), self._of_layer(l), x, n.copies.ptr + 2 * n._at[2 * l], y, self._mid[l].ptr, bias=n.params.ptr + 4 * n._at[2 * l + 1], residual=residual, pre=pre, workspace=self.workspace, stream=stream)

    def _layer_backward(self, l, desc, x, delta, pre, add, dx, dpre, stream):
        n = self.network
        adapter_linear_backward(desc, self._groups_of(l), self._of_layer(l), x, n.copies.ptr + 2 * n._at[2 * l] if dpre else None, delta, mid=self._mid[l].ptr, pre=pre, add=add, dx=dx, dpre=dpre, dmid=self._dmid.ptr,
                                ddown=self.grads.ptr + 4 * self._at[2 * l], dup=self.grads.ptr + 4 * self._at[2 * l + 1], workspace=self.workspace, stream=stream)
