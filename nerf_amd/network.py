"""A host's own network next to the fields of the library: a stack of linear
layers with residual connections, its gradients and its Adam step, all on the
device through nerf_ext_linear_*, nerf_ext_grad_norm and nerf_ext_adam_step.

    net = Network([63, 256, 256, 256, 4], activation="relu")
    y = net.forward(features, rows)            # fp32 [rows][4]
    net.backward(delta, rows)                  # delta fp16 [rows][4] = loss_scale d loss / d y
    net.step(hyper)                            # clip, skip guard and Adam
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


def _check_rows(array: DeviceArray, rows: int, width: int, what: str) -> None:
    """Rows of `width` 16-bit values, `rows` of them at least: an array of rows of
    any inner shape, or a flat one."""
    if array.dtype not in (np.float16, np.uint16):
        raise ValueError(f"{what} is {array.dtype}: it must be float16, or its bits as uint16")
    size = int(np.prod(array.shape, dtype=np.int64))
    fits = size >= rows * width if len(array.shape) == 1 else array.shape[0] >= rows and size == array.shape[0] * width
    if not fits:
        raise ValueError(f"{what} has shape {array.shape}: {rows} rows of {width} values are needed")


class Network:
    """Layers widths[0] -> ... -> widths[-1]: hidden layers act(x W^T + b), plus
    x where a layer is as wide as its input, then a linear layer with fp32
    outputs.  fp32 masters, fp16 working copies of the weights."""

    def __init__(self, widths: list[int], activation: str = "relu", seed: int = 0, max_rows: int = 1 << 16):
        if len(widths) < 2 or min(widths) < 1:
            raise ValueError("a network has an input and an output width, all positive")
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}")
        self.widths, self.max_rows, self.steps_done = list(widths), int(max_rows), 0
        self.act = ACTIVATIONS[activation]
        self._rows, self._input = None, None  # of the last forward pass
        self.layers = len(widths) - 1
        self.residual = [l < self.layers - 1 and widths[l] == widths[l + 1] for l in range(self.layers)]
        sizes, self._at, at = [], [], 0
        for i, o in zip(widths, widths[1:]):
            sizes += [o * i, o]
        for n in sizes:
            self._at.append(at)
            at += -(-n // ALIGN) * ALIGN
        self._sizes = sizes
        rng = np.random.default_rng(seed)
        host = np.zeros(at, np.float32)
        for l, (i, o) in enumerate(zip(widths, widths[1:])):
            bound = np.sqrt(6.0 / (i + o))
            host[self._at[2 * l] : self._at[2 * l] + o * i] = rng.uniform(-bound, bound, o * i)
        self.params = DeviceArray.from_numpy(host)
        self.copies = DeviceArray.from_numpy(host.astype(np.float16))
        self.grads, self.m, self.v = (DeviceArray.zeros((at,), np.float32) for _ in range(3))
        self.norm = DeviceArray.zeros((1,), np.float32)
        self.skipped = DeviceArray.zeros((1,), np.uint32)
        self.workspace = DeviceArray((L.NERF_EXT_LINEAR_WORKSPACE,), np.uint8)
        wide = max(widths[1:-1], default=0)
        # Inputs of every layer but the first, z of every hidden layer, and two deltas
        # and gradients in turn for the way back.
        self._x = [None] + [DeviceArray((self.max_rows, w), np.float16) for w in widths[1:-1]]
        self._z = [DeviceArray((self.max_rows, w), np.float16) for w in widths[1:-1]]
        self._delta, self._g = ([DeviceArray((self.max_rows, max(wide, 1)), np.float16) for _ in range(2)] for _ in range(2))
        self.y = DeviceArray((self.max_rows, widths[-1]), np.float32)
        n = len(sizes)
        self._grad_list = (L.NerfExtGradTensor * n)(*[L.NerfExtGradTensor(self.grads.ptr + 4 * a, None, s, L.NERF_EXT_F32, 0) for a, s in zip(self._at, sizes)])
        self._adam_list = (L.NerfExtAdamTensor * n)(
            *[L.NerfExtAdamTensor(self.params.ptr + 4 * a, self.grads.ptr + 4 * a, self.m.ptr + 4 * a, self.v.ptr + 4 * a, self.copies.ptr + 2 * a, s, L.NERF_EXT_F16, 0) for a, s in zip(self._at, sizes)])

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

    def step(self, hyper: L.NerfHyperParams, stream: Stream | None = None) -> None:
        """Norm of all gradients, then the update of all parameters (clipping and
        skip guard included)."""
        handle = stream.handle if stream else None
        L.call("nerf_ext_grad_norm", self._grad_list, len(self._grad_list), self.norm.ptr, self.workspace.ptr, self.workspace.nbytes, handle)
        L.call("nerf_ext_adam_step", self._adam_list, len(self._adam_list), C.byref(hyper), self.steps_done + 1, self.norm.ptr, self.skipped.ptr, handle)
        self.steps_done += 1
