"""Rows in groups, grouped layers, adapters, the gradient norm and the Adam step
used together: networks of many regions and of many scenes against their
definitions in 64 bits, their training, and the same work recorded in graphs."""
import ctypes as C

import numpy as np
import pytest

from conftest import announce
from linear_cases import act, decode, encode, slope
from nerf_amd import ext
from nerf_amd.device import DeviceArray, Stream, synchronize
from nerf_amd.network import Adapters, GroupedNetwork, Network

pytestmark = pytest.mark.gpu


def _f16(a):
    return decode(encode(a, "f16"), "f16")


def _device(a):
    return DeviceArray.from_numpy(encode(a, "f16").view(np.float16))


def _copies(net, index):
    return decode(net.tensor(index, "copies").view(np.uint16), "f16")


def layers_of(net, g):
    """(weight, bias, down, up, scale) of every layer for rows of group g (None: in none)."""
    out = []
    for l in range(net.layers):
        if isinstance(net, GroupedNetwork):
            out.append((_copies(net, 2 * l)[g], net.tensor(2 * l + 1)[g].astype(np.float64), None, None, 0.0))
        else:
            n = net.network
            down, up = (None, None) if g is None else (_copies(net, 2 * l)[g], _copies(net, 2 * l + 1)[g])
            out.append((decode(n.weight(l, "copies").view(np.uint16), "f16"), n.bias(l).astype(np.float64), down, up, 0.0 if g is None else float(net.scales.numpy()[g])))
    return out


def definition(net, x, delta, g, name):
    """Outputs, and gradients of the group's tensors, with activations and deltas
    rounded to fp16 where the network keeps them."""
    layers = layers_of(net, g)
    xs, zs, mids = [x], [], []
    for l, (w, b, down, up, scale) in enumerate(layers):
        z = xs[-1] @ w.T + b
        mids.append(None if down is None else xs[-1] @ down.T)
        if down is not None:
            z = z + scale * (mids[-1] @ up.T)
        if l == net.layers - 1:
            y = z
            break
        zs.append(_f16(z))
        xs.append(_f16(act(z, name) + (xs[-1] if net.residual[l] else 0.0)))
    grads, gx = {}, None
    for l in reversed(range(net.layers)):
        w, _, down, up, scale = layers[l]
        dx = delta @ w
        if isinstance(net, GroupedNetwork):
            grads[2 * l], grads[2 * l + 1] = delta.T @ xs[l], delta.sum(0)
        elif down is not None:
            dmid = scale * (delta @ up)
            grads[2 * l], grads[2 * l + 1] = dmid.T @ xs[l], scale * (delta.T @ mids[l])
            dx = dx + dmid @ down
        if l:
            dx = dx + (gx if net.residual[l] else 0.0)
            delta, gx = _f16(dx * slope(zs[l - 1], name)), _f16(dx)
    return y, grads


def _inputs(rows, widths, groups, seed):
    rng = np.random.default_rng(seed)
    return _f16(rng.normal(0, 1, (rows, widths[0]))), _f16(rng.normal(0, 0.1, (rows, widths[-1]))), rng.integers(0, groups + 1, rows).astype(np.uint32)


def _adapters(widths, groups, name, rows, rank):
    net = Adapters(Network(widths, name, seed=1, max_rows=1), groups, rank, scale=0.5, seed=2, max_rows=rows)
    rng = np.random.default_rng(3)
    for l in range(net.layers):  # as after some training
        a, n = net._at[2 * l + 1], net._sizes[2 * l + 1]
        up = rng.normal(0, 0.3 / rank**0.5, n).astype(np.float16)
        ext.write_device(net.copies.ptr + 2 * a, up)
    return net


CASES = [([63, 64, 64, 64, 4], 300, 5, "relu", 0), ([31, 40, 40, 24, 24, 3], 129, 40, "gelu", 0), ([8, 1], 5, 2, "relu", 0), ([63, 256, 256, 1], 20000, 9, "silu", 0), ([63, 64, 64, 64, 4], 300, 5, "relu", 16), ([24, 24, 24, 3], 129, 40, "gelu", 7), ([63, 256, 256, 1], 20000, 3, "silu", 16)]


@pytest.mark.parametrize("widths,rows,groups,name,rank", CASES)
def test_outputs_and_gradients(widths, rows, groups, name, rank):
    announce(f"{'adapters' if rank else 'grouped network'} {widths}, {rows} rows, {groups} groups")
    net = _adapters(widths, groups, name, rows, rank) if rank else GroupedNetwork(widths, groups, name, seed=1, max_rows=rows)
    x, delta, ids = _inputs(rows, widths, groups, 4)
    dx, dd, di = _device(x), _device(delta), DeviceArray.from_numpy(ids)
    y = net.forward(dx, di, rows).numpy()[:rows]
    net.backward(dd, rows)
    synchronize()

    # A value that lies within 32-bit rounding of the middle between two fp16
    # numbers may be kept as either, 2^-10 of it apart, and a relu's sign may
    # follow: rare, so the differences are small in the 2-norm.
    def close(got, ref):
        return np.linalg.norm(got - ref) <= 2e-3 * np.linalg.norm(ref)

    got = [net.tensor(i, "grads") for i in range(2 * net.layers)]
    for g in range(groups):
        at = np.nonzero(ids == g)[0]
        want, grads = definition(net, x[at], delta[at], g, name)
        assert close(y[at], want), g
        for i, ref in grads.items():
            assert close(got[i][g], ref), (g, i)
    at = np.nonzero(ids == groups)[0]
    if rank:
        assert close(y[at], definition(net, x[at], delta[at], None, name)[0])
    else:
        assert (y[at] == 0.0).all()


def test_new_adapters_are_the_network():
    net = Network([24, 32, 32, 5], "relu", seed=1, max_rows=200)
    x, _, ids = _inputs(200, net.widths, 3, 5)
    dx, di = _device(x), DeviceArray.from_numpy(ids)
    adapters = Adapters(net, 3, 4)
    a, b = adapters.forward(dx, di, 200).numpy(), net.forward(dx, 200).numpy()
    # Two kernels that sum in other orders: 32 terms of size 1 a layer, and an fp16
    # rounding that may fall to the other side.
    assert np.linalg.norm(a - b) <= 2e-3 * np.linalg.norm(b)


@pytest.mark.parametrize("rank", [0, 8])
def test_steps_follow_the_gradient(rank):
    """A small step against the gradient changes a linear loss by minus its square, to
    first order: the sums of the kernels, the norm and the update agree."""
    announce(f"steps, rank {rank}")
    widths, rows, groups = [16, 32, 3], 400, 4
    net = _adapters(widths, groups, "silu", rows, rank) if rank else GroupedNetwork(widths, groups, "silu", seed=1, max_rows=rows)
    x, delta, ids = _inputs(rows, widths, groups, 6)
    dx, dd, di = _device(x), _device(delta), DeviceArray.from_numpy(ids)
    y = net.forward(dx, di, rows).numpy().astype(np.float64)
    net.backward(dd, rows)
    before = net.params.numpy().copy()
    net.step(ext.hyper_params(lr=1e-3, eps=1e-8))
    synchronize()
    grads, moved = net.grads.numpy().astype(np.float64), net.params.numpy() - before
    assert abs(float(net.norm.numpy()[0]) - np.linalg.norm(grads)) <= 1e-5 * np.linalg.norm(grads)
    # The first step of Adam is lr times the gradient's sign.
    assert (np.sign(moved) == -np.sign(grads)).all() and np.abs(np.abs(moved[grads != 0]) - 1e-3).max() < 1e-5


def _replayed(net, rows, groups, seed):
    """Forward and backward in a graph, replayed between eager work on other inputs:
    the bits of the eager calls every time."""
    hip = C.CDLL("libamdhip64.so")
    stream, widths = Stream(), net.widths
    sets = [_inputs(rows, widths, groups, seed + k) for k in range(3)]
    host = [(encode(x, "f16").view(np.float16), encode(d, "f16").view(np.float16), i) for x, d, i in sets]
    x, d, ids = (DeviceArray.from_numpy(a) for a in host[0])

    def load(k):
        for a, h in zip((x, d, ids), host[k]):
            a.upload(h)

    def work():
        net.forward(x, ids, rows, stream)
        net.backward(d, rows, stream)

    def read():
        stream.synchronize()
        return net.y.numpy(), net.grads.numpy()

    want = []
    for k in range(3):
        load(k)
        net.y.fill_bytes(0)
        work()
        want.append(read())
    graph, run, handle = C.c_void_p(), C.c_void_p(), C.c_void_p(stream.handle)
    assert hip.hipStreamBeginCapture(handle, 1) == 0
    work()
    assert hip.hipStreamEndCapture(handle, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    try:
        for k in (1, 0, 2, 1):
            load(k)
            net.y.fill_bytes(0)
            net.grads.fill_bytes(0)
            assert hip.hipGraphLaunch(run, handle) == 0
            for got, ref in zip(read(), want[k]):
                assert np.array_equal(got, ref)
            load((k + 1) % 3)
            work()  # eager work in between
            stream.synchronize()
    finally:
        assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0


@pytest.mark.parametrize("rows", [3000, 70000])
@pytest.mark.parametrize("rank", [0, 16])
def test_recorded_work_is_the_eager_one(rank, rows):
    announce(f"recorded work, rank {rank}, {rows} rows")
    widths, groups = [63, 128, 128, 5], 6
    net = _adapters(widths, groups, "relu", rows, rank) if rank else GroupedNetwork(widths, groups, "relu", seed=5, max_rows=rows)
    _replayed(net, rows, groups, 7)


def test_two_streams_at_once():
    """Two networks on two streams, their work under way together: each as alone."""
    widths, groups, rows = [24, 64, 64, 3], 5, 9000
    nets = [GroupedNetwork(widths, groups, "relu", seed=1, max_rows=rows), _adapters(widths, groups, "relu", rows, 8)]
    streams = [Stream(), Stream()]
    x, delta, ids = _inputs(rows, widths, groups, 8)
    dx, dd, di = _device(x), _device(delta), DeviceArray.from_numpy(ids)
    want = []
    for n in nets:
        n.forward(dx, di, rows)
        n.backward(dd, rows)
        synchronize()
        want.append((n.y.numpy(), n.grads.numpy()))
    for _ in range(5):
        for n, s in zip(nets, streams):
            n.forward(dx, di, rows, s)
            n.backward(dd, rows, s)
    for n, s, w in zip(nets, streams, want):
        s.synchronize()
        assert np.array_equal(n.y.numpy(), w[0]) and np.array_equal(n.grads.numpy(), w[1])


def test_refusals():
    with pytest.raises(ValueError):
        GroupedNetwork([4], 2)
    with pytest.raises(ValueError):
        GroupedNetwork([4, 4], 0)
    with pytest.raises(ValueError):
        GroupedNetwork([4, 4], 4097)
    with pytest.raises(ValueError):
        GroupedNetwork([4, 4], 2, "tanh")
    net = GroupedNetwork([4, 4], 2, max_rows=8)
    x, ids = DeviceArray((9, 4), np.float16), DeviceArray.zeros((9,), np.uint32)
    for call in (lambda: net.forward(x, ids, 9), lambda: net.forward(DeviceArray((8, 5), np.float16), ids, 8), lambda: net.forward(x, DeviceArray.zeros((7,), np.uint32), 8), lambda: net.forward(x, DeviceArray.zeros((8,), np.float32), 8),
                 lambda: net.backward(x, 8)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        Adapters(Network([4, 4], max_rows=8), 2, 0)
    with pytest.raises(ValueError):
        Adapters(Network([4, 4], max_rows=8), 2, 257)
