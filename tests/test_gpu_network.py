"""The linear layer, its gradients, the gradient norm and the Adam step used
together: a residual network against its definition in 64 bits, its training,
and the same work recorded in a graph."""
import ctypes as C
import sys
from pathlib import Path

import numpy as np
import pytest

from linear_cases import act, decode, encode, slope
from nerf_amd import _lib as L, ext
from nerf_amd.device import DeviceArray, Stream, synchronize
from nerf_amd.network import Network

pytestmark = pytest.mark.gpu


def _f16(a):
    return decode(encode(a, "f16"), "f16")


def definition(net, x, delta, name):
    """Outputs and gradients in 64 bits, with activations and deltas rounded to
    fp16 where the network keeps them."""
    w = [decode(net.weight(l, "copies").view(np.uint16), "f16") for l in range(net.layers)]
    b = [net.bias(l).astype(np.float64) for l in range(net.layers)]
    xs, zs = [x], []
    for l in range(net.layers - 1):
        z = xs[-1] @ w[l].T + b[l]
        zs.append(_f16(z))
        xs.append(_f16(act(z, name) + (xs[-1] if net.residual[l] else 0.0)))
    y = xs[-1] @ w[-1].T + b[-1]
    grads, g = {}, None
    for l in reversed(range(net.layers)):
        grads[l] = (delta.T @ xs[l], delta.sum(0))
        if l:
            dx = delta @ w[l] + (g if net.residual[l] else 0.0)
            delta, g = _f16(dx * slope(zs[l - 1], name)), _f16(dx)
    return y, grads


@pytest.mark.parametrize("widths,rows,name", [([63, 64, 64, 64, 4], 300, "relu"), ([31, 40, 40, 24, 24, 3], 129, "gelu"), ([8, 1], 5, "relu"), ([63, 256, 256, 256, 1], 20000, "silu")])
def test_network_gradients(widths, rows, name):
    net = Network(widths, name, seed=1, max_rows=rows)
    rng = np.random.default_rng(2)
    x, delta = _f16(rng.normal(0, 1, (rows, widths[0]))), _f16(rng.normal(0, 0.1, (rows, widths[-1])))
    dx, dd = DeviceArray.from_numpy(encode(x, "f16").view(np.float16)), DeviceArray.from_numpy(encode(delta, "f16").view(np.float16))
    y = net.forward(dx, rows).numpy()[:rows]
    net.backward(dd, rows)
    synchronize()
    want, grads = definition(net, x, delta, name)

    # A value that lies within 32-bit rounding of the middle between two fp16
    # numbers may be kept as either, 2^-10 of it apart, and a relu's sign may
    # follow: rare, so the differences are small in the 2-norm.
    def close(got, ref):
        return np.linalg.norm(got - ref) <= 2e-3 * np.linalg.norm(ref)

    assert close(y, want)
    for l in range(net.layers):
        assert close(net.weight(l, "grads"), grads[l][0]), l
        assert close(net.bias(l, "grads"), grads[l][1]), l


def test_network_trains():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    from fit_density import fit

    losses = fit(150)
    assert np.isfinite(losses).all()
    assert np.mean(losses[-10:]) < 0.1 * np.mean(losses[:3]), losses[::15]


def test_refusals():
    with pytest.raises(ValueError):
        Network([4])
    with pytest.raises(ValueError):
        Network([4, 4], "tanh")
    net = Network([4, 4], max_rows=8)
    with pytest.raises(ValueError):
        net.forward(DeviceArray((9, 4), np.float16), 9)


def test_recorded_step_is_the_eager_one():
    """Forward, backward and norm in a graph, replayed between eager work on other
    inputs: the bits of the eager calls every time."""
    hip = C.CDLL("libamdhip64.so")
    rows, rng = 3000, np.random.default_rng(4)
    net = Network([63, 128, 128, 5], seed=5, max_rows=rows)
    stream = Stream()
    xs = [encode(rng.normal(0, 1, (rows, 63)), "f16").view(np.float16) for _ in range(3)]
    ds = [encode(rng.normal(0, 0.1, (rows, 5)), "f16").view(np.float16) for _ in range(3)]
    x, d = DeviceArray.from_numpy(xs[0]), DeviceArray.from_numpy(ds[0])
    hyper = ext.hyper_params()

    def work():
        net.forward(x, rows, stream)
        net.backward(d, rows, stream)
        L.call("nerf_ext_grad_norm", net._grad_list, len(net._grad_list), net.norm.ptr, net.workspace.ptr, net.workspace.nbytes, stream.handle)

    def read():
        stream.synchronize()
        return net.y.numpy(), net.grads.numpy(), net.norm.numpy()

    want = []
    for a, b in zip(xs, ds):
        x.upload(a)
        d.upload(b)
        work()
        want.append(read())
    graph, run = C.c_void_p(), C.c_void_p()
    handle = C.c_void_p(stream.handle)
    assert hip.hipStreamBeginCapture(handle, 1) == 0
    work()
    assert hip.hipStreamEndCapture(handle, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0)) == 0
    try:
        for i in (1, 0, 2, 1):
            x.upload(xs[i])
            d.upload(ds[i])
            net.grads.fill_bytes(0)
            assert hip.hipGraphLaunch(run, handle) == 0
            for got, ref in zip(read(), want[i]):
                assert np.array_equal(got, ref)
            x.upload(xs[(i + 1) % 3])
            work()  # eager work in between
            stream.synchronize()
    finally:
        assert hip.hipGraphExecDestroy(run) == 0 and hip.hipGraphDestroy(graph) == 0
    net.step(hyper)
    synchronize()
    assert np.isfinite(net.params.numpy()).all()
