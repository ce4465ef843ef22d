"""What Network refuses before it calls the library: arrays too small or of
another type or width, and a way back that no way forward leads to.  Device
arrays and the library's calls are stand-ins here, so no GPU is needed."""
import numpy as np
import pytest

from nerf_amd import network


class HostArray:
    """A DeviceArray's shape and type, with an address that is never followed."""

    def __init__(self, shape, dtype=np.float32):
        self.shape = tuple(shape)
        self.dtype = np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
        self.ptr = 1 << 20

    @classmethod
    def from_numpy(cls, a):
        return cls(a.shape, a.dtype)

    zeros = classmethod(lambda cls, shape, dtype=np.float32: cls(shape, dtype))


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(network, "DeviceArray", HostArray)
    monkeypatch.setattr(network.L, "call", lambda name, *args: made.append(name))
    return made


def _net():
    return network.Network([6, 8, 8, 3], max_rows=16)


@pytest.mark.parametrize("shape,dtype", [((9, 6), np.float16), ((10, 5), np.float16), ((10, 7), np.float16), ((10, 6), np.float32), ((10, 6), np.uint8), ((10, 6), np.int16), ((59,), np.float16), ((6, 10), np.float16), ((2, 5, 3), np.float16)])
def test_inputs_that_do_not_fit(calls, shape, dtype):
    net = _net()
    with pytest.raises(ValueError):
        net.forward(HostArray(shape, dtype), 10)
    assert not calls


@pytest.mark.parametrize("shape,dtype", [((9, 3), np.float16), ((10, 4), np.float16), ((10, 2), np.float16), ((10, 3), np.float32), ((29,), np.float16)])
def test_deltas_that_do_not_fit(calls, shape, dtype):
    net = _net()
    net.forward(HostArray((10, 6), np.float16), 10)
    del calls[:]
    with pytest.raises(ValueError):
        net.backward(HostArray(shape, dtype), 10)
    assert not calls


@pytest.mark.parametrize("x,delta", [(((10, 6), np.float16), ((10, 3), np.float16)), (((16, 6), np.uint16), ((12, 3), np.uint16)), (((60,), np.float16), ((40,), np.float16)), (((10, 2, 3), np.float16), ((10, 3, 1), np.float16))])
def test_arrays_that_fit(calls, x, delta):
    """Whole or with rows to spare, numbers or their bits, rows of any inner shape."""
    net = _net()
    net.forward(HostArray(*x), 10)
    net.backward(HostArray(*delta), 10)
    assert calls == ["nerf_ext_linear_forward"] * 3 + ["nerf_ext_linear_backward"] * 3


def test_backward_follows_its_forward(calls):
    delta = HostArray((16, 3), np.float16)
    net = _net()
    with pytest.raises(ValueError):
        net.backward(delta, 10)
    net.forward(HostArray((16, 6), np.float16), 10)
    for rows in (9, 11, 16, 0):
        with pytest.raises(ValueError):
            net.backward(delta, rows)
    with pytest.raises(ValueError):
        net.forward(HostArray((16, 6), np.float32), 12)  # refused: what the last forward kept stays
    del calls[:]
    net.backward(delta, 10)
    net.backward(delta, 10)
    assert calls == ["nerf_ext_linear_backward"] * 6


def test_a_forward_that_failed_has_no_backward(calls, monkeypatch):
    net, delta = _net(), HostArray((16, 3), np.float16)
    net.forward(HostArray((16, 6), np.float16), 10)

    def fails(name, *args):
        raise network.L.NerfError(name, network.L.NERF_STATUS_INVALID_USAGE, "no")

    with monkeypatch.context() as m:
        m.setattr(network.L, "call", fails)
        with pytest.raises(network.L.NerfError):
            net.forward(HostArray((16, 6), np.float16), 10)
    with pytest.raises(ValueError):
        net.backward(delta, 10)
