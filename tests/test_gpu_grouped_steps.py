"""Networks of many groups: what a step changes their loss by, against the inner
product of the kernels' gradients and what the step moved."""
import numpy as np
import pytest

from conftest import announce
from linear_cases import decode, encode
from nerf_amd import ext
from nerf_amd.device import DeviceArray, synchronize
from nerf_amd.network import Adapters, GroupedNetwork, Network

pytestmark = pytest.mark.gpu


def _typed(a):
    return decode(encode(a, "f16"), "f16")


def _network(rank, name, widths, rows, groups, rng):
    if not rank:
        return GroupedNetwork(widths, groups, name, seed=1, max_rows=rows)
    net = Adapters(Network(widths, name, seed=1, max_rows=1), groups, rank, scale=0.5, seed=2, max_rows=rows)
    for l in range(net.layers):  # as after some training
        a, n = net._at[2 * l + 1], net._sizes[2 * l + 1]
        up = rng.normal(0, 0.3 / rank**0.5, n).astype(np.float32)
        ext.write_device(net.params.ptr + 4 * a, up)
        ext.write_device(net.copies.ptr + 2 * a, up.astype(np.float16))
    return net


@pytest.mark.parametrize("rank", [0, 8])
@pytest.mark.parametrize("name", ["softplus", "silu", "gelu"])
def test_a_step_changes_the_loss_by_the_gradient(rank, name):
    """loss = sum(y delta) before and after a step, its gradient g at both ends and the
    move s of what the forward pass multiplies by (working copies, fp32 biases).

    Bound.  change - s (g0 + g1) / 2 is a third derivative's share; with a curvature
    b = s (g1 - g0) it is of the size b^2 / (s g0).  The first step of Adam is against
    every gradient's sign, so all terms of s g0 have one sign, and the fp16 roundings of
    activations, pre-activations and deltas (2^-11 each, on the way there and back
    through two hidden layers, twice) leave 16 of them at most: 2^-7 of it."""
    announce(f"loss change of a step, rank {rank}, {name}")
    widths, rows, groups, rng = [16, 32, 32, 3], 400, 4, np.random.default_rng(6)
    net = _network(rank, name, widths, rows, groups, rng)
    x, delta = _typed(rng.normal(0, 1, (rows, widths[0]))), _typed(rng.normal(0, 0.1, (rows, widths[-1])))
    dx, dd = (DeviceArray.from_numpy(encode(a, "f16").view(np.float16)) for a in (x, delta))
    ids = DeviceArray.from_numpy(rng.integers(0, groups, rows).astype(np.uint32))

    def tensors(of_weights, of_biases):
        """One array of all tensors; every second one of a grouped network is a bias."""
        return np.concatenate([(of_biases if i % 2 and not rank else of_weights).numpy().astype(np.float64)[a : a + s] for i, (a, s) in enumerate(zip(net._at, net._sizes))])

    def forward_and_backward():
        loss = (net.forward(dx, ids, rows).numpy().astype(np.float64) * delta).sum()
        net.backward(dd, rows)
        synchronize()
        return loss, tensors(net.copies, net.params), tensors(net.grads, net.grads)

    loss0, at0, g0 = forward_and_backward()
    net.step(ext.hyper_params(lr=5e-4, eps=1e-8))
    loss1, at1, g1 = forward_and_backward()
    first, second = ((at1 - at0) * g0).sum(), ((at1 - at0) * g1).sum()
    assert first < 0.0 and abs(second - first) < 0.25 * abs(first), "a step that is too long to compare"
    assert abs(loss1 - loss0 - 0.5 * (first + second)) <= (second - first) ** 2 / abs(first) + 2.0**-7 * abs(first)
