"""The 64-bit definitions of grouped layers and adapters that the GPU tests compare
with, against central differences through an activation: dpre is the loss' derivative
in what the layer's inputs are the activations of."""
import numpy as np
import pytest

import grouped_cases as G
from linear_cases import act

H = 2.0**-9


@pytest.mark.parametrize("name", ["softplus", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("rank", [0, 3])
def test_gradients_through_an_activation(name, rank):
    """loss = sum(delta y) with y = W act(pre) + b: dpre, dx, and the sums over rows at
    x = act(pre).  The activations' third derivatives are at most 2, so a difference is
    off by H^2 / 6 of twice the sum of what multiplies them, below 2^-16 of 1 plus the
    gradient's terms here; rounding leaves 2^-50 / H."""
    c = G.Case(12, 3, 5, 4, "f16", seed=1, rank=rank, gather=True, scatter=True, extra=3)
    c.residual = np.zeros_like(c.residual)
    c.x = act(c.pre, name)
    mid = G.forward(c, "none", "f32")["mid"][0] if rank else None
    got = G.backward(c, name, add=False, mid=mid)

    def loss():
        c.x = act(c.pre, name)
        return (G.forward(c, "none", "f32")["y"][0] * c.delta).sum()

    rows = c.xr() if rank else c.xr()[c.offsets[0] : c.offsets[-1]]
    checks = [("dpre", c.pre, rows)] + ([("ddown", c.down, None), ("dup", c.up, None)] if rank else [("dw", c.w, None), ("db", c.bias, None)])
    rng = np.random.default_rng(2)
    for key, array, only in checks:
        flat, want = array.reshape(-1), got[key][0].reshape(-1)
        places = np.arange(array.size) if only is None else (only[:, None] * array.shape[1] + np.arange(array.shape[1])).reshape(-1)
        for at in rng.choice(places, min(25, len(places)), replace=False):
            old = flat[at]
            flat[at] = old + H
            up = loss()
            flat[at] = old - H
            down = loss()
            flat[at] = old
            assert abs((up - down) / (2 * H) - want[at]) <= 2.0**-16 * (1 + abs(want[at])), (key, at)
    assert np.abs(got["dpre"][0] - got["dx"][0])[rows].max() > 0.01  # the derivative takes part
