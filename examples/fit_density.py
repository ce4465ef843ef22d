"""Fits a residual network of the user's own to the density of an analytic scene:
63 frequency-encoded coordinates -> 256 -> 256 -> 256 -> 1.

    python examples/fit_density.py [steps]
"""
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from nerf_amd import _lib as L, ext  # noqa: E402
from nerf_amd.device import DeviceArray, synchronize  # noqa: E402
from nerf_amd.network import Network  # noqa: E402

ROWS, LOSS_SCALE = 8192, 128.0


def encode(p: np.ndarray) -> np.ndarray:
    """x, then sin and cos of 2^k pi x, k = 0..9: 63 features."""
    a = (p[:, None, :] * (np.pi * 2.0 ** np.arange(10))[None, :, None]).reshape(len(p), 30)
    return np.concatenate([p, np.sin(a), np.cos(a)], 1).astype(np.float16)


def fit(steps: int = 200, seed: int = 0) -> list[float]:
    """The mean squared error of the scaled density at each step's points."""
    rng = np.random.default_rng(seed)
    gaussians = DeviceArray.from_numpy(ext.scene_gaussians(8, seed=3))
    net = Network([63, 256, 256, 256, 1], seed=seed, max_rows=ROWS)
    hyper = ext.hyper_params(lr=2e-3, eps=1e-8, clip=1.0, guard=1e4, loss_scale=LOSS_SCALE)
    density, x, delta = DeviceArray((ROWS,), np.float32), DeviceArray((ROWS, 63), np.float16), DeviceArray((ROWS, 1), np.float16)
    losses = []
    for _ in range(steps):
        p = rng.random((ROWS, 3), np.float32)
        points = DeviceArray.from_numpy(p)
        L.call("nerf_ext_scene_density", gaussians.ptr, 8, points.ptr, ROWS, density.ptr, None)
        x.upload(encode(p))
        y = net.forward(x, ROWS).numpy()[:, 0]
        error = y - density.numpy() / 10.0
        losses.append(float((error * error).mean()))
        delta.upload((LOSS_SCALE * 2.0 / ROWS * error)[:, None].astype(np.float16))
        net.backward(delta, ROWS)
        net.step(hyper)
    synchronize()
    return losses


if __name__ == "__main__":
    history = fit(int(sys.argv[1]) if len(sys.argv) > 1 else 200)
    for i in range(0, len(history), max(1, len(history) // 10)):
        print(f"step {i}: mean squared error {history[i]:.5f}")
    print(f"last: {history[-1]:.5f}")
