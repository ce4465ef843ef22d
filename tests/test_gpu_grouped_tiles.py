"""Grouped layers and adapters at sizes that reach each tile of their kernels
on a GPU of 256 CUs: few outputs with a tile's k over a workgroup's waves (16 and
32 wide, whole steps and not), tiles of 128 and 256, sums in tiles of 256.  On
whole numbers, whose sums are exact in 32 bits in any order."""
import numpy as np
import pytest

import grouped_cases as G
from linear_exact import equal
from test_gpu_grouped import INDEXES, backward_equal, forward_equal, run_backward, workspace  # noqa: F401

pytestmark = pytest.mark.gpu

# rows, groups, in, out, and the adapters' rank.
TILES = [(300, 2, 256, 256, 16), (300, 2, 250, 250, 7), (1000, 4, 256, 256, 8), (1000, 4, 250, 252, 33), (2000, 6, 256, 64, 64), (700, 40, 1024, 96, 256), (40000, 3, 515, 301, 12), (40000, 3, 514, 302, 20), (20000, 3, 520, 520, 16), (16301, 3, 1024, 1024, 24), (16300, 60, 1024, 1024, 7)]


@pytest.mark.parametrize("rank", [False, True])
@pytest.mark.parametrize("n,groups,i,o,r", TILES)
@pytest.mark.parametrize("kind,index", [("f16", 1), ("bf16", 0)])
def test_tiles(workspace, n, groups, i, o, r, rank, kind, index):  # noqa: F811
    print(f"[case] {n} x {i} -> {o}, {groups} groups, rank {r if rank else 0}, {kind}, {INDEXES[index]}", flush=True)
    c = G.Case(n, groups, i, o, kind, seed=n + i, rank=r if rank else 0, whole=True, **INDEXES[index])
    forward_equal(c, "relu", "f32" if kind == "bf16" else kind, workspace)
    backward_equal(c, "relu", workspace)


@pytest.mark.parametrize("kind,index", [("f16", 1), ("bf16", 0)])
def test_widest_sums(workspace, kind, index):  # noqa: F811
    print(f"[case] sums over 33000 rows of 2048 x 2056, 2 groups, {kind}, {INDEXES[index]}", flush=True)
    c = G.Case(33000, 2, 2048, 2056, kind, seed=5, whole=True, **INDEXES[index])
    got = run_backward(c, "relu", workspace, dx=False, dpre=False)
    d, x = c.delta[c.yr()].astype(np.float32), c.x[c.xr()].astype(np.float32)
    for g, (a, b) in enumerate(zip(c.offsets, c.offsets[1:])):
        equal(got["dw"][g], (d[a:b].T @ x[a:b]).astype(np.float64), f"dw {g}")
        equal(got["db"][g], d[a:b].sum(0).astype(np.float64), f"db {g}")
