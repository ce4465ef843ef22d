"""Layers with adapters whose rows are streamed past the weights: every number of
steps of k and of blocks of ranks, forward and backward, and so many groups that the
same layer takes tiles.  On whole numbers, whose sums are exact in 32 bits."""
import pytest

import grouped_cases as G
from conftest import announce
from test_gpu_grouped import INDEXES, backward_equal, forward_equal, workspace  # noqa: F401

pytestmark = pytest.mark.gpu


# With 5 groups streamed, with 3000 by tiles.
@pytest.mark.parametrize("groups", [5, 3000])
@pytest.mark.parametrize("rank", [13, 32, 50])
@pytest.mark.parametrize("wide", [64, 128])
@pytest.mark.parametrize("kind,index", [("f16", 1), ("bf16", 0)])
def test_streamed_layers(workspace, wide, rank, groups, kind, index):  # noqa: F811
    announce(f"66000 x {wide} -> {wide}, {groups} groups, rank {rank}, {kind}")
    c = G.Case(66000, groups, wide, wide, kind, seed=wide + rank, rank=rank, whole=True, **INDEXES[index])
    forward_equal(c, "relu", "f32" if kind == "bf16" else kind, workspace)
    backward_equal(c, "relu", workspace)


# Streamed from 196608 rows and 98304 (gradients) on where the rank is above 48.
@pytest.mark.parametrize("n,rank,kind,index", [(66000, 32, "f16", 1), (66000, 32, "bf16", 0), (200000, 49, "f16", 0), (200000, 64, "bf16", 1), (100500, 56, "f16", 1), (66000, 33, "bf16", 1)])
def test_streamed_wide_layers(workspace, n, rank, kind, index):  # noqa: F811
    announce(f"{n} x 256 -> 256, 4 groups, rank {rank}, {kind}")
    c = G.Case(n, 4, 256, 256, kind, seed=rank, rank=rank, whole=True, **INDEXES[index])
    forward_equal(c, "relu", "f32" if kind == "bf16" else kind, workspace)
    backward_equal(c, "relu", workspace)


# Rows of odd length in tiles of 128, which few products do not take; the same in
# groups of fewer rows, and so many groups of whole chunks that most tiles are empty.
@pytest.mark.parametrize("n,groups,i,o", [(17000, 5, 1021, 1001), (17000, 200, 1021, 1001), (9000, 3000, 96, 136), (70000, 1000, 264, 128)])
@pytest.mark.parametrize("kind,index", [("f16", 1), ("bf16", 0)])
def test_grouped_tiles_by_rows_and_groups(workspace, n, groups, i, o, kind, index):  # noqa: F811
    announce(f"grouped {n} x {i} -> {o}, {groups} groups, {kind}")
    c = G.Case(n, groups, i, o, kind, seed=n, whole=True, **INDEXES[index])
    forward_equal(c, "relu", "f32" if kind == "bf16" else kind, workspace)
    backward_equal(c, "relu", workspace)
