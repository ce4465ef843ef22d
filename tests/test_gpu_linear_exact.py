"""The linear layer and its gradients on whole numbers, whose sums are exact in
32 bits in any order: outputs equal their definition, rounded once.  The shapes
reach every kernel that a call can reach on 256 CUs, with ragged edges: tiles
of 256, 128 and 64 of each product, their sums whole and split over k, whole
chunks, even and odd rows, rows streamed past the weights, few outputs, and
operands of a few values."""
import numpy as np
import pytest

import linear_exact
from conftest import announce
from linear_exact import equal, inputs
from nerf_amd import _lib as L
from test_gpu_linear import run_backward, run_forward

pytestmark = pytest.mark.gpu
KINDS = ("f16", "bf16")


def check_forward(n, i, o, kind, y_kind, act="relu", seed=0, most=2, bias=True, residual=True, pre=True, **kw):
    announce(f"exact forward n={n} in={i} out={o} {kind}->{y_kind} {act} {kw}")
    v = inputs(n, i, o, seed, most)
    y, z = run_forward(v, kind, y_kind, act, bias=bias, residual=residual, pre=pre, **kw)
    want_y, want_z = linear_exact.forward(v, act, kind, y_kind, bias, residual)
    equal(y, want_y, "y")
    if pre:
        equal(z, want_z, "pre")


def check_backward(n, i, o, kind, act="relu", seed=0, most=2, add=True, **kw):
    announce(f"exact backward n={n} in={i} out={o} {kind} {act} {kw}")
    v = inputs(n, i, o, seed, most)
    got = run_backward(v, kind, act, add=add, **kw)
    want = linear_exact.backward(v, act, kind, add)
    for k, value in got.items():
        equal(value.reshape(want[k].shape), want[k], k)


# Tiles of 256: at least as many as CUs, 512 k and more; an odd and an even number
# of steps of 64 k, the last of them cut.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,k,p", [(4099, 520, 4088), (4099, 1000, 4088), (8200, 584, 2056), (65544, 576, 136)])
def test_largest_tiles(n, k, p, kind):
    check_forward(n, k, p, kind, kind)
    check_forward(n, k, p, kind, "f32", "none", bias=False, residual=False, pre=False)
    check_backward(n, p, k, kind, dw=False, db=False)


@pytest.mark.parametrize("kind", KINDS)
def test_largest_tiles_in_bands_with_strides(kind):
    """More than four tiles across, and a last band of fewer than four; columns of
    wider arrays."""
    check_forward(1288, 520, 12296, kind, kind, strides=(528, 12304, 12312))
    check_backward(1288, 12296, 520, kind, strides=(12304, 528), dw=False, db=False)


# Weight gradients by tiles of 256 (from 2^35 products on): ten parts, three
# parts, whole.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,i,o", [(33001, 1032, 1040), (8205, 2040, 2056), (4105, 4088, 2056)])
def test_largest_tiles_of_weight_gradients(n, i, o, kind):
    check_backward(n, i, o, kind, dx=False, dpre=False)


# Tiles of 128: whole chunks, rows of even length, of odd length.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,k,p", [(3001, 520, 1208), (2050, 264, 2056), (3001, 518, 1210), (3001, 517, 1207), (3001, 521, 1210)])
def test_middle_tiles(n, k, p, kind):
    check_forward(n, k, p, kind, kind)
    check_backward(n, p, k, kind, dw=False, db=False)


# Weight gradients by tiles of 128 (from 2^32 products on): split in 32, in 6, whole.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,i,o", [(20011, 480, 488), (20011, 476, 492), (20011, 475, 491), (5001, 1032, 1048), (5001, 1030, 1050), (5001, 1031, 1049), (530, 4088, 2056), (530, 4084, 2058), (530, 4083, 2057)])
def test_middle_tiles_of_weight_gradients(n, i, o, kind):
    check_backward(n, i, o, kind, dx=False, dpre=False)


# Tiles of 64: whole and split, each way of reading.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,k,p", [(1000, 264, 520), (1000, 262, 522), (1000, 261, 521), (700, 1104, 520), (700, 1102, 522), (300, 4104, 264), (300, 4102, 262), (300, 4101, 261), (70, 8200, 520)])
def test_smallest_tiles(n, k, p, kind):
    check_forward(n, k, p, kind, kind)
    check_forward(n, k, p, kind, "f32", "none", residual=False)


# Input gradients by tiles of 64, the sums over outputs whole and split; weight
# gradients of a head of a few outputs.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,i,o", [(300, 96, 8200), (300, 98, 8202), (300, 97, 8201), (5000, 40, 1104), (5000, 42, 1102), (5000, 41, 1101), (9001, 256, 4), (9001, 255, 4), (9001, 63, 5), (9001, 62, 6), (2100, 1032, 1032), (2100, 1030, 1034), (2100, 1031, 1033)])
def test_smallest_tiles_of_gradients(n, i, o, kind):
    check_backward(n, i, o, kind)
    check_backward(n, i, o, kind, "none", dw=False, db=False, add=False, dx=False)


# Split sums: no workspace, one that holds a part less than is worth a split, the
# least that is, a few parts, all.
@pytest.mark.parametrize("parts", [0, 1, 3, 4, 7, 1000])
@pytest.mark.parametrize("kind", KINDS)
def test_workspaces(kind, parts):
    def size(part, least=0):
        return min(L.NERF_EXT_LINEAR_WORKSPACE, max(0, 4 * (part * parts + least)))

    for n, k, p in ((300, 4104, 264), (70, 8201, 57), (64, 8192, 64)):
        check_forward(n, k, p, kind, kind, workspace=size(n * p))
        check_backward(n, p, k, kind, workspace=size(n * p), dw=False, db=False)
    for n, i, o in ((20011, 40, 24), (9001, 255, 4), (20011, 475, 491), (33001, 1032, 1040)):
        # The first part of a weight gradient lies in its place, the others and all
        # parts of the bias gradient in the workspace; then four bytes less.
        for less in (0, 1):
            check_backward(n, i, o, kind, workspace=size(i * o + o, -i * o - less) & ~3, dx=False, dpre=False)
    check_backward(20011, 40, 24, kind, workspace=size(40 * 24), dx=False, dpre=False, db=False)


# Rows streamed past the weights: 1, 2, 4 and 8 steps of 32 k; whole, cut and odd
# rows; one to four waves across, narrow outputs, more than 256 of them.
STREAMED = [(16400, 32, 72), (16399, 24, 40), (16390, 31, 33), (16385, 1, 8), (32770, 64, 264), (32771, 57, 24), (32770, 58, 130), (65541, 128, 72), (65543, 96, 32), (65537, 128, 520), (131077, 256, 136), (131075, 224, 24), (131073, 160, 296),
            (16400, 32, 24), (16399, 30, 32), (16390, 8, 5), (16400, 28, 100), (32770, 64, 32), (32772, 58, 24), (32771, 57, 72), (32769, 33, 256)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,k,p", STREAMED)
def test_streamed_rows(n, k, p, kind):
    check_forward(n, k, p, kind, kind if p % 16 else "f32")
    check_backward(n, p, k, kind, dw=False, db=False)


def test_more_rows_than_one_launch():
    check_forward(65535 * 64 + 100, 9, 2, "f16", "f16", most=1)
    check_backward(65535 * 64 + 100, 2, 9, "bf16", most=1)


# Operands of a few values, and one and few outputs around the smallest tiles.
@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 9])
def test_few_values(n):
    for i in (1, 2, 3, 7, 8, 9, 17):
        for o in (1, 2, 5, 8, 9):
            check_forward(n, i, o, "f16", "f16")
            check_backward(n, i, o, "bf16")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,i,o", [(1, 256, 256), (1, 4096, 1000), (15, 33, 31), (16, 1601, 999), (33, 512, 513), (100, 788, 64), (129, 1023, 65), (353, 1115, 705), (500, 64, 520), (1024, 96, 130), (2048, 256, 256), (2047, 255, 257), (1, 4097, 5), (1, 1, 4096)])
def test_few_outputs(n, i, o, kind):
    check_forward(n, i, o, kind, kind)
    check_backward(n, i, o, kind)


# The strides and starts that choose how rows are read, around each kind of tile.
@pytest.mark.parametrize("strides,shift", [((536, 1216, 1224), 8), ((522, 1210, 1212), 2), ((521, 1209, 1211), 1), ((520, 1208, 1208), 3)])
def test_strides_and_starts(strides, shift):
    for n, k, p in ((3001, 520, 1208), (400, 520, 1208)):
        check_forward(n, k, p, "f16", "f16", strides=strides, shift=shift)
        check_backward(n, k, p, "bf16", strides=strides[:2], shift=shift)


def test_every_call_gives_the_same_bits():
    """Weight gradients of ten parts and of random values."""
    rng = np.random.default_rng(4)
    v = {k: a * (1.0 + 2.0**-6 * rng.integers(0, 8, a.shape)) for k, a in inputs(33001, 1032, 1040, 4).items()}
    first, second = (run_backward(v, "f16", "relu", dx=False, dpre=False) for _ in range(2))
    for k in first:
        equal(second[k], first[k], k)
