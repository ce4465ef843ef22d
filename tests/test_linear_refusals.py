"""What nerf_ext_linear_*, nerf_ext_grad_* and nerf_ext_adam_step refuse,
decided on the host before any GPU work; and the 64-bit definitions that the
GPU tests compare with, checked against finite differences."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from linear_cases import ACTS, act, backward, decode, encode, slope
from nerf_amd import _lib as L

BAD = L.NERF_STATUS_INVALID_USAGE
A = 1 << 20  # an address that is never followed


def desc(**kw):
    d = L.NerfExtLinearDesc(4, 8, 16, L.NERF_EXT_F16, L.NERF_EXT_F16, L.NERF_EXT_ACT_RELU, 0, 0, 0, 0)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def fwd(d, x=A, w=A, b=A, r=A, y=A, z=A, ws=A, nb=1 << 20):
    return L.status_of("nerf_ext_linear_forward", C.byref(d) if d else None, x, w, b, r, y, z, ws, nb, None)


def bwd(d, x=A, w=A, g=A, z=A, a=A, dx=A, dz=A, dw=A, db=A, ws=A, nb=1 << 20):
    return L.status_of("nerf_ext_linear_backward", C.byref(d) if d else None, x, w, g, z, a, dx, dz, dw, db, ws, nb, None)


@pytest.mark.parametrize("change,word", [(dict(in_features=0), "features"), (dict(out_features=0), "features"), (dict(in_features=65537), "features"), (dict(out_features=1 << 31), "features"), (dict(rows=(1 << 30) + 1), "rows"),
                                         (dict(dtype=L.NERF_EXT_F32), "dtype"), (dict(dtype=3), "dtype"), (dict(out_dtype=L.NERF_EXT_BF16), "out_dtype"), (dict(activation=6), "activation"), (dict(x_stride=7), "stride"),
                                         (dict(y_stride=15), "stride"), (dict(residual_stride=15), "stride"), (dict(x_stride=(1 << 20) + 1), "stride"), (dict(reserved=1), "reserved")])
def test_descriptors(lib, change, word):
    for call in (fwd, bwd):
        assert call(desc(**change)) == BAD
        assert word in L.last_error()


def test_forward_arrays(lib):
    assert fwd(None) == BAD
    for kw in (dict(x=None), dict(w=None), dict(y=None), dict(x=A + 1), dict(w=A + 1), dict(b=A + 2), dict(r=A + 1), dict(y=A + 1), dict(z=A + 1), dict(ws=A + 8)):
        assert fwd(desc(), **kw) == BAD, kw
        assert "nerf_ext_linear_forward" in L.last_error()
    assert fwd(desc(out_dtype=L.NERF_EXT_F32), y=A + 2) == BAD


def test_backward_arrays(lib):
    assert bwd(None) == BAD
    for kw in (dict(x=None), dict(w=None), dict(g=None), dict(z=None), dict(dx=None, dz=None, dw=None, db=None), dict(dw=None), dict(x=A + 1), dict(g=A + 1), dict(dw=A + 2), dict(db=A + 2), dict(dx=A + 1), dict(a=A + 1), dict(dz=A + 1),
               dict(z=A + 1), dict(w=A + 1), dict(ws=A + 8)):
        assert bwd(desc(), **kw) == BAD, kw
        assert "nerf_ext_linear_backward" in L.last_error()


def test_no_rows_need_no_arrays(lib):
    assert fwd(desc(rows=0), x=None, w=None, b=None, r=None, y=None, z=None, ws=None, nb=0) == L.NERF_STATUS_OK


def grads(n=1, **kw):
    t = L.NerfExtGradTensor(A, A, 10, L.NERF_EXT_F32, 0)
    for k, v in kw.items():
        setattr(t, k, v)
    return (L.NerfExtGradTensor * n)(*[t] * n)


def test_gradient_lists(lib):
    nb = L.NERF_EXT_NORM_WORKSPACE
    for fn, args in (("nerf_ext_grad_norm", ()), ("nerf_ext_grad_clip", (1.0,))):
        def call(t, n=1, norm=A, ws=A, b=nb):
            return L.status_of(fn, t, n, *args, norm, ws, b, None)

        assert call(None) == BAD
        assert call(grads(), norm=None) == BAD and call(grads(), norm=A + 1) == BAD
        assert call(grads(), ws=None) == BAD and call(grads(), ws=A + 8) == BAD and call(grads(), b=nb - 1) == BAD
        for kw in (dict(dtype=3), dict(reserved=1), dict(grad=None), dict(grad=A + 2), dict(count=(1 << 34) + 1), dict(grad=A + 1, dtype=L.NERF_EXT_F16)):
            assert call(grads(**kw)) == BAD, kw
            assert fn in L.last_error()
        assert call(grads(), n=(1 << 20) + 1) == BAD
    assert L.status_of("nerf_ext_grad_clip", grads(out=None), 1, 1.0, A, A, nb, None) == BAD
    assert L.status_of("nerf_ext_grad_clip", grads(out=A + 2), 1, 1.0, A, A, nb, None) == BAD
    for most in (-1.0, float("nan")):
        assert L.status_of("nerf_ext_grad_clip", grads(), 1, most, A, A, nb, None) == BAD


def test_adam_arguments(lib):
    hyper = L.NerfHyperParams(1e-2, 0.9, 0.99, 1e-8, 1.0, 1e30, 128.0, 0)

    def call(h=hyper, step=1, norm=A, skipped=None, n=1, **kw):
        t = L.NerfExtAdamTensor(A, A, A, A, A, 10, L.NERF_EXT_F16, 0)
        for k, v in kw.items():
            setattr(t, k, v)
        return L.status_of("nerf_ext_adam_step", (L.NerfExtAdamTensor * 1)(t), n, C.byref(h) if h else None, step, norm, skipped, None)

    assert L.status_of("nerf_ext_adam_step", None, 1, C.byref(hyper), 1, A, None, None) == BAD
    for kw in (dict(h=None), dict(step=0), dict(norm=None), dict(norm=A + 2), dict(skipped=A + 2), dict(n=(1 << 20) + 1), dict(param=None), dict(grad=None), dict(m=None), dict(v=None), dict(param=A + 2), dict(copy=A + 1),
               dict(copy_dtype=L.NERF_EXT_F32), dict(reserved=1), dict(count=(1 << 34) + 1)):
        assert call(**kw) == BAD, kw
        assert "nerf_ext_adam_step" in L.last_error()
    for field, value in (("loss_scale", 0.0), ("loss_scale", float("nan")), ("adam_beta1", 1.0), ("adam_beta2", -0.1), ("adam_beta2", float("nan"))):
        h = L.NerfHyperParams(1e-2, 0.9, 0.99, 1e-8, 1.0, 1e30, 128.0, 0)
        setattr(h, field, value)
        assert call(h=h) == BAD, (field, value)


def test_structures_as_c_lays_them_out(tmp_path):
    sizes = {"NerfExtLinearDesc": L.NerfExtLinearDesc, "NerfExtGradTensor": L.NerfExtGradTensor, "NerfExtAdamTensor": L.NerfExtAdamTensor}
    lines = ["#include <stddef.h>", '#include "nerf_ext.h"']
    for name, struct in sizes.items():
        lines.append(f'_Static_assert(sizeof({name}) == {C.sizeof(struct)}, "{name}");')
        lines += [f'_Static_assert(offsetof({name}, {field[0]}) == {getattr(struct, field[0]).offset}, "{name}.{field[0]}");' for field in struct._fields_]
    for name in ("NERF_EXT_BF16", "NERF_EXT_ACT_NONE", "NERF_EXT_ACT_RELU", "NERF_EXT_ACT_SOFTPLUS", "NERF_EXT_ACT_SIGMOID", "NERF_EXT_ACT_SILU", "NERF_EXT_ACT_GELU", "NERF_EXT_LINEAR_WORKSPACE", "NERF_EXT_NORM_WORKSPACE"):
        lines.append(f'_Static_assert({name} == {getattr(L, name)}, "{name}");')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines) + "\n")
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{include}", "-fsyntax-only", str(src)], check=True)


@pytest.mark.parametrize("name", list(ACTS))
def test_slopes_are_the_activations_differences(name):
    z = np.linspace(-8.0, 8.0, 400)  # no point at 0, where relu has none
    h = 1e-4
    numeric = (act(z + h, name) - act(z - h, name)) / (2.0 * h)
    assert np.abs(numeric - slope(z, name)).max() < 1e-7


def test_gradients_are_the_layers_differences():
    """sum c (act(x W^T + b) through a layer behind act(pre)): 64-bit differences."""
    rng = np.random.default_rng(0)
    n, i, o = 7, 5, 6
    pre, w, c, add = rng.normal(size=(n, i)), rng.normal(size=(o, i)), rng.normal(size=(n, o)), rng.normal(size=(n, i))
    want = backward(act(pre, "silu"), w, c, pre, add, "silu", "f32")
    loss = lambda p, u, b: (c * (act(p, "silu") @ u.T + b)).sum() + (add * act(p, "silu")).sum()  # noqa: E731
    h = 1e-5
    for _ in range(5):
        dp, dw, db = rng.normal(size=pre.shape), rng.normal(size=w.shape), rng.normal(size=o)
        numeric = (loss(pre + h * dp, w + h * dw, h * db) - loss(pre - h * dp, w - h * dw, -h * db)) / (2.0 * h)
        analytic = (want["dpre"][0] * dp).sum() + (want["dw"][0] * dw).sum() + (want["db"][0] * db).sum()
        assert abs(numeric - analytic) < 1e-7 * (1.0 + abs(analytic))


def test_bf16_conversion():
    v = np.float32([1.0, 1.00390625, 1.01171875, -2.5, 3.4e38, np.inf, np.nan])
    got = decode(encode(v, "bf16"), "bf16")
    assert got[0] == 1.0 and got[1] == 1.0 and got[2] == 1.015625 and got[3] == -2.5 and np.isinf(got[4]) and np.isinf(got[5]) and np.isnan(got[6])
