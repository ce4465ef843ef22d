"""Norm and clipping of many gradient tensors and the Adam step
(nerf_ext_grad_norm, nerf_ext_grad_clip, nerf_ext_adam_step) against their
definitions in 64 bits."""
import numpy as np
import pytest

from conftest import announce
from linear_cases import CODES, EPS, UNIT, decode, encode, within
from nerf_amd import _lib as L, ext
from nerf_amd.device import DeviceArray, synchronize

pytestmark = pytest.mark.gpu


def _place(values, kind, shift):
    """Device copies of the arrays at starts `shift` elements off alignment, with
    a guard after each."""
    out = []
    for i, v in enumerate(values):
        lead = 64 + (shift * (i + 1)) % 9
        host = np.full(lead + v.size + 64, 0x5A5A if kind != "f32" else 1234.5, np.uint16 if kind != "f32" else np.float32)
        host[lead : lead + v.size] = encode(v, kind)
        out.append((DeviceArray.from_numpy(host), lead, v.size, host))
    return out


def _ptr(a):
    return a[0].ptr + a[1] * a[3].itemsize


def _read(a, kind):
    now = a[0].numpy()
    got = now[a[1] : a[1] + a[2]].copy()
    now[a[1] : a[1] + a[2]] = a[3][a[1] : a[1] + a[2]]
    assert np.array_equal(now.view(np.uint8), a[3].view(np.uint8)), "bytes outside a tensor changed"
    return decode(got, kind)


def _grads(sizes, kind, seed, scale=1e-2):
    rng = np.random.default_rng(seed)
    return [decode(encode(rng.normal(0, scale, n), kind), kind) for n in sizes]


def clip(values, kind, max_norm, shift=0, inplace=False, use_clip=True):
    g = _place(values, kind, shift)
    o = g if inplace else _place([np.zeros_like(v) for v in values], kind, shift + 1)
    tensors = (L.NerfExtGradTensor * max(1, len(values)))(*[L.NerfExtGradTensor(_ptr(a), _ptr(b) if use_clip else None, a[2], CODES[kind], 0) for a, b in zip(g, o)])
    norm, ws = DeviceArray((1,), np.float32), DeviceArray((L.NERF_EXT_NORM_WORKSPACE,), np.uint8)
    if use_clip:
        L.call("nerf_ext_grad_clip", tensors, len(values), max_norm, norm.ptr, ws.ptr, ws.nbytes, None)
    else:
        L.call("nerf_ext_grad_norm", tensors, len(values), norm.ptr, ws.ptr, ws.nbytes, None)
    synchronize()
    return float(norm.numpy()[0]), [_read(a, kind) for a in o]


SIZES = [[1], [3, 0, 5], [64, 1, 63, 65], [4095, 4096, 4097], [128 * 64, 128 * 128, 128 * 48, 16 * 128, 7], [1000003], [17] * 300, [0], [(1 << 21) + 5, 12, 70001]]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("shift,inplace", [(0, False), (1, True)])
def test_norm_and_clip(sizes, kind, shift, inplace):
    announce(f"clip {len(sizes)} tensors of up to {max(sizes)} {kind} shift {shift} inplace {inplace}")
    values = _grads(sizes, kind, 1)
    want = np.sqrt(sum((v * v).sum() for v in values))
    # The sum is taken in 64 bits: the norm is off by its own rounding alone.
    bound = 2.0**-24 * want + 2.0**-140
    norm, _ = clip(values, kind, 1.0, shift, use_clip=False)
    assert abs(norm - want) <= bound
    for ratio in (0.25, 2.0):
        most = float(np.float32(ratio * want))
        norm, out = clip(values, kind, most, shift, inplace)
        assert abs(norm - want) <= bound
        factor = most / want if want > most else 1.0
        for a, v in zip(out, values):
            if factor == 1.0:
                assert np.array_equal(a, v)
            else:  # norm, quotient and product rounded to 32 bits, then to the type
                w = v * factor
                within(a, w, 3.0 * EPS * np.abs(w) + UNIT[kind] * 1.01 * np.maximum(np.abs(w), 2.0**-14 if kind == "f16" else 2.0**-126), "clipped")


def test_no_tensors():
    norm, _ = clip([], "f32", 1.0)
    assert norm == 0.0
    norm, _ = clip([np.zeros(0)], "f32", 1.0, use_clip=False)
    assert norm == 0.0


def test_zero_gradients_and_zero_limit():
    norm, out = clip([np.zeros(1000)], "f32", 0.0)
    assert norm == 0.0 and not out[0].any()
    norm, out = clip([np.ones(1000)], "f32", 0.0)
    assert not out[0].any()


def test_large_and_small_gradients():
    """Squares beyond and below 32 bits."""
    big = [np.full(100, 1e30), np.full(50, 1e-3)]
    norm, out = clip(big, "f32", 1.0)
    assert abs(norm - 1e31) <= 1e31 * 1e-6
    within(out[0], np.full(100, 0.1), 1e-6, "clipped")
    small = [np.full(400, 1e-30)]
    norm, _ = clip(small, "f32", 1.0)
    assert abs(norm - 2e-29) <= 2e-29 * 1e-6


@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_norm_that_is_not_finite_leaves_gradients(value):
    values = _grads([5000, 77], "f32", 4)
    values[1][13] = value
    norm, out = clip(values, "f32", 1e-3)
    assert not np.isfinite(norm)
    for a, v in zip(out, values):
        assert np.array_equal(a, v, equal_nan=True)


def test_more_elements_than_32_bits_count():
    """2^32 + 4097 equal fp16 gradients, clipped in place."""
    n = (1 << 32) + 4097
    g = DeviceArray((n,), np.float16)
    g.fill_bytes(0x3C)  # 0x3C3C = 1.05859375
    value = float(np.uint16(0x3C3C).view(np.float16))
    want = value * np.sqrt(float(n))
    tensors = (L.NerfExtGradTensor * 1)(L.NerfExtGradTensor(g.ptr, g.ptr, n, CODES["f16"], 0))
    norm, ws = DeviceArray((1,), np.float32), DeviceArray((L.NERF_EXT_NORM_WORKSPACE,), np.uint8)
    L.call("nerf_ext_grad_clip", tensors, 1, float(np.float32(want / 4.0)), norm.ptr, ws.ptr, ws.nbytes, None)
    synchronize()
    assert abs(float(norm.numpy()[0]) - want) <= 2.0**-23 * want
    for at in (0, (1 << 31) - 3, (1 << 32) - 5, n - 7):
        got = ext.read_device(g.ptr + 2 * at, (7,), np.float16).astype(np.float64)
        assert np.abs(got - value / 4.0).max() <= 2.0**-11 * value / 4.0 * 1.01, at


def test_same_norm_every_time():
    values = _grads([300007, 1234567], "f32", 5)
    assert len({clip(values, "f32", 1.0, use_clip=False)[0] for _ in range(5)}) == 1


def adam(p, g, m, v, copy_kind, hyper, step, norm, shift=0):
    arrays = [_place(a, "f32", shift + i) for i, a in enumerate((p, g, m, v))]
    copies = _place([np.zeros_like(a) for a in p], copy_kind, shift) if copy_kind else None
    rows = [L.NerfExtAdamTensor(*[_ptr(a[i]) for a in arrays], _ptr(copies[i]) if copies else None, p[i].size, CODES[copy_kind] if copy_kind else 0, 0) for i in range(len(p))]
    n, skipped = DeviceArray.from_numpy(np.array([norm], np.float32)), DeviceArray.from_numpy(np.array([7], np.uint32))
    import ctypes as C

    L.call("nerf_ext_adam_step", (L.NerfExtAdamTensor * len(rows))(*rows), len(rows), C.byref(hyper), step, n.ptr, skipped.ptr, None)
    synchronize()
    got = [[_read(a, "f32") for a in k] for k in arrays]
    return got[0], got[2], got[3], [_read(a, copy_kind) for a in copies] if copies else None, int(skipped.numpy()[0])


def _state(sizes, seed):
    rng = np.random.default_rng(seed)
    f = lambda scale: [rng.normal(0, scale, n).astype(np.float32).astype(np.float64) for n in sizes]  # noqa: E731
    v = [np.float32(np.abs(a)).astype(np.float64) for a in f(1e-4)]
    return f(0.1), f(1.0), f(1e-2), v


HYPER = dict(learning_rate=1e-2, adam_beta1=0.9, adam_beta2=0.99, adam_eps=1e-8, grad_clip_norm=1e30, update_guard_grad_norm=1e30, loss_scale=128.0, lr_decay_ksteps=0)


@pytest.mark.parametrize("sizes", SIZES[:7] + SIZES[8:], ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("copy_kind,step,ksteps,ratio,shift", [("f16", 1, 0, 2.0, 0), ("bf16", 100, 1, 0.25, 1), (None, 7, 0, 0.5, 0)])
def test_adam(sizes, copy_kind, step, ksteps, ratio, shift):
    announce(f"adam {len(sizes)} tensors of up to {max(sizes)} copy {copy_kind} step {step}")
    p, g, m, v = _state(sizes, 2)
    norm = float(np.float32(np.sqrt(sum((a * a).sum() for a in g))))
    hyper = L.NerfHyperParams(**{**HYPER, "lr_decay_ksteps": ksteps, "grad_clip_norm": ratio * norm / 128.0})
    gp, gm, gv, gc, skipped = adam(p, g, m, v, copy_kind, hyper, step, norm, shift)
    assert skipped == 0
    b1, b2, lr, eps, most = (float(getattr(hyper, k)) for k in ("adam_beta1", "adam_beta2", "learning_rate", "adam_eps", "grad_clip_norm"))
    if ksteps:
        lr *= 0.1 ** (step / (1000.0 * ksteps))
    scale = min(1.0, most / (norm / 128.0)) / 128.0
    for i in range(len(sizes)):
        r = g[i] * scale
        wm = b1 * m[i] + (1 - b1) * r
        wv = b2 * v[i] + (1 - b2) * r * r
        mh, vh = wm / (1 - b1**step), wv / (1 - b2**step)
        wp = p[i] - lr * mh / (np.sqrt(vh) + eps)
        # Each term takes a handful of 32-bit roundings; m's terms may cancel.
        em = 8 * EPS * (np.abs(b1 * m[i]) + np.abs((1 - b1) * r))
        ev = 12 * EPS * wv + 2.0**-140
        within(gm[i], wm, em, "m")
        within(gv[i], wv, ev, "v")
        move = lr / (np.sqrt(vh) + eps)
        ep = 2 * EPS * np.abs(p[i]) + move * (em / (1 - b1**step) + 32 * EPS * np.abs(mh))
        within(gp[i], wp, ep, "param")
        if gc:
            within(gc[i], wp, ep + UNIT[copy_kind] * 1.01 * np.maximum(np.abs(wp), 2.0**-14), "copy")


@pytest.mark.parametrize("norm,guard", [(np.inf, 1e30), (np.nan, 1e30), (300.0, 2.0)])
def test_adam_skips(norm, guard):
    p, g, m, v = _state([100, 5000], 3)
    gp, gm, gv, gc, skipped = adam(p, g, m, v, "f16", L.NerfHyperParams(**{**HYPER, "update_guard_grad_norm": guard}), 3, norm)
    assert skipped == 1
    for got, old in ((gp, p), (gm, m), (gv, v)):
        assert all(np.array_equal(a, b) for a, b in zip(got, old))
    assert not any(c.any() for c in gc)
