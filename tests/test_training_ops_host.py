"""Argument checks of the training operators' C entry points, on the CPU: no call here launches anything."""
import ctypes

import pytest

from comfy_ui_gfx906_tools_b200 import _lib

INVALID, UNSUPPORTED, WORKSPACE = _lib.GFX_ERR_INVALID, _lib.GFX_ERR_UNSUPPORTED, _lib.GFX_ERR_WORKSPACE


def _adamw(lib, p=(16, 32), g=(16, 32), m=(16, 32), v=(16, 32), ms=(16, 32), vs=(16, 32), n=(0, 0), count=2, pd=2, gd=2,
           bits=32, step=1, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0):
    def arr(x):
        return (ctypes.c_void_p * len(x))(*x) if x is not None else None
    return lib.adamw_step(arr(p), arr(g), arr(m), arr(v), arr(ms), arr(vs),
                          (ctypes.c_int64 * len(n))(*n) if n is not None else None, count, pd, gd, bits, step, lr, b1,
                          b2, eps, wd, None, None)


@pytest.mark.parametrize("kw,needle", [
    (dict(count=-1), "count"), (dict(pd=3), "dtype"), (dict(gd=-1), "dtype"), (dict(bits=16), "state_bits"),
    (dict(step=0), "step"), (dict(b1=1.0), "betas"), (dict(b2=float("nan")), "betas"), (dict(lr=-1.0), "lr"),
    (dict(eps=float("nan")), "eps"), (dict(wd=-0.1), "weight_decay"), (dict(p=None), "null"), (dict(n=None), "null"),
    (dict(ms=None, bits=8), "null"), (dict(n=(4, -1)), "tensor 1 has -1"), (dict(n=(4, 4), g=(16, None)), "tensor 1"),
    (dict(n=(4, 4), vs=(16, None), bits=8), "tensor 1"), (dict(n=(4, 4), p=(17, 32)), "tensor 0 is not aligned"),
    (dict(n=(4, 4), m=(16, 34)), "tensor 1 is not aligned"),
])
def test_adamw_argument_checks(built_lib, kw, needle):
    assert _adamw(built_lib, **kw) == INVALID
    assert needle in _lib.last_error()


def test_adamw_nothing_to_do(built_lib):
    assert _adamw(built_lib, count=0, p=None) == _lib.GFX_OK
    assert _adamw(built_lib) == _lib.GFX_OK  # tensors without elements
    assert built_lib.adamw_moment_values(None, None, None, 0, 0, None) == _lib.GFX_OK
    assert built_lib.adamw_moment_values(None, None, None, 4, 0, None) == INVALID
    assert built_lib.adamw_moment_values(16, 18, 16, 4, 0, None) == INVALID
    assert built_lib.adamw_moment_values(16, 16, 16, -1, 0, None) == INVALID


def _rope(lib, back=False, q=16, k=16, dt=2, pos=16, pdt=1, qs=16, ks=16, sdt=2, out=16, B=1, Hq=2, Hk=1, L=3, D=64,
          axes=(64,), theta=1e4, inter=1, eps=1e-6, strides=True, ws=16, wsb=None, dqs=16):
    st = (ctypes.c_int64 * 3)(64, 64, 64) if strides else None
    ax = (ctypes.c_int * len(axes))(*axes) if axes is not None else None
    n = len(axes) if axes is not None else 1
    tail = (B, Hq, Hk, L, D, ax, n, theta, inter, eps)
    if not back:
        return lib.qk_norm_rope(q, st, k, st, dt, pos, pdt, st, qs, ks, sdt, out, st, out, st, *tail, None)
    need = lib.qk_norm_rope_workspace_bytes(D) if wsb is None else wsb
    return lib.qk_norm_rope_backward(16, st, 16, st, q, st, k, st, dt, pos, pdt, st, qs, ks, sdt, out, st, out, st, dqs,
                                     None, *tail, ws, need, None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(dt=3), INVALID, "dtype"), (dict(sdt=7), INVALID, "dtype"), (dict(pdt=3), INVALID, "positions"),
    (dict(B=-1), INVALID, "B=-1"), (dict(B=1 << 20, L=1 << 11), UNSUPPORTED, "2^30 tokens"),
    (dict(Hk=1 << 21), UNSUPPORTED, "2^20 heads"), (dict(D=20), UNSUPPORTED, "multiple of 8"), (dict(D=264), UNSUPPORTED, "up to 256"),
    (dict(axes=None), INVALID, "axes"), (dict(axes=(2,) * 9), INVALID, "between 1 and 8"),
    (dict(axes=(5,)), INVALID, "even"), (dict(axes=(0, 64)), INVALID, "even"), (dict(axes=(64, 2)), INVALID, "add up"),
    (dict(axes=(2 ** 30, 2 ** 30, 2 ** 30, 2 ** 30)), INVALID, "add up"),
    (dict(axes=(12,), inter=0), UNSUPPORTED, "split halves"), (dict(theta=float("nan")), INVALID, "theta"),
    (dict(eps=-1.0), INVALID, "eps"), (dict(q=None), INVALID, "q is a null"), (dict(k=None), INVALID, "k is a null"),
    (dict(out=None), INVALID, "q"), (dict(pos=None), INVALID, "positions"), (dict(strides=False), INVALID, "strides"),
    (dict(q=17), INVALID, "aligned"), (dict(pos=18), INVALID, "aligned"), (dict(qs=17), INVALID, "aligned"),
])
def test_rope_argument_checks(built_lib, kw, code, needle):
    for back in (False, True):
        assert _rope(built_lib, back, **kw) == code
        assert needle in _lib.last_error()


def test_rope_backward_checks(built_lib):
    assert _rope(built_lib, True, ws=None) == WORKSPACE and "workspace" in _lib.last_error()
    assert _rope(built_lib, True, wsb=16) == WORKSPACE
    assert _rope(built_lib, True, ws=8) == WORKSPACE
    assert _rope(built_lib, True, qs=None) == INVALID and "scale is null" in _lib.last_error()
    assert _rope(built_lib, True, dqs=17) == INVALID
    assert _rope(built_lib, False, B=0, q=None, k=None, pos=None) == _lib.GFX_OK
    assert _rope(built_lib, False, Hq=0, Hk=0) == _lib.GFX_OK
    assert _rope(built_lib, True, L=0, dqs=None, qs=None) == _lib.GFX_OK


def _gated(lib, back=False, x=16, wg=16, wu=16, h=16, save=16, bg=None, dt=2, act=0, M=3, K=64, F=72, ldx=64, ldg=64,
           ldu=64, lddh=72, ws=16, wsb=1 << 20, dx=16, dw=16):
    if not back:
        return lib.gated_linear(x, ldx, wg, ldg, wu, ldu, bg, None, dt, act, h, save, M, K, F, ws, wsb, None)
    return lib.gated_linear_backward(h, lddh, x, ldx, wg, ldg, wu, ldu, save, dt, act, dx, dw, None, bg, None, M, K, F,
                                     ws, wsb, None)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(dt=0), UNSUPPORTED, "dtype"), (dict(act=3), INVALID, "act"), (dict(M=-1), INVALID, "M >= 0"),
    (dict(K=60), INVALID, "multiples of 8"), (dict(F=70), INVALID, "multiples of 8"), (dict(K=0), INVALID, "K=0"),
    (dict(F=1 << 23), UNSUPPORTED, "2^22"), (dict(ldx=56), INVALID, "row strides"), (dict(ldg=65), INVALID, "row strides"),
    (dict(x=None), INVALID, "null"), (dict(wu=None), INVALID, "null"), (dict(h=None), INVALID, "null"),
    (dict(x=24), INVALID, "16-byte"), (dict(h=8), INVALID, "16-byte"), (dict(save=4), INVALID, "16-byte"),
    (dict(bg=17), INVALID, "bias"),
])
def test_gated_argument_checks(built_lib, kw, code, needle):
    for back in (False, True):
        assert _gated(built_lib, back, **kw) == code
        assert needle in _lib.last_error()


def test_gated_backward_checks(built_lib):
    assert _gated(built_lib, True, lddh=64) == INVALID and "dh's row stride" in _lib.last_error()
    assert _gated(built_lib, True, save=None) == INVALID
    assert _gated(built_lib, True, dx=18) == INVALID
    assert _gated(built_lib, True, ws=None) == WORKSPACE
    assert _gated(built_lib, True, ws=24) == WORKSPACE
    assert _gated(built_lib, True, wsb=100) == WORKSPACE and "workspace of" in _lib.last_error()
    many = dict(M=700, K=6400, ldx=6400, ldg=6400, ldu=6400)  # few tiles, a long contraction: cut and joined
    assert built_lib.gated_linear_workspace_bytes(700, 6400, 72) > 1 << 18
    assert _gated(built_lib, False, ws=None, **many) == WORKSPACE and "workspace of" in _lib.last_error()
    assert _gated(built_lib, False, wsb=1000, **many) == WORKSPACE
    assert _gated(built_lib, False, M=0, x=None, h=None) == _lib.GFX_OK
    assert _gated(built_lib, True, M=0, dx=None, dw=None, x=None) == _lib.GFX_OK
    assert built_lib.gated_linear_backward_workspace_bytes(0, 8, 8) == 0
    assert built_lib.gated_linear_workspace_bytes(4, 0, 8) == 0
