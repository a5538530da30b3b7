"""Limits of the 8-bit serving entry points, found out before any CUDA call."""

import ctypes

import pytest  # noqa: F401


def linear_args(rt, **kw):
    a = rt.LinearI8Args()
    a.x, a.w, a.w_scale, a.out = 1 << 20, 1 << 30, 64, 1 << 40
    a.ld_x, a.ld_w, a.ld_resid, a.ld_out, a.m, a.n, a.k = 64, 64, 64, 64, 100, 64, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def linear(rt, **kw):
    """The call without a workspace: -12 if its other arguments are taken."""
    return rt.lib().b200_linear_i8(ctypes.byref(linear_args(rt, **kw)), None)


def test_sums_stay_in_32_bits_for_every_code(pkg):
    """Codes of x lie in -127 .. 127, of w in -128 .. 127: 127 * 128 * k < 2^31."""
    rt = pkg.runtime
    most = (2 ** 31 - 1) // (127 * 128)
    ld = (most + 31) // 16 * 16
    assert linear(rt, k=most, ld_x=ld, ld_w=ld) == -12
    assert linear(rt, k=most + 1, ld_x=ld, ld_w=ld) == -2
