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
    """The call without a workspace: -12 if its sizes are taken."""
    return rt.lib().b200_linear_i8(ctypes.byref(linear_args(rt, **kw)), None)


def test_sums_stay_in_32_bits_for_every_code(pkg):
    """Codes of x lie in -127 .. 127, of w in -128 .. 127: 127 * 128 * k < 2^31."""
    rt = pkg.runtime
    most = (2 ** 31 - 1) // (127 * 128)
    ld = (most + 31) // 16 * 16
    assert linear(rt, k=most, ld_x=ld, ld_w=ld) == -12
    assert linear(rt, k=most + 1, ld_x=ld, ld_w=ld) == -2


def test_linear_refuses_outputs_that_overlap(pkg):
    rt = pkg.runtime

    def laid(rt, **kw):  # -5 (a workspace off 16 bytes, looked at last) if the layout is taken
        return linear(rt, workspace=4097, workspace_bytes=1 << 40, **kw)

    x, w, out = 1 << 20, 1 << 30, 1 << 40
    assert laid(rt) == -5
    assert laid(rt, out=x) == -9
    assert laid(rt, out=x + 99 * 128 + 120) == -9              # its first bytes are x's last
    assert laid(rt, out=x + 100 * 128) == -5                  # right behind x
    assert laid(rt, out=x - 100 * 128) == -5 and laid(rt, out=x - 99 * 128) == -9
    assert laid(rt, out=w + 64 * 63) == -9
    assert laid(rt, w_scale=out + 64) == -9 and laid(rt, bias=out + 12736) == -9
    assert laid(rt, w_scale=out + 12800) == -5 and laid(rt, w_scale=out - 256) == -5
    # columns of one wider buffer, side by side
    assert laid(rt, ld_x=128, ld_out=128, out=x + 128) == -5
    assert laid(rt, ld_x=128, ld_out=128, out=x + 120) == -9 and laid(rt, ld_x=128, ld_out=128, out=x + 136) == -9
    assert laid(rt, ld_x=192, ld_out=192, out=x - 128) == -5 and laid(rt, ld_x=192, ld_out=192, out=x + 200) == -5
    assert laid(rt, ld_x=192, ld_out=128, out=x + 128) == -9   # other pitches: not told apart
    # the residual: out itself, or beside it
    assert laid(rt, out_type=2, resid=out) == -5
    assert laid(rt, out_type=2, resid=out + 16) == -9 and laid(rt, out_type=2, resid=out, ld_resid=128) == -9
    assert laid(rt, out_type=2, resid=out + 256, ld_resid=128, ld_out=128) == -5
    assert laid(rt, m=65, out_type=2, resid=out + 64 * 256, ld_resid=64) == -9
    assert laid(rt, m=65, out_type=2, resid=out + 65 * 256, ld_resid=64) == -5
    assert laid(rt, m=1, k=9000, ld_x=9000, ld_w=9008, out_type=2, resid=out, ld_resid=640) == -5  # one row has no pitch


def kv8(rt, **kw):
    c = rt.KvCache8()
    for i, name in enumerate(("k_pages", "v_pages", "k_scale", "v_scale", "k_newest", "v_newest", "table")):
        setattr(c, name, (i + 1) << 44)
    c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.newest_rows, c.table_width, c.batch = 8, 2, 64, 64, 4, 2, 4
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_attention_refuses_outputs_that_overlap(pkg):
    rt = pkg.runtime
    q = 1 << 20

    def attend(out, ld_q=256, ld_out=256, tokens=100):
        return rt.lib().b200_kv8_attention(kv8(rt), q, ld_q, out, ld_out, 256, 64, tokens, 4, 1, 1.0, 4097, 1 << 40, None)

    assert attend(q) == -5 and attend(1 << 30) == -5 and attend(q + 100 * 512) == -5
    assert attend(q + 512) == -9 and attend(q + 99 * 512) == -9 and attend(q - 16) == -9
    assert attend(q, ld_out=512) == -9 and attend(q, ld_out=512, tokens=1) == -5
    assert attend(q + 512, 512, 512) == -5 and attend(q + 496, 512, 512) == -9


def test_append_refuses_outputs_that_overlap(pkg):
    rt = pkg.runtime
    qkv = 1 << 20

    def append(out, tokens, ld=512):
        return rt.lib().b200_kv8_append(kv8(rt), qkv, ld, out, 256, 64, None, None, 0, 0, 0, tokens, 4, None)

    for out, tokens in ((qkv, 3), (qkv, 1), (qkv + 512, 1), (qkv + 1008, 1), (qkv - 496, 1), (qkv + 3 * 1024 - 16, 3), (qkv - 1024, 3)):
        assert append(out, tokens) == -9, (out - qkv, tokens)


def test_attention_over_wide_tables_is_taken(pkg):
    """Work that the warps' kernel could not number in 32 bits goes to the other one, which has no such line."""
    rt = pkg.runtime

    def attend(c, tokens, most, heads):  # -5: a workspace off 16 bytes, looked at last
        return rt.lib().b200_kv8_attention(c, 1 << 20, 64 * heads, 1 << 40, 64 * heads, 256, 64, tokens, heads, most, 1.0, 4097,
                                           1 << 40, None)

    wide = kv8(rt, kv_heads=16, table_width=1 << 24)
    assert attend(wide, 1, 1, 16) == -5
    assert attend(wide, 4, 1, 16) == -5
    assert attend(kv8(rt, kv_heads=8, table_width=4096, batch=2048), 1 << 19, 256, 64) == -5
    assert attend(kv8(rt, kv_heads=1024), 0x7fffffff, 1 << 20, 1024) == -2   # items of 256 rows that 32 bits do not number
    assert attend(kv8(rt), 0x7fffffff, 1 << 20, 4) == -2                     # rows that 32 bits do not number
