"""The 8-bit serving entry points refuse what they do not take, before any CUDA call."""

import ctypes

import pytest
import torch


def cache(rt, **kw):
    c = rt.KvCache8()
    for name in ("k_pages", "v_pages", "k_scale", "v_scale", "k_newest", "v_newest", "table"):
        setattr(c, name, 4096)
    c.num_pages, c.kv_heads, c.page_size, c.head_dim, c.newest_rows, c.table_width, c.batch = 8, 2, 64, 64, 4, 2, 4
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def test_cache_checks(pkg):
    rt = pkg.runtime
    lib = rt.lib()

    def read(c, tokens=1):
        return lib.b200_kv8_read(c, 64, 64, 64, 4096, 4096, tokens, None)

    assert read(cache(rt), 0) == 0
    assert read(cache(rt, k_pages=None)) == -9
    assert read(cache(rt, table=None)) == -9
    assert read(cache(rt, head_dim=80)) == -6
    assert read(cache(rt, page_size=24)) == -2
    assert read(cache(rt, batch=5000)) == -2
    assert read(cache(rt, v_newest=4100)) == -5
    assert read(cache(rt, num_pages=0)) == -9
    assert read(cache(rt, table_width=1 << 30)) == -2
    assert read(cache(rt), -1) == -9


def test_append_checks(pkg):
    rt = pkg.runtime
    lib = rt.lib()

    def append(qkv=4096, ld=6 * 64, q=8192, cu=64, start=64, cos=None, sin=None, rot=0, rows=0, tokens=1, heads=2):
        return lib.b200_kv8_append(cache(rt), qkv, ld, q, cu, start, cos, sin, rot, 0, rows, tokens, heads, None)

    assert append(tokens=0) == 0
    assert append(heads=3) == -9
    assert append(ld=6 * 64 - 8) == -9
    assert append(ld=6 * 64 + 4) == -5
    assert append(qkv=4104) == -5
    assert append(cos=64) == -9
    assert append(cos=64, sin=64, rot=24, rows=8) == -2
    assert append(cos=64, sin=64, rot=80, rows=8) == -2
    assert append(cu=None) == -9


def test_attention_checks(pkg):
    rt = pkg.runtime
    lib = rt.lib()

    def attend(c=None, ld=4 * 64, tokens=1, heads=4, most=1, ws=4096, size=1 << 40):
        return lib.b200_kv8_attention(cache(rt) if c is None else c, 4096, ld, 8192, 256, 64, 64, tokens, heads, most, 1.0, ws,
                                      size, None)

    assert attend(tokens=0) == 0
    assert attend(heads=3) == -9
    assert attend(most=0) == -9
    assert attend(ld=128) == -9
    assert attend(ld=260) == -5
    assert attend(ws=None) == -12
    assert attend(size=16) == -12
    assert attend(cache(rt, batch=4096, table_width=1 << 20)) == -2  # work that 32 bits do not number
    assert lib.b200_kv8_attention_workspace_bytes(0, 4, 2, 64, 1) == 0
    assert lib.b200_kv8_attention_workspace_bytes(4, 4, 2, 64, 1) > 0


def test_linear_checks(pkg):
    rt = pkg.runtime
    lib = rt.lib()

    def linear(**kw):
        a = rt.LinearI8Args()
        a.x, a.w, a.w_scale, a.out, a.workspace, a.workspace_bytes = 4096, 4096, 64, 4096, 4096, 1 << 30
        a.ld_x, a.ld_w, a.ld_resid, a.ld_out, a.m, a.n, a.k = 64, 64, 64, 64, 1, 64, 64
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.b200_linear_i8(ctypes.byref(a), None)

    assert linear(m=0) == 0
    assert linear(x=None) == -9
    assert linear(k=0) == -9
    assert linear(x_type=3) == -1
    assert linear(resid=4096) == -1                 # fp16 output
    assert linear(resid=4096, out_type=2, gelu=1) == -1
    assert linear(ld_x=63) == -9
    assert linear(ld_w=72) == -5
    assert linear(w=4104) == -5
    assert linear(k=200000, ld_x=200000, ld_w=200000) == -2  # sums past int32
    assert linear(m=100, workspace_bytes=8) == -12
    assert lib.b200_linear_i8_workspace_bytes(64, 64) == 0 < lib.b200_linear_i8_workspace_bytes(65, 64)  # few rows need none
    assert lib.b200_quantize_rows_i8(4096, 5, 8, 4096, 16, 64, 1, 8, None) == -1
    assert lib.b200_quantize_rows_i8(4096, 0, 7, 4096, 16, 64, 1, 8, None) == -9
    assert lib.b200_quantize_rows_i8(4096, 0, 8, 4096, 16, 64, 0, 8, None) == 0


def test_cpu_tensors_are_refused(pkg):
    sv = pkg.serving
    table = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        sv.PagedKV8.allocate(8, 2, 64, 64, table)
    with pytest.raises(RuntimeError, match="CUDA"):
        sv.quantize_weight(torch.randn(4, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        sv.linear_int8(torch.randn(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4))
    with pytest.raises(ValueError):
        sv.PagedKV8.allocate(8, 2, 48, 64, table)


def test_ops_fake_shapes(pkg):
    """torch.ops.b200's serving ops under a fake mode (what torch.compile traces with)."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.b200
    with FakeTensorMode():
        def t(*shape, dtype=torch.float16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        x, w, ws = t(5, 100), t(40, 112, dtype=torch.int8), t(40, dtype=torch.float32)
        assert ops.linear_int8(x, w, ws, None, True, None, False).shape == (5, 40)
        assert ops.linear_int8(x, w, ws, None, False, t(5, 40, dtype=torch.float32), False).dtype == torch.float32
        u8, f32, i32 = torch.uint8, torch.float32, torch.int32
        cache = (t(9, 2, 16, 64, dtype=u8), t(9, 2, 4, 64, 4, dtype=u8), t(9, 2, dtype=f32), t(9, 2, dtype=f32),
                 t(3, 2, 2, 16, 64), t(3, 2, 2, 4, 64, 4), t(3, 3, dtype=i32), None)
        cu, at = t(4, dtype=i32), t(3, dtype=i32)
        q = ops.kv8_append(t(7, 8 * 64), *cache, cu, at, 4, None, None, False)
        assert q.shape == (7, 4, 64) and q.dtype == torch.float16
        k, v = ops.kv8_read(*cache, cu, at, at, 11)
        assert k.shape == v.shape == (11, 2, 64)
        assert ops.kv8_attention(q, *cache, cu, at, 3, None).shape == q.shape
