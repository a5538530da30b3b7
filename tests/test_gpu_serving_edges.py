"""Corners of the 8-bit serving operators, on a B200: sequences shortened more than once, values and scales at the
ends of their ranges, arguments that overlap or wrap, shapes that take the kernels' longer paths."""

import math

import pytest
import torch

from test_gpu_serving import U, Model, close, i32, starts

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sv(tt):
    return tt.serving


# ------------------------------------------------------------------ shortened sequences
def test_decoder_rewound_twice(sv, tt):
    """What is left after two rewinds across a block is what a fresh sequence of those tokens holds: the kept tokens
    are 16-bit values or codes made from them, so the outputs that follow are the same bits; further back is refused."""
    cfg = tt.TransformerConfig(1, 64, 128, 2, 256, 1, True)
    torch.manual_seed(3)
    model = tt.UserOptimizedTransformer(cfg).cuda().eval()
    x = torch.randn(64, 128, device="cuda")
    with torch.inference_mode():
        dec = sv.Int8Decoder(model, max_sequences=2, max_tokens=64, page_size=16)
        a, b = dec.open(), dec.open()
        dec.forward(x[:48], [a], [48])                     # blocks 1 and 2 are kept
        dec.forward(torch.randn(1, 128, device="cuda"), [a], [1])  # and now 2 and 3
        dec.rewind(a, 1)
        for n in (17, 30):
            with pytest.raises(ValueError):
                dec.rewind(a, n)
        dec.rewind(a, 10)  # 38 tokens
        with pytest.raises(ValueError):
            dec.rewind(a, 7)
        dec.forward(x[:38], [b], [38])
        y = dec.forward(torch.cat([x[38:41], x[38:41]]), [a, b], [3, 3])
        assert torch.equal(y[:3], y[3:])


# ------------------------------------------------------------------ attention: values of very different sizes
def compare(m, out, q, counts, heads, far):
    """out against 64 bits.  A weight's relative error is test_gpu_serving's, and where V scales lie far from 1
    (2^-125 .. 2^125: their logarithms are below 128, known to 2^-17, and enter two sums and a difference that round
    alike) 4 * 2^-17 * ln 2 < 2^-15 more.  Weights carry V's scale and are held in fp16 times 2^14 of the largest:
    2^-39 of the largest (weight times the largest value of a block) a key.  No absolute allowance but the type's
    smallest step."""
    g, at, d = heads // m.kv, 0, m.dim
    for b, n in enumerate(counts):
        length = m.lens[b]
        k, v = m.seen(b, 0), m.seen(b, 1)
        top = torch.zeros(length, m.kv, dtype=torch.float64, device="cuda")
        for i in range(0, length, m.page):
            top[i:i + m.page] = v[i:i + m.page].abs().amax((0, 2))
        for i0 in range(0, n, 128):
            i1 = min(n, i0 + 128)
            x = q[at + i0:at + i1].double().view(i1 - i0, m.kv, g, d)
            hide = torch.arange(length, device="cuda") > (length - n + torch.arange(i0, i1, device="cuda"))[:, None]
            w = (torch.einsum("qhgd,khd->qhgk", x, k) / math.sqrt(d)).masked_fill(hide[:, None, None], -math.inf)
            size = torch.einsum("qhgd,khd->qhgk", x.abs(), k.abs()).masked_fill(hide[:, None, None], 0).amax(-1, keepdim=True) / math.sqrt(d)
            p = torch.softmax(w, -1)
            ref = torch.einsum("qhgk,khd->qhgd", p, v).reshape(i1 - i0, heads, d)
            eps = 2.0 ** -11 + 2.0 ** -20 + 2 * (d + 8) * 2.0 ** -24 * size + (2.0 ** -15 if far else 0)
            err = torch.einsum("qhgk,khd->qhgd", 2 * eps * p, v.abs()).reshape(ref.shape)
            low = length * 2.0 ** -39 * (p * top.T[None, :, None]).amax(-1).reshape(i1 - i0, heads, 1)
            step = 2.0 ** -24 if m.dtype == torch.float16 else 2.0 ** -133
            close(out[at + i0:at + i1], ref, err + low + U[m.dtype] * ref.abs() + step)
        at += n


@pytest.mark.parametrize("kv", [2, 16])  # the warps' kernel, and the 256-row kernel
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_many_values_of_zero_before_others(sv, pkg, dtype, kv):
    """40000 keys of about equal weight whose values are zero, then 700 others: the sum of the weights must stay in
    range, and the outputs are small averages."""
    m = Model(sv, 1, kv, 64, 128, 41000, dtype)
    k, v = kv * 64, 2 * kv * 64
    x = m.rows(40700, 3 * kv * 64)
    x[:, :v] *= 2 ** -4
    x[:40000, v:] = 0
    q = m.append([40700], kv, qkv=x)[40000:].contiguous()
    out = m.c.attend(q, starts([700]), i32([40700]), max_q_len=700)
    compare(m, out, q, [700], kv, False)
    assert pkg.runtime.device_error() == 0


@pytest.mark.parametrize("kv", [2, 16])
def test_values_of_any_size(sv, kv):
    """bf16 blocks of values from 2^-112 to 2^100, zeros between them and in the newest block: rows that see the small
    ones only, and rows that see them beside large ones."""
    sizes = [0, 2.0 ** -112, 2.0 ** -111, 0, 2.0 ** -60, 2.0 ** -38, 1.0, 0, 2.0 ** 50, 2.0 ** -30, 2.0 ** 100, 0]
    m = Model(sv, 1, kv, 64, 64, 1024, torch.bfloat16)
    v = 2 * kv * 64
    x = m.rows(64 * len(sizes) + 50, 3 * kv * 64)
    x[:, :v] *= 2 ** -3
    for i, f in enumerate(sizes):
        x[64 * i:64 * i + 64, v:] *= f
    x[-50:-25, v:] = 0
    x[-20:, v:] *= 2.0 ** 90
    n = x.shape[0]
    q = m.append([n], kv, qkv=x)
    for upto in (n, n - 22, 64 * 6, 64 * 5 + 3):  # (shortened: what is read must not depend on what came later)
        m.k[0], m.v[0] = m.k[0][:upto], m.v[0][:upto]
        if upto < 64 * (len(sizes) - 1):
            m = Model(sv, 1, kv, 64, 64, 1024, torch.bfloat16)
            m.append([upto], kv, qkv=x[:upto])
        out = m.c.attend(q[:upto].contiguous(), starts([upto]), i32([upto]), max_q_len=upto)
        compare(m, out, q[:upto], [upto], kv, True)


# ------------------------------------------------------------------ arguments
def test_one_row_whose_channels_are_strided_is_refused(sv):
    m = Model(sv, 1, 2, 64, 16, 64, torch.float16)
    wide = m.rows(1, 2 * 6 * 64)
    for strided in (wide[:, ::2], wide.view(6 * 64, 2).t()[:1]):
        assert strided.shape == (1, 6 * 64) and strided.stride(1) == 2
        with pytest.raises(ValueError):
            m.c.append(strided, starts([1]), i32([0]), heads=2)
    m.append([1], 2, qkv=wide[:, 8:8 + 6 * 64])  # a row of a wider buffer
    assert m.c.append(wide[:0, ::2], starts([0]), i32([1]), heads=2).shape == (0, 2, 64)
    m.check_read()


@pytest.mark.parametrize("cu", [[2 ** 31 - 1, -2, 3], [0, 8, 0], [-2 ** 31, 2 ** 31 - 1, 2 ** 31 - 1], [0, -1, 8], [0, 2 ** 31 - 1, -2 ** 31]])
@pytest.mark.parametrize("wide", [128, 9000, 100000])
def test_rows_that_wrap_or_decrease_are_reported_not_followed(sv, pkg, cu, wide):
    """cu whose differences leave 32 bits, or that decreases: no rows, the error word, and the cache as it was (but for the
    sequences whose own rows are in order, which append takes one by one)."""
    m = Model(sv, 2, 2, 64, 16, wide, torch.float16)
    m.append([40, 20], 2)
    before = [t.clone() for t in m.c.tensors[:6]]
    for n, most in ((8, 4), (8000, 4000)):
        heads = 2
        q = m.rows(n, heads * 64).view(n, heads, 64)
        out = torch.full_like(q, 7.0)
        assert pkg.runtime.device_error() == 0
        m.c.attend(q, i32(cu), i32([40, 20]), max_q_len=most, out=out)
        assert pkg.runtime.device_error() == 7 and bool((out == 7).all())
        m.c.append(m.rows(n, 6 * 64), i32(cu), i32([40, 20]), heads=2)
        assert pkg.runtime.device_error() == 7
        if cu == [0, 8, 0]:  # the first sequence's rows are as they should be: append stores them
            continue
        for t, was in zip(m.c.tensors[:6], before):
            assert torch.equal(t.view(torch.uint8), was.view(torch.uint8))


def test_starts_that_wrap_are_reported_not_followed(sv, pkg):
    m = Model(sv, 2, 2, 64, 16, 128, torch.float16)
    m.append([40, 20], 2)
    before = [t.clone() for t in m.c.tensors[:6]]
    for n in (1, 10, 300):
        for start in (2 ** 31 - 1, 2 ** 31 - 5, -1, -2 ** 31):
            m.c.append(m.rows(n, 6 * 64), starts([n, 0]), i32([start, 2 ** 31 - 1]), heads=2)
            assert pkg.runtime.device_error() == 7
            m.c.read(starts([n, 0]), i32([start, 0]), i32([40, 20]), total=n)
            assert pkg.runtime.device_error() == 7
    m.c.append(m.rows(3, 6 * 64), starts([0, 3]), i32([-1, 20]), heads=2)  # no new tokens: its start is not looked at
    assert pkg.runtime.device_error() == 0
    for t, was in zip(m.c.tensors[:4], before):
        assert torch.equal(t.view(torch.uint8), was.view(torch.uint8))


@pytest.mark.parametrize("dtype,code", [(torch.float16, 0), (torch.bfloat16, 1), (torch.float32, 2)])
@pytest.mark.parametrize("m,k", [(3, 1), (5, 17), (2, 100), (2100, 40), (2100, 1009), (7, 5000)])
def test_quantized_rows_leave_their_neighbours_alone(pkg, dtype, code, m, k):
    """Codes as a range of columns of a wider buffer: nothing beside them is written."""
    x = torch.randn(m, (k + 23) // 8 * 8, device="cuda").to(dtype)
    wide = torch.full((m, k + 48 - k % 16), 99, dtype=torch.int8, device="cuda")
    scale = torch.empty(m, device="cuda")
    rc = pkg.runtime.lib().b200_quantize_rows_i8(x.data_ptr(), code, x.shape[1], wide.data_ptr() + 16, wide.shape[1],
                                                 scale.data_ptr(), m, k, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    top = x[:, :k].float().abs().amax(1)
    assert torch.equal(scale, top * (1 / 127))
    assert torch.equal(wide[:, 16:16 + k].float(), (x[:, :k].float() / scale[:, None]).round())
    assert bool((wide[:, :16] == 99).all()) and bool((wide[:, 16 + k:] == 99).all())


def test_outputs_over_inputs(sv, pkg):
    """out may be q (attention) and resid (linear); what overlaps otherwise is refused, columns side by side are not."""
    refused = pkg.runtime.B200Error
    for kv, n, most in ((2, 3, 128), (2, 3, 9000), (16, 800, 1024)):  # the warps' two ways, the 256-row kernel
        for dtype in (torch.float16, torch.bfloat16):
            m = Model(sv, 1, kv, 64, 16, most, dtype)
            q = m.append([n + 90], 2 * kv)[90:].contiguous()
            want = m.c.attend(q, starts([n]), i32(m.lens), max_q_len=n)
            assert m.c.attend(q, starts([n]), i32(m.lens), max_q_len=n, out=q) is q and torch.equal(q, want)
            both = torch.zeros(n, 4 * kv * 64, dtype=dtype, device="cuda")
            left, right = (both[:, i:i + 2 * kv * 64].view(n, 2 * kv, 64) for i in (0, 2 * kv * 64))
            m.c.attend(left, starts([n]), i32(m.lens), max_q_len=n, out=right)
            with pytest.raises(refused):
                m.c.attend(q[1:], starts([n - 1]), i32(m.lens), max_q_len=n, out=q[:-1])
    qkv = m.rows(2, 6 * 16 * 64)
    with pytest.raises(refused):
        m.c.append(qkv[:1], starts([1]), i32(m.lens), heads=64, out=qkv[:1, :64 * 64].view(1, 64, 64))
    w, ws = sv.quantize_weight(torch.randn(64, 64, device="cuda"))
    for rows in (5, 100):
        x = torch.randn(rows, 128, device="cuda")
        y = x.clone()
        want = sv.linear_int8(x[:, :64], w, ws)
        sv.linear_int8(x[:, :64], w, ws, out=x[:, 64:])
        assert torch.equal(x[:, 64:], want) and torch.equal(x[:, :64], y[:, :64])
        with pytest.raises(refused):
            sv.linear_int8(x[:, :64], w, ws, out=x[:, :64])
        with pytest.raises(refused):
            sv.linear_int8(y[:, :64], w, ws, resid=x[:, :64], out=x[:, 4:68])


# ------------------------------------------------------------------ infinities and NaN
@pytest.mark.parametrize("kv", [2, 16])  # the warps' kernel, and the 256-row kernel
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("page", [16, 128])
def test_values_that_are_not_finite_stay_in_their_channel(sv, dtype, kv, page):
    """Infinities and NaN among the newest block's values: their channel of the rows that see them, nothing else."""
    n = 7 * 128 + 13
    m = Model(sv, 2, kv, 64, page, 1024, dtype)
    v = 2 * kv * 64
    x = m.rows(2 * n, 3 * kv * 64)
    x[:, :v] *= 2 ** -3   # (flat weights: none is 0, whose product with an infinity is NaN)
    clean = x.clone()
    x[n - 11, v + 7] = math.inf              # head 0
    x[n - 9, v + 9] = -math.inf
    x[n - 4, v + 7] = -math.inf              # inf and -inf: NaN
    x[n - 10, v + 64:v + 128] = math.nan     # head 1: all of a token's channels
    x[2 * n - 1, v + 5] = math.nan           # the other sequence's last token
    q = m.c.append(x, starts([n, n]), i32([0, 0]), heads=kv)
    out = m.c.attend(q, starts([n, n]), i32([n, n]), max_q_len=n)
    m.append([n, n], kv, qkv=clean, start=[0, 0])
    want = m.check_attend(q, [n, n], kv)
    bad = torch.zeros_like(out, dtype=torch.bool)
    assert bool((out[n - 11:n - 4, 0, 7] == math.inf).all()) and bool(out[n - 4:n, 0, 7].isnan().all())
    assert bool((out[n - 9:n, 0, 9] == -math.inf).all())
    assert bool(out[n - 10:n, 1].isnan().all()) and bool(out[2 * n - 1, 0, 5].isnan())
    bad[n - 11:n, 0, 7] = bad[n - 9:n, 0, 9] = bad[n - 10:n, 1] = bad[2 * n - 1, 0, 5] = True
    assert bool(out[~bad].isfinite().all())
    # elsewhere what the rows give without them, within the two calls' own errors (a token's power of two may differ):
    # 2^-10 of the average of |v|, which is below 6, and the rounding
    off = (out.double() - want.double()).abs()[~bad]
    assert bool((off <= 2 * (2.0 ** -10 * 6 + U[dtype] * want.double().abs()[~bad])).all())


# ------------------------------------------------------------------ int8 linear
def linear64(sv, m, k, n, dtype, seed, spread=3.0):
    """x, a quantized weight, and (round(x / sx) w) sx sw in 64 bits."""
    g = torch.Generator("cuda").manual_seed(seed)
    x = (torch.randn(m, k, generator=g, device="cuda") * spread).to(dtype)
    w, ws = sv.quantize_weight(torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k))
    xs = x.float().abs().amax(1, keepdim=True) * (1 / 127)
    xc = (x.float() / xs).round().clamp(-127, 127)
    return x, w, ws, (xc.double() @ w[:, :k].double().T) * xs.double() * ws.double()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [(1, 256, 512), (64, 512, 200), (100, 300, 130), (600, 256, 512), (520, 1152, 300)])
def test_gelu_of_fp32_results_is_exact_to_fp32(sv, m, k, n, dtype):
    """y is off by six fp32 roundings; erff by 2 ulp (2^-23 near 1), its argument by 2^-23 (which moves erf by less than
    that), 1 + erf by 2^-24 of at most 2, and two products by 2^-24 each: |y| / 2 * 3 * 2^-23 and 2^-23 of the result."""
    x, w, ws, part = linear64(sv, m, k, n, dtype, m + k)
    bias = torch.randn(n, device="cuda")
    y = sv.linear_int8(x, w, ws, bias, gelu=True, out_dtype=torch.float32)
    size = part.abs() + bias.abs().double()
    part = part + bias.double()
    ref = torch.nn.functional.gelu(part)
    close(y, ref, 1.13 * 6 * 2.0 ** -24 * size + 1.5 * 2.0 ** -23 * part.abs() + 2.0 ** -23 * ref.abs() + 2.0 ** -60)


# ------------------------------------------------------------------ attention: which kernel
@pytest.mark.parametrize("kv,group,new", [(16, 1, 1), (4, 3, 2), (8, 4, 30)])
def test_idle_slots_change_nothing(sv, kv, group, new):
    """A sequence among 31 that have no new tokens is attended to as it is alone: by the warps' kernel, whose work is
    cut alike then, so the bits are the same."""
    n = 3000
    alone = Model(sv, 1, kv, 64, 64, 9000, torch.float16, seed=1)
    among = Model(sv, 32, kv, 64, 64, 9000, torch.float16, seed=2)
    heads = kv * group
    x = alone.rows(n, (heads + 2 * kv) * 64)
    q = alone.append([n], heads, qkv=x)[n - new:].contiguous()
    counts = [0] * 32
    counts[17] = n
    among.append(counts, heads, qkv=x)
    counts[17] = new
    want = alone.check_attend(q, [new], heads)
    got = among.c.attend(q, starts(counts), i32(among.lens), max_q_len=new)
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [[1, 1, 0, 2], [40, 1, 300, 7]])
def test_attend_in_a_table_of_a_billion_positions(sv, pkg, new):
    m = Model(sv, 4, 16, 64, 64, 1024, torch.float16)
    m.append([700, 0, 64, 130], 16)
    q = m.append(new, 16)
    table = torch.zeros(4, 1 << 24, dtype=torch.int32, device="cuda")
    table[:, :m.table.shape[1]] = m.table
    m.c = sv.PagedKV8(*m.c.tensors[:6], table)
    m.check_attend(q, new, 16)
    assert pkg.runtime.device_error() == 0


# ------------------------------------------------------------------ the decoder and the host
def test_decoder_steps_do_not_wait_for_the_device(sv, tt):
    """No call of a step synchronises, new pages or not, and steps that are issued far ahead of the device give what
    steps one by one give (the host's buffers are not used again too early)."""
    cfg = tt.TransformerConfig(1, 64, 256, 4, 512, 2, True)
    torch.manual_seed(6)
    model = tt.UserOptimizedTransformer(cfg).cuda().eval()
    prompt = torch.randn(40, 256, device="cuda")
    outs = []
    with torch.inference_mode():
        for ahead in (False, True):
            dec = sv.Int8Decoder(model, max_sequences=3, max_tokens=160, page_size=16)
            a, b = dec.open(), dec.open()
            y = dec.forward(prompt, [a, b], [25, 15])
            dec.forward(y[:1].contiguous(), [a], [1])
            dec.rewind(a, 1)
            x = torch.stack([y[24], y[39]])
            got = []
            torch.cuda.synchronize()
            if ahead:
                torch.cuda._sleep(200_000_000)  # (0.1 s: the steps below are all issued meanwhile)
            torch.cuda.set_sync_debug_mode("error")
            try:
                for i in range(100):
                    x = dec.forward(x, [a, b], [1, 1])
                    got.append(x)
                    if not ahead:
                        torch.cuda.set_sync_debug_mode("default")
                        torch.cuda.synchronize()
                        torch.cuda.set_sync_debug_mode("error")
            finally:
                torch.cuda.set_sync_debug_mode("default")
            outs.append(torch.stack(got))
    assert torch.equal(*outs)


# ------------------------------------------------------------------ int8 linear: every lap of the rings
@pytest.mark.parametrize("epi", ["bias", "gelu", "resid"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [
    (2500, 700, 2100),    # CTA pairs: 90 tiles on 74 pairs, two laps of K's ring; 16 epilogue warps for GELU
    (5000, 1160, 2061),   # 180 tiles, a third for some pairs; 8 epilogue warps; rows of out off 16 bytes
    (700, 2300, 300),     # few tiles of a long K
    (511, 700, 10000),    # 128x128 tiles: 316 on 148 CTAs, a third for some
    (3000, 650, 250),     # 128x128 tiles of few columns
])
def test_linear_of_many_tiles(sv, pkg, m, k, n, dtype, epi):
    x, w, ws, part = linear64(sv, m, k, n, dtype, m + n)
    bias = torch.randn(n, device="cuda")
    resid = torch.randn(m, n, device="cuda") if epi == "resid" else None
    y = sv.linear_int8(x, w, ws, bias, gelu=epi == "gelu", resid=resid)
    bound = 6 * 2.0 ** -24 * (part.abs() + bias.abs().double())  # test_gpu_serving's bounds
    part = part + bias.double()
    if epi == "gelu":
        part = torch.nn.functional.gelu(part)
        bound = 1.2 * bound + 2.0 ** -18 * (1 + part.abs())
    if epi == "resid":
        part = part + resid.double()
        bound = bound + 2.0 ** -24 * part.abs()
    close(y, part, bound + 2.0 ** -40 + U[y.dtype] * part.abs() + (2.0 ** -25 if y.dtype != torch.float32 else 0))
    if epi == "resid":  # in place: the same bits
        assert torch.equal(sv.linear_int8(x, w, ws, bias, resid=resid, out=resid), y)
    assert pkg.runtime.device_error() == 0


@pytest.mark.parametrize("m,k,n", [(1, 9000, 130), (64, 8193, 64), (3, 20000, 17), (64, 8192, 200)])
def test_linear_of_few_rows_and_a_long_k(sv, m, k, n):
    """Few rows whose K the cluster's shared memory does not hold, and one that it just does."""
    x, w, ws, part = linear64(sv, m, k, n, torch.bfloat16, k)
    y = sv.linear_int8(x, w, ws, out_dtype=torch.float32)
    close(y, part, 6 * 2.0 ** -24 * part.abs() + 2.0 ** -40)


def test_linear_beyond_31_bits(sv):
    """An output whose offsets pass 2^31 elements, rows of x and of the residual that start beyond 2^31."""
    x, w, ws, part = linear64(sv, 300, 64, 20000, torch.float16, 1)
    big = x.repeat(400, 1)[:110000]
    y = sv.linear_int8(big, w, ws)
    assert y.numel() > 2 ** 31
    for at in (0, 107700, 109800 - 300):
        part_at = part.roll(-(at % 300), 0)[:300]
        close(y[at:at + 300], part_at, 6 * 2.0 ** -24 * part_at.abs() + U[torch.float16] * part_at.abs() + 2.0 ** -25)
    del y
    wide = torch.zeros(80, 2 ** 26, dtype=torch.float16, device="cuda")
    wide[:, -64:] = x[:80]
    for rows in (40, 80):
        y = sv.linear_int8(wide[:rows, -64:], w, ws)
        close(y, part[:rows], 6 * 2.0 ** -24 * part[:rows].abs() + U[torch.float16] * part[:rows].abs() + 2.0 ** -25)


# ------------------------------------------------------------------ the cache at its limits
def test_rows_beyond_31_bits(sv, pkg):
    """qkv, queries and outputs whose rows lie 2^26 elements apart."""
    m = Model(sv, 2, 2, 64, 16, 64, torch.float16)
    wide = torch.zeros(40, 2 ** 26, dtype=torch.float16, device="cuda")
    wide[:, 72:72 + 8 * 64] = m.rows(40, 8 * 64)
    q = m.append([22, 18], 4, qkv=wide[:, 72:72 + 8 * 64])
    m.check_read()
    wide[:, 1024:1024 + 256] = q.view(40, 256)
    far, out = (wide[:, i:i + 256].view(40, 4, 64) for i in (1024, 2048))
    m.c.attend(far, starts([22, 18]), i32(m.lens), max_q_len=22, out=out)
    m.compare(out, q, [22, 18], 4)
    assert pkg.runtime.device_error() == 0


@pytest.mark.parametrize("new", [1, 3])
def test_the_largest_batch(sv, pkg, new):
    m = Model(sv, 2048, 1, 32, 16, 48, torch.bfloat16)
    m.append([(i * 7) % 30 for i in range(2048)], 2)
    counts = [new if i % 5 else 0 for i in range(2048)]
    q = m.append(counts, 2)
    m.check_read()
    m.check_attend(q, counts, 2)
    assert pkg.runtime.device_error() == 0


@pytest.mark.parametrize("group,new,before", [(71, 1, 500), (40, 3, 77), (64, 300, 10), (128, 1, 3000)])
def test_many_query_heads_share_a_key_head(sv, pkg, group, new, before):
    m = Model(sv, 2, 1, 64, 32, 4096, torch.float16)
    m.append([before, 5], group)
    q = m.append([new, 1], group)
    m.check_attend(q, [new, 1], group)
    assert pkg.runtime.device_error() == 0
