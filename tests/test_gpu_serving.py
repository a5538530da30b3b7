"""8-bit serving operators against 64-bit references, on a B200.

Bounds (u = the 16-bit type's relative rounding error, 2^-11 for fp16 and 2^-8 for bf16):
* a rotated value is one 16-bit rounding of a sum whose fp32 error is at most 2^-22 of its terms;
* a cached value is within half a step of its 16-bit value, and a 16-bit rounding of that;
* an attention weight p carries a relative error of 2^-11 (its own fp16 rounding) + 2^-20 (exponential, fp32
  sums) + twice the error of its score, (D + 8) 2^-24 of the score's absolute terms; so an output is off by
  at most that times sum p |v|, and its own rounding;
* a linear output is exact in int32, then at most six fp32 roundings; GELU adds 2^-18 (absolute, and relative
  for large values).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def sv(tt):
    return tt.serving


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts(counts):
    return i32([0] + torch.tensor(counts).cumsum(0).tolist())


class Model:
    """A cache and, beside it, the 16-bit keys and values that went in (sequence by sequence)."""

    def __init__(self, sv, batch, kv, dim, page, most, dtype, seed=0, rows=False, pages=None):
        self.g = torch.Generator("cuda").manual_seed(seed)
        self.batch, self.kv, self.dim, self.page, self.dtype = batch, kv, dim, page, dtype
        wide = (most + page - 1) // page
        n = batch * wide
        pool = n if pages is None else pages
        self.table = (pool - 1 - torch.randperm(n, generator=self.g, device="cuda")).to(torch.int32).view(batch, wide)
        r = i32(list(range(batch + 2, 2, -1))) if rows else None
        self.c = sv.PagedKV8.allocate(pool, kv, page, dim, self.table, newest_rows=batch + 3, rows=r, dtype=dtype)
        for t in self.c.tensors[:6]:
            t.fill_(255 if t.dtype == torch.uint8 else float("nan"))  # what was never written must not matter
        self.k = [torch.empty(0, kv, dim, dtype=dtype, device="cuda") for _ in range(batch)]
        self.v = [x.clone() for x in self.k]

    @property
    def lens(self):
        return [x.shape[0] for x in self.k]

    def rows(self, n, width):
        x = torch.randn(n, width, generator=self.g, device="cuda")
        x[:, :: 17] *= 5
        return x.to(self.dtype)

    def append(self, counts, heads, cos=None, sin=None, interleaved=False, qkv=None, start=None):
        width = (heads + 2 * self.kv) * self.dim
        qkv = self.rows(sum(counts), width) if qkv is None else qkv
        start = self.lens if start is None else start
        q = self.c.append(qkv, starts(counts), i32(start), heads=heads, cos=cos, sin=sin, interleaved=interleaved)
        at, want = 0, []
        for b, n in enumerate(counts):
            x = qkv[at:at + n].reshape(n, heads + 2 * self.kv, self.dim)
            at += n
            qk, err = rotate64(x[:, :heads + self.kv], range(start[b], start[b] + n), cos, sin, interleaved)
            want.append((qk[:, :heads], err[:, :heads]))
            k = qk[:, heads:].to(self.dtype)
            if cos is not None:  # fp32 before the 16-bit rounding: take the stored rounding, checked by its bound
                k = rotate32(x[:, heads:heads + self.kv], range(start[b], start[b] + n), cos, sin, interleaved).to(self.dtype)
                close(k, qk[:, heads:], err[:, heads:] + U[self.dtype] * qk[:, heads:].abs() + 2.0 ** -25)
            self.k[b] = torch.cat([self.k[b][:start[b]], k])
            self.v[b] = torch.cat([self.v[b][:start[b]], x[:, heads + self.kv:]])
        ref, err = torch.cat([w[0] for w in want]), torch.cat([w[1] for w in want])
        close(q, ref, err + U[self.dtype] * ref.abs() + 2.0 ** -25)
        return q

    def seen(self, b, which):
        """What the cache stands for, 64 bits: whole blocks by their codes, the rest in 16 bits."""
        x = (self.k, self.v)[which][b]
        whole = x.shape[0] // self.page * self.page
        y = x[:whole].view(-1, self.page, self.kv, self.dim).float()
        scale = y.abs().amax((1, 3), keepdim=True) * (1 / 127)
        codes = torch.where(scale > 0, y / scale, 0).round()
        return torch.cat([(codes.double() * scale.double()).view(whole, self.kv, self.dim), x[whole:].double()])

    def check_read(self):
        lens = self.lens
        k, v = self.c.read(starts(lens), i32([0] * self.batch), i32(lens), total=sum(lens))
        at = 0
        for b, n in enumerate(lens):
            for got, which in ((k, 0), (v, 1)):
                want, src = self.seen(b, which), (self.k, self.v)[which][b]
                part = got[at:at + n]
                whole = n // self.page * self.page
                assert torch.equal(part[whole:], src[whole:])
                assert torch.equal(part[:whole], want[:whole].float().to(self.dtype))  # fp32 product, one rounding
                step = src[:whole].double().view(-1, self.page, self.kv, self.dim).abs().amax((1, 3), keepdim=True) / 127
                off = (part[:whole].double() - src[:whole].double()).abs().view(-1, self.page, self.kv, self.dim)
                assert bool((off <= step * (0.5 + 1e-5) + 127.5 * step * U[self.dtype] + 2.0 ** -24).all())
            at += n

    def check_attend(self, q, counts, heads, scale=None):
        out = self.c.attend(q, starts(counts), i32(self.lens), max_q_len=max(counts), scale=scale)
        self.compare(out, q, counts, heads, scale)
        return out

    def compare(self, out, q, counts, heads, scale=None):
        g, at = heads // self.kv, 0
        sc = 1 / math.sqrt(self.dim) if scale is None else scale
        for b, n in enumerate(counts):
            length = self.lens[b]
            k, v = self.seen(b, 0), self.seen(b, 1)
            for i0 in range(0, n, 128):
                i1 = min(n, i0 + 128)
                x = q[at + i0:at + i1].double().view(i1 - i0, self.kv, g, self.dim)
                w = torch.einsum("qhgd,khd->qhgk", x, k) * sc
                size = torch.einsum("qhgd,khd->qhgk", x.abs(), k.abs()) * sc
                pos = length - n + torch.arange(i0, i1, device="cuda")
                hide = torch.arange(length, device="cuda") > pos[:, None]
                w = w.masked_fill(hide[:, None, None], -math.inf)
                p = torch.where((pos >= 0)[:, None, None, None], torch.softmax(w, -1), 0) if length else w
                ref = torch.einsum("qhgk,khd->qhgd", p, v).reshape(i1 - i0, heads, self.dim)
                eps = 2.0 ** -11 + 2.0 ** -20 + 2 * (self.dim + 8) * 2.0 ** -24 * size.masked_fill(hide[:, None, None], 0).amax(
                    -1, keepdim=True) if length else torch.zeros_like(w)
                # the error of a weight also moves the sum it is divided by: twice
                err = torch.einsum("qhgk,khd->qhgd", 2 * eps * p, v.abs()).reshape(ref.shape)
                close(out[at + i0:at + i1], ref, err + U[self.dtype] * ref.abs() + 2.0 ** -25)
            at += n


def rotate64(x, positions, cos, sin, interleaved):
    """x [n, heads, d] -> the rotation in 64 bits and what fp32 may be off by."""
    x = x.double()
    if cos is None:
        return x, torch.zeros_like(x)
    at = torch.tensor(list(positions), dtype=torch.long, device="cuda")
    c, s = cos[at].double()[:, None], sin[at].double()[:, None]
    return _turn(x, c, s, interleaved), _turn(x.abs(), c.abs(), s.abs(), interleaved, True) * 2.0 ** -22


def rotate32(x, positions, cos, sin, interleaved):
    at = torch.tensor(list(positions), dtype=torch.long, device="cuda")
    return _turn(x.float(), cos[at][:, None], sin[at][:, None], interleaved)


def _turn(x, c, s, interleaved, plus=False):
    r, half = 2 * c.shape[-1], c.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :half], x[..., half:r])
    ya, yb = (a * c + b * s if plus else a * c - b * s), b * c + a * s
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., r:]], -1)


def close(got, want, bound):
    got = got.double()
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (int(bad.sum()), off[bad].max().item(), bound[bad].min().item())


def turns(n, rot):
    t = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    return t.cos().float(), t.sin().float()


# ------------------------------------------------------------------ append and read
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("page,dim,kv,group,rot,inter", [(16, 64, 2, 3, 32, False), (32, 128, 1, 4, 128, True),
                                                          (64, 32, 4, 1, 16, False), (128, 128, 2, 1, 128, False),
                                                          (16, 32, 1, 8, 0, False), (64, 64, 3, 2, 64, True)])
def test_append_read(sv, pkg, page, dim, kv, group, rot, inter, dtype):
    m = Model(sv, 5, kv, dim, page, 6 * page, dtype, rows=True)
    cos, sin = turns(6 * page, rot) if rot else (None, None)
    for counts in ([1, 0, page, 2 * page + 1, page - 1], [1, 3, 1, page, 1], [0, 0, 0, 0, 1], [2 * page - 2, page + 5, 1, 1, 7],
                   [1, 1, 1, 1, 1]):
        m.append(counts, kv * group, cos, sin, inter)
        m.check_read()
    assert pkg.runtime.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_cache_does_not_depend_on_the_split(sv, dtype):
    """All at once, token by token, or in pieces that cross blocks (a kept block then takes the slot of the
    block whose earlier tokens are still needed): the same bytes."""
    page, dim, kv, n = 16, 64, 2, 16 * 9 + 5
    cos, sin = turns(256, 64)
    states = []
    for pieces in ([n], [1] * n, [10, 40, n - 50], [15, 33, 34, n - 82], [7, 95, n - 102]):
        m = Model(sv, 2, kv, dim, page, 256, dtype, seed=3)
        full = m.rows(2 * n, (kv + 2 * kv) * dim).view(2, n, -1)
        at = 0
        for c in pieces:
            m.append([c, c], kv, cos, sin, qkv=full[:, at:at + c].reshape(2 * c, -1))
            at += c
        m.check_read()
        blocks = n // page
        used = m.table[:, :blocks].long()
        states.append([t[used] for t in m.c.tensors[:4]])
        # the newest blocks' values up to the last token
        last = m.c.tensors[4][:2, blocks % 2, :, :n % page]
        states[-1].append(last)
    for other in states[1:]:
        for a, b in zip(states[0], other):
            assert torch.equal(a, b)


def test_rewind(sv):
    """Drafted tokens that were refused: the next append starts earlier, in the block before the last."""
    m = Model(sv, 1, 2, 64, 16, 128, torch.float16)
    m.append([30], 2)
    m.append([5], 2)  # 35 tokens: block 1 is whole
    m.k[0], m.v[0] = m.k[0][:29], m.v[0][:29]
    m.check_read()
    m.append([6], 2)
    m.check_read()
    q = m.append([1], 2)
    m.check_attend(q, [1], 2)


def test_append_strided_rows_and_other_stream(sv):
    m = Model(sv, 3, 2, 64, 32, 128, torch.float16)
    wide = torch.randn(3 * 40, 6 * 64 + 72, device="cuda", dtype=torch.float16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q = m.append([40, 40, 40], 2, qkv=wide[:, 8:8 + 6 * 64])
        m.check_read()
        m.check_attend(q, [40] * 3, 2)
    torch.cuda.current_stream().wait_stream(s)


def test_block_with_nan_reads_as_nan(sv):
    """A block that holds an infinity or NaN is NaN as a whole, and rows that see none of it are not touched."""
    for bad in (float("nan"), float("inf")):
        m = Model(sv, 1, 1, 64, 16, 64, torch.bfloat16)
        x = m.rows(40, 3 * 64)
        x[20, 128 + 5] = bad  # a value channel of token 20: block 1
        c = m.c
        q = c.append(x, starts([40]), i32([0]), heads=1)
        k, v = c.read(starts([40]), i32([0]), i32([40]), total=40)
        assert bool(v[16:32].isnan().all()) and not bool(v[:16].isnan().any()) and not bool(v[32:].isnan().any())
        assert not bool(k.isnan().any())
        out = c.attend(q, starts([40]), i32([40]), max_q_len=40)
        assert not bool(out[:16].isnan().any()) and bool(out[16:].isnan().all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_nan_in_the_newest_block_stays_with_the_rows_that_see_it(sv, dtype):
    m = Model(sv, 1, 1, 64, 64, 64, dtype)
    x = m.rows(50, 3 * 64)
    clean = x.clone()
    x[33, 128:192] = float("inf")
    x[41, 64:128] = float("nan")  # a key
    q = m.c.append(x, starts([50]), i32([0]), heads=1)
    out = m.c.attend(q, starts([50]), i32([50]), max_q_len=50)
    m.append([50], 1, qkv=clean, start=[0])
    want = m.c.attend(q, starts([50]), i32([50]), max_q_len=50)
    assert torch.equal(out[:33], want[:33])
    assert bool(out[33:41].isinf().all()) and bool(out[41:].isnan().all())


# ------------------------------------------------------------------ attention
CASES = [  # page, dim, kv, group, lens before, new tokens
    (16, 64, 2, 1, [0, 1, 15, 16, 17, 33, 500], [1] * 7),
    (32, 128, 2, 4, [0, 31, 32, 63, 64, 1000], [1] * 6),
    (64, 32, 4, 3, [5, 63, 64, 127, 700], [1] * 5),
    (128, 128, 1, 8, [3000, 0, 127, 128], [1] * 4),
    (64, 64, 16, 1, [1000], [1]),
    (16, 64, 4, 6, [0, 7, 100, 333], [5, 4, 3, 5]),           # drafted tokens
    (32, 128, 2, 5, [0, 31, 90], [16, 2, 9]),
    (64, 32, 2, 2, [0, 64, 100], [37, 64, 129]),              # chunks of prompts
    (128, 128, 1, 3, [0, 200], [300, 77]),
    (64, 64, 2, 1, [0, 700, 65], [513, 0, 300]),              # a sequence without new tokens
    (16, 32, 1, 1, [2, 0], [0, 1]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attend(sv, pkg, case, dtype):
    page, dim, kv, group, before, new = CASES[case]
    most = max(a + b for a, b in zip(before, new))
    m = Model(sv, len(before), kv, dim, page, most, dtype, seed=case, rows=case % 2 == 1)
    if sum(before):
        m.append(before, kv * group)
    q = m.append(new, kv * group)
    a = m.check_attend(q, new, kv * group)
    b = m.check_attend(q, new, kv * group)
    assert torch.equal(a, b)  # no atomics, a fixed order
    assert pkg.runtime.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attend_in_a_wide_table(sv, case, dtype):
    """The same where the table could hold long sequences: the work is then one line cut among all warps."""
    page, dim, kv, group, before, new = CASES[case]
    m = Model(sv, len(before), kv, dim, page, 9000, dtype, seed=case + 20, rows=case % 2 == 0)
    if sum(before):
        m.append(before, kv * group)
    q = m.append(new, kv * group)
    a = m.check_attend(q, new, kv * group)
    assert torch.equal(a, m.check_attend(q, new, kv * group))


def test_attend_ragged_in_a_wide_table(sv):
    """Many sequences, short and long: pieces that hold ends and starts of several."""
    m = Model(sv, 40, 4, 64, 16, 5000, torch.float16, seed=4)
    before = [(i * 997) % 1300 if i % 3 else i for i in range(39)] + [4990]
    m.append(before, 8)
    q = m.append([1 + i % 3 for i in range(40)], 8)
    m.check_attend(q, [1 + i % 3 for i in range(40)], 8)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_attend_long(sv, dtype):
    """A long sequence beside short ones: its keys are cut among many warps."""
    m = Model(sv, 3, 2, 64, 64, 40000, dtype)
    m.append([39990, 70, 3], 4)
    q = m.append([1, 1, 1], 4)
    m.check_attend(q, [1, 1, 1], 4)


def test_attend_many_chunks_of_rows(sv):
    """Prompts of several sequences, and one new token beside them."""
    m = Model(sv, 4, 8, 64, 64, 2500, torch.float16)
    m.append([0, 100, 1200, 64], 16)
    q = m.append([2500, 1500, 1300, 1], 16)
    m.check_attend(q, [2500, 1500, 1300, 1], 16)


PROMPTS = [  # page, dim, kv, group, lens before, new tokens: about as many rows as the 256-row kernel takes, and more
    (64, 64, 8, 1, [0, 129], [640, 257]),
    (128, 128, 4, 2, [1000, 0], [300, 511]),
    (16, 32, 8, 3, [7, 300], [401, 255]),
    (32, 128, 2, 5, [63], [301]),
    (16, 64, 16, 1, [0, 0, 33], [1, 385, 700]),
    (128, 32, 8, 8, [4000], [200]),
    (32, 64, 4, 4, [31, 500], [333, 0]),
    (64, 64, 8, 1, [0, 129], [1000, 513]),
    (128, 128, 4, 2, [1000, 0], [700, 511]),
    (32, 128, 2, 5, [63], [901]),
    (16, 64, 4, 4, [31, 500], [700, 0]),
    (64, 32, 16, 1, [0, 257], [900, 3]),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_attend_prompts(sv, pkg, case, dtype):
    page, dim, kv, group, before, new = PROMPTS[case]
    assert sum(new) * group // len(new) >= 128 and sum(new) * group * kv * dim >= 300000
    m = Model(sv, len(before), kv, dim, page, max(a + b for a, b in zip(before, new)), dtype, seed=50 + case)
    if sum(before):
        m.append(before, kv * group)
    q = m.append(new, kv * group)
    a = m.check_attend(q, new, kv * group)
    assert torch.equal(a, m.check_attend(q, new, kv * group))
    assert pkg.runtime.device_error() == 0


@pytest.mark.parametrize("kv", [8, 16])  # the warps' kernel, and the 256-row kernel
def test_prompt_rows_without_keys(sv, kv):
    """More new rows than cached tokens: the first rows see nothing."""
    m = Model(sv, 2, kv, 64, 16, 512, torch.float16)
    m.append([300, 0], kv)
    q = m.rows(1200, kv * 64).view(1200, kv, 64)
    out = m.check_attend(q, [600, 600], kv)
    assert not bool(out[:300].any()) and not bool(out[600:].any())


@pytest.mark.parametrize("kv", [8, 16])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_prompt_scales_far_apart(sv, dtype, kv):
    """Blocks of very different sizes and of zeros."""
    m = Model(sv, 1, kv, 64, 32, 1024, dtype)
    k, v = kv * 64, 2 * kv * 64
    x = m.rows(1000, 3 * kv * 64)
    x[:, v:] *= (torch.arange(1000, device="cuda") // 32 % 5).to(dtype)[:, None] * 0.25
    x[128:256, k:] *= 2 ** -6
    x[256:288, k:] = 0
    x[:32, v:] = 0
    x[990:, v:] *= 2 ** -5
    q = m.append([1000], kv, qkv=x)
    m.check_attend(q, [1000], kv)
    if dtype == torch.float16:
        m.check_attend(q, [1000], kv, scale=-0.05)  # a factor that is not positive


@pytest.mark.parametrize("kv", [8, 16])
def test_prompt_nan_stays_with_the_rows_that_see_it(sv, kv):
    m = Model(sv, 1, kv, 64, 64, 1024, torch.float16)
    k, v = kv * 64, 2 * kv * 64
    x = m.rows(1000, 3 * kv * 64)
    clean = x.clone()
    x[400, v + 7] = float("nan")  # a value of head 0: block 6 is NaN as a whole
    x[990, v + 70] = float("inf")  # a value of head 1 in the newest block
    x[980, k + 128] = float("nan")  # a key of head 2 in the newest block
    out = m.c.attend(m.c.append(x, starts([1000]), i32([0]), heads=kv), starts([1000]), i32([1000]), max_q_len=1000)
    q = m.append([1000], kv, qkv=clean, start=[0])
    want = m.check_attend(q, [1000], kv)
    assert torch.equal(out[:384, 0], want[:384, 0]) and bool(out[384:, 0].isnan().all())
    # (the channel it is in; the 256-row kernel gives NaN to all channels of a row that sees it)
    assert torch.equal(out[:990, 1], want[:990, 1]) and not bool(out[990:, 1, 6].isfinite().any())
    assert torch.equal(out[:980, 2], want[:980, 2]) and bool(out[980:, 2].isnan().all())
    assert torch.equal(out[:, 3:], want[:, 3:])


def test_rows_without_keys_are_zero(sv):
    """Queries of tokens before the sequence's first key (lens < new tokens), and an empty sequence."""
    m = Model(sv, 3, 1, 64, 16, 64, torch.float16)
    m.append([3, 0, 20], 2)
    q = m.rows(15, 2 * 64).view(15, 2, 64)
    out = m.check_attend(q, [5, 5, 5], 2)
    assert not bool(out[:2].any()) and not bool(out[5:10].any())


def test_scores_far_apart(sv):
    """Scores of thousands: the running maximum moves, single keys take all the weight; all-zero blocks and rows."""
    m = Model(sv, 1, 1, 64, 16, 256, torch.float16)
    x = m.rows(200, 3 * 64)
    x[:, :128] *= 20
    x[48:64, 64:] = 0      # a block of zeros: scale 0
    x[150, :64] = 0
    q = m.append([200], 1, qkv=x)
    m.check_attend(q, [200], 1)


def test_bf16_rows_of_any_size(sv):
    """bf16 rows far outside fp16's range."""
    m = Model(sv, 1, 1, 64, 16, 64, torch.bfloat16)
    m.append([50], 1)
    q = m.rows(50, 64).view(50, 1, 64) * torch.tensor([1e-30, 1e30, 1.0, 1e5, 1e-6], device="cuda").repeat(10)[:, None, None]
    q = q.to(torch.bfloat16)
    for i, scale in ((0, 1e29), (1, 1e-31), (2, 0.125), (3, 1e-6), (4, 1e5)):
        pick = torch.zeros_like(q)
        pick[i::5] = q[i::5]
        m.check_attend(pick, [50], 1, scale=scale)


def test_attend_strided_rows(sv):
    m = Model(sv, 2, 2, 32, 32, 128, torch.float16)
    m.append([100, 50], 4)
    wide = torch.randn(4, 4 * 32 + 40, device="cuda", dtype=torch.float16)
    q = wide[:, 16:16 + 128].view(4, 4, 32)
    out = torch.zeros(4, 4 * 32 + 24, device="cuda", dtype=torch.float16)
    m.c.attend(q, starts([2, 2]), i32(m.lens), max_q_len=2, out=out[:, :128].view(4, 4, 32))
    m.compare(out[:, :128].reshape(4, 4, 32), q, [2, 2], 4)
    assert not bool(out[:, 128:].any())


def test_pages_beyond_31_bits(sv):
    """A pool whose byte offsets pass 2^31."""
    m = Model(sv, 1, 8, 128, 128, 700, torch.float16, pages=2 ** 31 // (128 * 8 * 128) + 9)
    m.append([640], 8)
    q = m.append([2], 8)
    m.check_read()
    m.check_attend(q, [2], 8)


def test_bad_indices_are_reported_not_followed(sv, pkg):
    m = Model(sv, 1, 1, 32, 16, 64, torch.float16)
    m.append([40], 1)
    q = m.rows(1, 32).view(1, 1, 32)
    assert pkg.runtime.device_error() == 0
    m.table[0, 1] = 10 ** 6
    m.c.attend(q, starts([1]), i32([40]), max_q_len=1)
    assert pkg.runtime.device_error() == 7
    m.c.read(starts([40]), i32([0]), i32([40]), total=40)
    assert pkg.runtime.device_error() == 7
    m.c.attend(q, starts([1]), i32([10 ** 6]), max_q_len=1)  # longer than the table
    assert pkg.runtime.device_error() == 7
    m.c.append(m.rows(1, 96), starts([1]), i32([64]), heads=1)  # past the table
    assert pkg.runtime.device_error() == 7
    cos, sin = turns(4, 32)
    m.c.append(m.rows(1, 96), starts([1]), i32([5]), heads=1, cos=cos, sin=sin)  # past the rotation table
    assert pkg.runtime.device_error() == 7


def test_graph_replays_with_other_lengths(sv):
    m = Model(sv, 2, 2, 64, 16, 512, torch.float16)
    m.append([100, 30], 4)
    qkv, start, lens = m.rows(2, 8 * 64), i32([0, 0]), i32([0, 0])
    cu = starts([1, 1])
    start.copy_(i32([100, 30]))
    lens.copy_(i32([101, 31]))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        m.c.attend(m.c.append(qkv, cu, start, heads=4), cu, lens, max_q_len=1)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = m.c.append(qkv, cu, start, heads=4)
        out = m.c.attend(q, cu, lens, max_q_len=1)
    for _ in range(40):
        qkv.copy_(m.rows(2, 8 * 64))
        start.copy_(i32(m.lens))
        lens.copy_(i32([n + 1 for n in m.lens]))
        graph.replay()
        for b in range(2):
            x = qkv[b:b + 1].view(1, 8, 64)
            m.k[b], m.v[b] = torch.cat([m.k[b], x[:, 4:6]]), torch.cat([m.v[b], x[:, 6:]])
    m.compare(out, q, [1, 1], 4)
    m.check_read()


# ------------------------------------------------------------------ int8 linear
def rule(x):
    """The quantization rule: fp32 scale, codes, and the 64-bit check that they are the nearest."""
    top = x.float().abs().amax(1, keepdim=True)
    scale = top * (1 / 127)
    codes = torch.where(scale > 0, x.float() / scale, 0).round().clamp(-127, 127)
    assert bool(((codes.double() * scale.double() - x.double()).abs() <= scale.double() * (0.5 + 2e-5)).all())
    return codes.double(), scale.double()


@pytest.mark.parametrize("epi", ["bias", "none", "gelu", "resid"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (1, 1, 1), (3, 17, 5), (7, 130, 33), (64, 512, 200), (129, 128, 256),
                                   (200, 1001, 130), (300, 640, 513), (1, 4096, 1024), (17, 2048, 96), (1000, 96, 1030)])
def test_linear(sv, pkg, m, k, n, dtype, epi):
    g = torch.Generator("cuda").manual_seed(m + k + n)
    x = torch.randn(m, k, generator=g, device="cuda") * 3
    x[:, ::5] *= 9
    x[m // 2] *= 0 if m > 1 else 1
    x = x.to(dtype)
    w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
    codes, scale = sv.quantize_weight(w)
    wc, ws = rule(w)
    assert torch.equal(codes[:, :k].double(), wc) and torch.equal(scale.double(), ws[:, 0])
    assert not bool(codes[:, k:].any())
    codes[:, k:] = 77  # what pads a row must not matter
    bias = None if epi == "none" else torch.randn(n, generator=g, device="cuda")
    resid = torch.randn(m, n, generator=g, device="cuda") if epi == "resid" else None
    xc, xs = rule(x)
    y = sv.linear_int8(x, codes, scale, bias, gelu=epi == "gelu", resid=resid)
    part = (xc @ wc.T) * xs * ws.T
    size = part.abs()
    if bias is not None:
        part, size = part + bias.double(), size + bias.abs().double()
    bound = 6 * 2.0 ** -24 * size + 2.0 ** -40
    if epi == "gelu":
        part = torch.nn.functional.gelu(part)
        bound = 1.2 * bound + 2.0 ** -18 * (1 + part.abs())  # |gelu'| < 1.13
    if epi == "resid":
        part = part + resid.double()
        bound = bound + 2.0 ** -24 * part.abs()
    assert y.dtype == (torch.float32 if epi == "resid" else dtype)
    close(y, part, bound + U[y.dtype] * part.abs() + (2.0 ** -25 if y.dtype != torch.float32 else 0))
    assert pkg.runtime.device_error() == 0


def test_linear_in_place_strided_and_types(sv):
    g = torch.Generator("cuda").manual_seed(1)
    wide = torch.randn(70, 300, generator=g, device="cuda").half()
    x = wide[:, 3:203]  # rows that start on odd addresses
    w, ws = sv.quantize_weight(torch.randn(72, 200, generator=g, device="cuda"))
    want = sv.linear_int8(x.contiguous(), w, ws, out_dtype=torch.float32)
    assert torch.equal(sv.linear_int8(x, w, ws, out_dtype=torch.float32), want)
    assert torch.equal(sv.linear_int8(x, w, ws, out_dtype=torch.bfloat16), want.bfloat16())
    out = torch.zeros(70, 80, device="cuda")
    sv.linear_int8(x, w, ws, out_dtype=torch.float32, out=out[:, 1:73])  # rows that start off 16 bytes
    assert torch.equal(out[:, 1:73], want) and not bool(out[:, 0].any()) and not bool(out[:, 73:].any())
    res = torch.randn(70, 72, generator=g, device="cuda")
    there = res.clone()
    assert sv.linear_int8(x, w, ws, resid=there, out=there) is there
    assert torch.equal(there, sv.linear_int8(x, w, ws, resid=res))


def test_linear_rows_with_nan_are_nan(sv):
    w, ws = sv.quantize_weight(torch.randn(40, 64, device="cuda"))
    x = torch.randn(9, 64, device="cuda")
    x[2, 3], x[5, 60] = float("nan"), -float("inf")
    y = sv.linear_int8(x, w, ws)
    bad = y.isnan()
    assert bool(bad[2].all()) and bool(bad[5].all()) and int(bad.sum()) == 80


# ------------------------------------------------------------------ together
def test_decoder_follows_the_model(sv, tt):
    """Prompt, single tokens and drafted ones against the fp32-accurate forward of the whole sequence.  8-bit
    weights, activations and cache: each product's error is about 1 % of its result (a step of amax / 127 at
    amax of about four deviations is 0.9 %, of both operands), less after the residual; 5 % of the normalised
    output covers two layers of four products and the cache."""
    cfg = tt.TransformerConfig(2, 100, 256, 4, 512, 2, True)
    torch.manual_seed(5)
    model = tt.UserOptimizedTransformer(cfg).cuda().eval()
    x = torch.randn(2, 100, 256, device="cuda")
    with torch.inference_mode():
        want = model(x)
        dec = sv.Int8Decoder(model, max_sequences=3, max_tokens=128, page_size=16)
        a, b = dec.open(), dec.open()
        got = [[], []]

        def step(na, nb):
            at = [sum(t.shape[0] for t in g) for g in got]
            y = dec.forward(torch.cat([x[0, at[0]:at[0] + na], x[1, at[1]:at[1] + nb]]), [a, b], [na, nb])
            got[0].append(y[:na])
            got[1].append(y[na:])

        step(60, 0)
        step(1, 77)
        for _ in range(5):
            step(1, 1)
        # drafted tokens, refused, and again
        dec.forward(torch.randn(6, 256, device="cuda"), [a, b], [3, 3])
        dec.rewind(a, 3)
        dec.rewind(b, 3)
        step(34, 18)
        for i in range(2):
            y = torch.cat(got[i])
            assert y.shape == (100, 256)
            rel = ((y - want[i]).norm() / want[i].norm()).item()
            assert rel < 0.05, rel
        dec.close(a)
        c = dec.open()
        assert c == a
        y = dec.forward(x[0, :10].contiguous(), [c], [10])
        assert ((y - want[0, :10]).norm() / want[0, :10].norm()).item() < 0.05


def test_ops_compiled_match_the_calls(sv):
    """A step written with torch.ops.b200, compiled with fullgraph=True, equals the calls."""
    m, n = (Model(sv, 2, 2, 64, 16, 64, torch.float16, seed=9) for _ in range(2))
    x = torch.randn(6, 128, device="cuda").half()
    w, ws = sv.quantize_weight(torch.randn(8 * 64, 128, device="cuda") / 11)
    cu, start, lens = starts([3, 3]), i32([0, 0]), i32([3, 3])
    ops = torch.ops.b200

    def step(x):
        qkv = ops.linear_int8(x, w, ws, None, False, None, False)
        q = ops.kv8_append(qkv, *m.c.tensors, cu, start, 4, None, None, False)
        return ops.kv8_attention(q, *m.c.tensors, cu, lens, 3, None), *ops.kv8_read(*m.c.tensors, cu, start, lens, 6)

    got = torch.compile(step, fullgraph=True)(x)
    q = n.c.append(sv.linear_int8(x, w, ws), cu, start, heads=4)
    want = (n.c.attend(q, cu, lens, max_q_len=3), *n.c.read(cu, start, lens, total=6))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ refusals
def test_refusals(sv):
    m = Model(sv, 2, 2, 64, 16, 64, torch.float16)
    c, cu, at = m.c, starts([1, 1]), i32([0, 0])
    x = m.rows(2, 6 * 64)
    q = x[:, :128].reshape(2, 2, 64)
    cos, sin = turns(64, 64)
    for bad in (lambda: c.append(x.bfloat16(), cu, at, heads=2), lambda: c.append(x, cu, at, heads=3),
                lambda: c.append(x, cu.long(), at, heads=2), lambda: c.append(x, cu[:2], at, heads=2),
                lambda: c.append(x, cu, at, heads=2, cos=cos), lambda: c.append(x, cu, at, heads=2, cos=cos[:, :4].contiguous(), sin=sin[:, :4].contiguous()),
                lambda: c.attend(q.float(), cu, at, max_q_len=1), lambda: c.attend(q[:, :1].expand(2, 3, 64), cu, at, max_q_len=1),
                lambda: c.attend(q, cu, at, max_q_len=0), lambda: c.attend(q, cu, at, max_q_len=1, out=q[:1]),
                lambda: c.read(cu, at, at, total=-1),
                lambda: sv.PagedKV8.allocate(4, 2, 24, 64, m.table), lambda: sv.PagedKV8.allocate(4, 2, 16, 80, m.table),
                lambda: sv.PagedKV8.allocate(4, 2, 16, 64, m.table.long()),
                lambda: sv.PagedKV8.allocate(4, 2, 16, 64, m.table, newest_rows=1)):
        with pytest.raises(ValueError):
            bad()
    w, ws = sv.quantize_weight(torch.randn(8, 64, device="cuda"))
    y = torch.randn(2, 64, device="cuda")
    for bad in (lambda: sv.linear_int8(y[:, :40], w, ws), lambda: sv.linear_int8(y.double(), w, ws),
                lambda: sv.linear_int8(y, w.float(), ws), lambda: sv.linear_int8(y, w, ws[:3]),
                lambda: sv.linear_int8(y, w, ws, gelu=True, resid=torch.zeros(2, 8, device="cuda")),
                lambda: sv.linear_int8(y, w, ws, resid=torch.zeros(2, 8, device="cuda"), out_dtype=torch.float16),
                lambda: sv.linear_int8(y, w, ws, out=torch.zeros(2, 9, device="cuda")),
                lambda: sv.linear_int8(torch.randn(65, 2, device="cuda").t(), w, ws)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        sv.linear_int8(y.cpu(), w, ws)
    with pytest.raises(RuntimeError):
        c.attend(q.cpu(), cu, at, max_q_len=1)
