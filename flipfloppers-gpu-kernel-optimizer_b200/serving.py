"""Decoding token by token in 8 bits.

* ``PagedKV8`` -- a paged key/value cache: whole blocks of tokens in 8 bits with one
  scale a block and key head, the newest two blocks of each sequence in 16 bits as
  well.  ``append`` rotates the queries and keys of new tokens by position and
  stores keys and values, ``attend`` is attention of the newest tokens over the
  cache (one token a sequence, several drafted ones, or a chunk of a prompt),
  ``read`` returns stored tokens as 16-bit rows;
* ``linear_int8`` -- rows quantized to 8 bits with a scale each, times an 8-bit
  weight with a scale a channel (``quantize_weight``), with bias, GELU or residual;
* ``Int8Decoder`` -- a block stack (``UserOptimizedTransformer``) served with them.

Everything runs on the current stream of the tensors' device, never synchronises
and raises on arguments the kernels do not take; there is no other implementation
behind it.  Row counts and lengths are device tensors (int32), so that a step can
be captured in a CUDA graph and replayed with other values in them.
"""

from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import runtime as rt

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MAX_BATCH = 2048


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


# The checks of a call cost as much as a small kernel runs: they compare first and put the message together
# only when one fails.
_raw_stream = torch._C._cuda_getCurrentRawStream
_f32, _i32 = torch.float32, torch.int32


def _stream(index: Optional[int], *ts: Optional[Tensor]) -> int:
    """The current stream of CUDA device ``index``, which every tensor must be on and which must be current."""
    for t in ts:
        if t is not None and (not t.is_cuda or t.get_device() != index):
            raise RuntimeError("libb200block kernels take CUDA tensors on one device only (no CPU fallback)")
    if index is None or index < 0 or torch._C._cuda_getDevice() != index:
        raise RuntimeError(f"tensors are on CUDA device {index}, which is not the current one (no CPU fallback)")
    return _raw_stream(index)


def _index(t: Tensor, n: int, name: str) -> int:
    """The address of an index tensor."""
    if t.dtype != _i32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 tensor with {n} entries expected")
    return t.data_ptr()


class PagedKV8:
    """An 8-bit paged key/value cache of ``batch`` sequences (page size P, D channels a head).

    ``k_pages`` uint8 [pages, kv_heads, P, D] and ``v_pages`` uint8 [pages, kv_heads, P/4, D, 4]
    hold codes c standing for (c - 128) * scale, ``k_scale`` / ``v_scale`` fp32
    [pages, kv_heads] the scale of each block and head.  ``k_newest`` [rows, 2, kv_heads, P, D]
    and ``v_newest`` [rows, 2, kv_heads, P/4, D, 4] (fp16 or bf16) hold the newest two blocks of
    each sequence, block j in slot j % 2; ``table`` int32 [batch, blocks] the page of each block,
    ``rows`` int32 [batch] (default 0, 1, ..) the row of each sequence's newest blocks.

    A block is quantized once, when its last token arrives, so the cache does not depend on how
    tokens were split among calls.  Appending at an earlier start shortens a sequence first; that
    may go back to the first token of its newest two blocks."""

    def __init__(self, k_pages: Tensor, v_pages: Tensor, k_scale: Tensor, v_scale: Tensor, k_newest: Tensor,
                 v_newest: Tensor, table: Tensor, rows: Optional[Tensor] = None):
        if k_pages.dim() != 4 or k_pages.dtype != torch.uint8:
            raise ValueError("k_pages: uint8 [pages, kv_heads, P, D] expected")
        n, h, p, d = k_pages.shape
        if p not in (16, 32, 64, 128) or d not in (32, 64, 128):
            raise ValueError(f"page size {p}, head_dim {d}: a page size of 16, 32, 64 or 128 and a head_dim of 32, 64 or 128 expected")
        if v_pages.dtype != torch.uint8 or v_pages.shape != (n, h, p // 4, d, 4):
            raise ValueError("v_pages: uint8 [pages, kv_heads, P/4, D, 4] expected")
        if k_scale.dtype != _f32 or v_scale.dtype != _f32 or k_scale.shape != (n, h) or v_scale.shape != (n, h):
            raise ValueError("k_scale, v_scale: fp32 [pages, kv_heads] expected")
        m, t16 = k_newest.shape[0], k_newest.dtype
        if (t16 != torch.float16 and t16 != torch.bfloat16) or k_newest.shape != (m, 2, h, p, d):
            raise ValueError("k_newest: fp16 or bf16 [rows, 2, kv_heads, P, D] expected")
        if v_newest.dtype != t16 or v_newest.shape != (m, 2, h, p // 4, d, 4):
            raise ValueError("v_newest: k_newest's type, [rows, 2, kv_heads, P/4, D, 4] expected")
        if table.dtype != _i32 or table.dim() != 2:
            raise ValueError("table: int32 [batch, blocks] expected")
        b, w = table.shape
        if not 1 <= b <= MAX_BATCH or w < 1 or n < 1 or m < 1:
            raise ValueError(f"batch of 1 to {MAX_BATCH}, at least one page, row and block expected")
        if rows is None and m < b:
            raise ValueError("fewer rows of newest blocks than sequences")
        self.tensors = ts = (k_pages, v_pages, k_scale, v_scale, k_newest, v_newest, table, rows)
        for t in ts:
            if t is not None and not t.is_contiguous():
                raise ValueError("cache tensors must be contiguous")
        self.device = k_pages.device
        self.index = self.device.index
        _stream(self.index, *ts)
        self.kv_heads, self.page_size, self.head_dim, self.dtype, self.batch = h, p, d, t16, b
        self._c = rt.KvCache8(
            k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k_newest.data_ptr(),
            v_newest.data_ptr(), table.data_ptr(), None if rows is None else _index(rows, b, "rows"), n, h, p, d, m, w, b,
            t16 == torch.bfloat16)

    @classmethod
    def allocate(cls, pages: int, kv_heads: int, page_size: int, head_dim: int, table: Tensor,
                 newest_rows: Optional[int] = None, rows: Optional[Tensor] = None,
                 dtype: torch.dtype = torch.float16) -> "PagedKV8":
        """An empty cache on table's device."""
        dev = table.device
        m = table.shape[0] if newest_rows is None else newest_rows
        n, h, p, d = pages, kv_heads, page_size, head_dim
        return cls(torch.empty(n, h, p, d, dtype=torch.uint8, device=dev),
                   torch.empty(n, h, p // 4, d, 4, dtype=torch.uint8, device=dev),
                   torch.empty(n, h, device=dev), torch.empty(n, h, device=dev),
                   torch.empty(m, 2, h, p, d, dtype=dtype, device=dev),
                   torch.empty(m, 2, h, p // 4, d, 4, dtype=dtype, device=dev), table, rows)

    def append(self, qkv: Tensor, cu: Tensor, start: Tensor, *, heads: int, cos: Optional[Tensor] = None,
               sin: Optional[Tensor] = None, interleaved: bool = False, out: Optional[Tensor] = None) -> Tensor:
        """Store the keys and values of new tokens; returns their rotated queries [tokens, heads, D].

        ``qkv`` [tokens, (heads + 2 kv_heads) * D] (q, k, v heads side by side; the rows may be
        strided): row cu[b] + i is token start[b] + i of sequence b (``cu`` int32 [batch + 1],
        ``start`` int32 [batch]).  ``cos`` / ``sin`` fp32 [positions, rot / 2]: the first ``rot``
        channels of a head turn in pairs (i, i + rot/2), or (2i, 2i + 1) if ``interleaved``."""
        d, n = self.head_dim, qkv.shape[0]
        width = (heads + 2 * self.kv_heads) * d
        if heads <= 0 or heads % self.kv_heads:
            raise ValueError(f"heads {heads}: a multiple of {self.kv_heads} expected")
        if qkv.dim() != 2 or qkv.shape[1] != width or qkv.dtype != self.dtype:
            raise ValueError(f"qkv: {self.dtype} [tokens, {width}] expected")
        ld = width
        if n > 1:
            ld, dense = qkv.stride()
            if dense != 1 or ld % 8 or ld < width:
                raise ValueError("qkv: dense rows that start 16-byte aligned and do not overlap expected")
        rot = turns = 0
        if cos is not None or sin is not None:
            if (cos is None or sin is None or cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != _f32 or
                    sin.dtype != _f32 or not cos.is_contiguous() or not sin.is_contiguous()):
                raise ValueError("cos, sin: both or neither, contiguous fp32 [positions, rot / 2] expected")
            turns, rot = cos.shape[0], 2 * cos.shape[1]
            if turns <= 0 or rot <= 0 or rot % 16 or rot > d:
                raise ValueError(f"rotated channels {rot}: a multiple of 16 up to {d} expected")
        if out is None:
            out = torch.empty(n, heads, d, dtype=self.dtype, device=self.device)
        elif out.shape != (n, heads, d) or out.dtype != self.dtype or not out.is_contiguous():
            raise ValueError(f"out: contiguous {self.dtype} [{n}, {heads}, {d}] expected")
        rc = rt.lib().b200_kv8_append(
            self._c, qkv.data_ptr(), ld, out.data_ptr(), _index(cu, self.batch + 1, "cu"),
            _index(start, self.batch, "start"), None if cos is None else cos.data_ptr(),
            None if sin is None else sin.data_ptr(), rot, interleaved, turns, n, heads,
            _stream(self.index, qkv, cu, start, cos, sin, out))
        if rc:
            rt.check(rc, "b200_kv8_append")
        return out

    def read(self, cu: Tensor, start: Tensor, lens: Tensor, *, total: int) -> Tuple[Tensor, Tensor]:
        """Keys and values as attention sees them, [total, kv_heads, D] each: row cu[b] + i is token
        start[b] + i of sequence b, of which lens[b] tokens are cached."""
        if total < 0:
            raise ValueError("total: the number of rows expected")
        k = torch.empty(2, total, self.kv_heads, self.head_dim, dtype=self.dtype, device=self.device)
        v = k[1]
        rc = rt.lib().b200_kv8_read(
            self._c, _index(cu, self.batch + 1, "cu"), _index(start, self.batch, "start"), _index(lens, self.batch, "lens"),
            k.data_ptr(), v.data_ptr(), total, _stream(self.index, cu, start, lens))
        if rc:
            rt.check(rc, "b200_kv8_read")
        return k[0], v

    def attend(self, q: Tensor, cu: Tensor, lens: Tensor, *, max_q_len: int, scale: Optional[float] = None,
               out: Optional[Tensor] = None) -> Tensor:
        """Attention of the newest tokens over the cache, [tokens, heads, D] like ``q``.

        Row cu[b] + i of ``q`` is the token at position lens[b] - n + i of sequence b (n = cu[b+1] -
        cu[b] <= ``max_q_len``), appended already; it sees the keys up to its own.  A row with no key
        gives zeros.  ``scale`` defaults to 1 / sqrt(D).  The same inputs give the same bits."""
        d = self.head_dim
        if q.dim() != 3 or q.shape[2] != d or q.dtype != self.dtype:
            raise ValueError(f"q: {self.dtype} [tokens, heads, {d}] expected")
        n, heads, _ = q.shape
        if heads <= 0 or heads % self.kv_heads:
            raise ValueError(f"heads {heads}: a multiple of {self.kv_heads} expected")
        if max_q_len < 1 and n:
            raise ValueError("max_q_len: at least 1 expected")
        ld_q = self._rows(q, n, heads, d)
        if out is None:
            out = torch.empty(n, heads, d, dtype=self.dtype, device=self.device)
            ld_out = heads * d
        else:
            if out.shape != q.shape or out.dtype != q.dtype:
                raise ValueError("out: q's shape and type expected")
            ld_out = self._rows(out, n, heads, d)
        lib = rt.lib()
        need = lib.b200_kv8_attention_workspace_bytes(self.batch, heads, self.kv_heads, d, max_q_len)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        rc = lib.b200_kv8_attention(
            self._c, q.data_ptr(), ld_q, out.data_ptr(), ld_out, _index(cu, self.batch + 1, "cu"),
            _index(lens, self.batch, "lens"), n, heads, max_q_len, 1 / math.sqrt(d) if scale is None else scale,
            ws.data_ptr(), need, _stream(self.index, q, cu, lens, out))
        if rc:
            rt.check(rc, "b200_kv8_attention")
        return out

    @staticmethod
    def _rows(t: Tensor, n: int, heads: int, d: int) -> int:
        """The row stride of [tokens, heads, D], whose heads lie side by side."""
        ld, per_head, dense = t.stride()
        if dense != 1 or (heads > 1 and per_head != d) or (n > 1 and (ld % 8 or ld < heads * d)):
            raise ValueError("q, out: the heads of a token must be dense, and rows start 16-byte aligned and not overlap")
        return ld if n > 1 else heads * d


# ------------------------------------------------------------------ int8 linear
def quantize_weight(w: Tensor) -> Tuple[Tensor, Tensor]:
    """w [n, k] (fp16, bf16 or fp32) -> int8 codes [n, k rounded up to 16] and fp32 scale [n] (largest magnitude / 127)."""
    _need(w.dim() == 2 and w.dtype in _TYPES and w.shape[1] > 0, "w: fp16, bf16 or fp32 [n, k] expected")
    _need(w.stride(1) == 1 or w.shape[1] == 1, "w: rows must be dense")
    stream = _stream(w.device.index, w)
    n, k = w.shape
    codes = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=w.device)
    scale = torch.empty(n, device=w.device)
    rt.check(rt.lib().b200_quantize_rows_i8(w.data_ptr(), _TYPES[w.dtype], max(w.stride(0), k), codes.data_ptr(),
                                            codes.shape[1], scale.data_ptr(), n, k, stream), "b200_quantize_rows_i8")
    return codes, scale


def linear_int8(x: Tensor, w: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, *, gelu: bool = False,
                resid: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                out: Optional[Tensor] = None) -> Tensor:
    """epi((round(x / sx) @ w.T) * sx * w_scale + bias), sx = each row's largest magnitude / 127.

    ``x`` [m, k] fp16, bf16 or fp32 (rows may be strided); ``w`` int8 [n, pitch], pitch a multiple
    of 16, at least k (``quantize_weight``); ``w_scale`` and ``bias`` fp32 [n].  With ``gelu`` the
    exact GELU follows.  ``resid`` fp32 [m, n] is added last: the result is fp32, and ``out`` may be
    ``resid`` itself.  Without it the result has ``out_dtype`` (default: x's type)."""
    xt = _TYPES.get(x.dtype)
    if xt is None or x.dim() != 2:
        raise ValueError("x: fp16, bf16 or fp32 [m, k] expected")
    m, k = x.shape
    ld_x, dense = x.stride()
    if k < 1 or (dense != 1 and k > 1) or (ld_x < k and m > 1):
        raise ValueError("x: dense rows that do not overlap expected")
    if w.dim() != 2 or w.dtype != torch.int8 or not k <= w.shape[1] < k + 16 or w.stride(1) != 1 or w.stride(0) % 16:
        raise ValueError(f"w: int8 [n, {(k + 15) // 16 * 16}] with a row pitch that is a multiple of 16 expected")
    n = w.shape[0]
    if w_scale.dtype != _f32 or w_scale.shape != (n,) or not w_scale.is_contiguous():
        raise ValueError(f"w_scale: contiguous fp32 [{n}] expected")
    if bias is not None and (bias.dtype != _f32 or bias.shape != (n,) or not bias.is_contiguous()):
        raise ValueError(f"bias: contiguous fp32 [{n}] expected")
    dt = x.dtype if out_dtype is None else out_dtype
    ld_r = n
    if resid is not None:
        if gelu or out_dtype not in (None, _f32):
            raise ValueError("with resid the result is fp32, and there is no GELU")
        if resid.dtype != _f32 or resid.shape != (m, n) or (resid.stride(1) != 1 and n > 1):
            raise ValueError(f"resid: fp32 [{m}, {n}] expected")
        dt, ld_r = _f32, max(resid.stride(0), n)
    ot = _TYPES.get(dt)
    if ot is None:
        raise ValueError("out_dtype: fp16, bf16 or fp32 expected")
    ld_out = n
    if out is None:
        out = torch.empty(m, n, dtype=dt, device=x.device)
    else:
        if out.shape != (m, n) or out.dtype != dt or (out.stride(1) != 1 and n > 1) or (out.stride(0) < n and m > 1):
            raise ValueError(f"out: {dt} [{m}, {n}] with dense rows expected")
        ld_out = max(out.stride(0), n)
    stream = _stream(x.device.index, x, w, w_scale, bias, resid, out)
    lib = rt.lib()
    need = lib.b200_linear_i8_workspace_bytes(m, k)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    a = rt.LinearI8Args(x.data_ptr(), w.data_ptr(), w_scale.data_ptr(), None if bias is None else bias.data_ptr(),
                        None if resid is None else resid.data_ptr(), out.data_ptr(), max(ld_x, k), w.stride(0), ld_r,
                        ld_out, m, n, k, xt, ot, gelu, ws.data_ptr(), need)
    rc = lib.b200_linear_i8(a, stream)
    if rc:
        rt.check(rc, "b200_linear_i8")
    return out


# ------------------------------------------------------------------ a block stack served in 8 bits
class Int8Decoder:
    """Serves a ``UserOptimizedTransformer`` token by token with 8-bit weights and cache.

    ``open()`` gives a sequence id; ``forward(x, seqs, counts)`` appends counts[i] tokens to sequence
    seqs[i] and returns their outputs: a prompt, a chunk of one, drafted tokens or one token a
    sequence, mixed at will.  ``rewind(seq, n)`` drops the last n tokens (of the newest two blocks),
    ``close(seq)`` frees a sequence's pages.  ``rope_base`` turns on the position rotation (the
    model itself has none: its inputs carry their positions).  Head dims 32, 64 and 128."""

    def __init__(self, model, max_sequences: int, max_tokens: int, page_size: int = 64,
                 rope_base: Optional[float] = None):
        cfg = model.config
        _need(bool(cfg.causal), "Int8Decoder: the model must be causal")
        self.config, self.page_size = cfg, page_size
        self.dev = next(model.parameters()).device
        d, self.heads = cfg.d_model, cfg.num_heads
        self.layers: List[dict] = []
        blocks = (max_tokens + page_size - 1) // page_size
        self.table = torch.zeros(max_sequences, blocks, dtype=torch.int32, device=self.dev)
        pages = max_sequences * blocks
        for layer in model.layers:
            a = layer.attention
            qkv = torch.cat([a.q_proj.weight, a.k_proj.weight, a.v_proj.weight]).detach().float().contiguous()
            bias = torch.cat([a.q_proj.bias, a.k_proj.bias, a.v_proj.bias]).detach().float().contiguous()
            w = {"qkv": (*quantize_weight(qkv), bias)}
            for name, lin in (("o", a.out_proj), ("in", layer.ffn_in), ("out", layer.ffn_out)):
                w[name] = (*quantize_weight(lin.weight.detach().float().contiguous()), lin.bias.detach().float())
            w["n1"], w["n2"] = ((n.weight.detach().float(), n.bias.detach().float(), n.eps) for n in (layer.norm1, layer.norm2))
            w["cache"] = PagedKV8.allocate(pages, self.heads, page_size, d // self.heads, self.table)
            self.layers.append(w)
        f = model.final_norm
        self.final = (f.weight.detach().float(), f.bias.detach().float(), f.eps)
        self.cos = self.sin = None
        if rope_base is not None:
            hd = d // self.heads
            turn = torch.arange(blocks * page_size, device=self.dev, dtype=torch.float64)[:, None] * rope_base ** (
                -torch.arange(0, hd, 2, device=self.dev, dtype=torch.float64) / hd)
            self.cos, self.sin = turn.cos().float(), turn.sin().float()
        self.lens = [-1] * max_sequences  # -1: not open
        self.pages: List[List[int]] = [[] for _ in range(max_sequences)]
        self.spare = list(range(pages - 1, -1, -1))

    def open(self) -> int:
        seq = self.lens.index(-1) if -1 in self.lens else -1
        _need(seq >= 0, "every sequence is in use")
        self.lens[seq] = 0
        return seq

    def close(self, seq: int) -> None:
        _need(self.lens[seq] >= 0, f"sequence {seq} is not open")
        self.spare += reversed(self.pages[seq])
        self.pages[seq], self.lens[seq] = [], -1

    def rewind(self, seq: int, n: int) -> None:
        """Drop the last n tokens of a sequence."""
        length, p = self.lens[seq], self.page_size
        _need(length >= 0, f"sequence {seq} is not open")
        _need(0 <= n <= length and (n == 0 or length - n >= max(0, (length - 1) // p - 1) * p),
              "rewind reaches back to the first token of the newest two blocks")
        self.lens[seq] = length - n

    def forward(self, x: Tensor, seqs: Sequence[int], counts: Sequence[int]) -> Tensor:
        """x fp32 [sum(counts), d_model], the tokens of seqs[0] first -> outputs of the same shape."""
        cfg, n, p = self.config, len(self.lens), self.page_size
        _need(len(seqs) == len(counts) and len(set(seqs)) == len(seqs) and min(counts, default=0) >= 0,
              "one count a sequence, each sequence once")
        _need(list(seqs) == sorted(seqs), "sequences in ascending order")
        _need(all(0 <= s < n and self.lens[s] >= 0 for s in seqs), "a sequence that is not open")
        total = sum(counts)
        _need(x.shape == (total, cfg.d_model) and x.dtype == torch.float32 and x.is_contiguous(),
              f"x: contiguous fp32 [{total}, {cfg.d_model}] expected")
        _stream(self.dev.index, x)
        _need(all(self.lens[s] + c <= self.table.shape[1] * p for s, c in zip(seqs, counts)), "a sequence over max_tokens")
        if total == 0:
            return torch.empty_like(x)
        new = [0] * n
        for s, c in zip(seqs, counts):
            new[s] = c
            grown = []
            while len(self.pages[s]) * p < self.lens[s] + c:
                self.pages[s].append(self.spare.pop())
                grown.append(self.pages[s][-1])
            if grown:
                first = len(self.pages[s]) - len(grown)
                self.table[s, first:first + len(grown)] = torch.tensor(grown, dtype=torch.int32).to(self.dev)
        start = [max(0, length) for length in self.lens]
        cu = [0]
        for c in new:
            cu.append(cu[-1] + c)
        meta = torch.tensor(cu + start + [a + b for a, b in zip(start, new)], dtype=torch.int32).to(self.dev)
        cu_t, start_t, lens_t = meta[:n + 1], meta[n + 1:2 * n + 1], meta[2 * n + 1:]
        res = x.clone()
        norm = torch.empty(x.shape, dtype=torch.float16, device=self.dev)
        for w in self.layers:
            rt.layernorm(res, w["n1"][0], w["n1"][1], norm, eps=w["n1"][2])
            qkv = linear_int8(norm, *w["qkv"])
            q = w["cache"].append(qkv, cu_t, start_t, heads=self.heads, cos=self.cos, sin=self.sin)
            ctx = w["cache"].attend(q, cu_t, lens_t, max_q_len=max(new))
            linear_int8(ctx.view(total, -1), *w["o"], resid=res, out=res)
            rt.layernorm(res, w["n2"][0], w["n2"][1], norm, eps=w["n2"][2])
            linear_int8(linear_int8(norm, *w["in"], gelu=True), *w["out"], resid=res, out=res)
        out = torch.empty_like(x)
        rt.layernorm(res, self.final[0], self.final[1], out, eps=self.final[2])
        for s, c in zip(seqs, counts):
            self.lens[s] += c
        return out
