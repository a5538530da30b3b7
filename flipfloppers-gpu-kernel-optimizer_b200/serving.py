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

import ctypes
import math
from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import runtime as rt

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
MAX_BATCH = 4096


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on_device(device: torch.device, *ts: Optional[Tensor]) -> None:
    for t in ts:
        if t is not None and t.device != device:
            raise RuntimeError("libb200block kernels take CUDA tensors on one device only (no CPU fallback)")
    if device.type != "cuda" or device.index != torch.cuda.current_device():
        raise RuntimeError(f"tensors are on {device}, which is not the current CUDA device")


def _index(t: Tensor, n: int, name: str) -> Tensor:
    if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name}: contiguous int32 tensor with {n} entries expected")
    return t


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
        _need(k_pages.dim() == 4 and k_pages.dtype == torch.uint8, "k_pages: uint8 [pages, kv_heads, P, D] expected")
        n, h, p, d = k_pages.shape
        _need(p in (16, 32, 64, 128), f"page size {p}: 16, 32, 64 or 128 expected")
        _need(d in (32, 64, 128), f"head_dim {d}: 32, 64 or 128 expected")
        _need(v_pages.dtype == torch.uint8 and v_pages.shape == (n, h, p // 4, d, 4),
              "v_pages: uint8 [pages, kv_heads, P/4, D, 4] expected")
        for t in (k_scale, v_scale):
            _need(t.dtype == torch.float32 and t.shape == (n, h), "scales: fp32 [pages, kv_heads] expected")
        m = k_newest.shape[0]
        _need(k_newest.dtype in (torch.float16, torch.bfloat16) and k_newest.shape == (m, 2, h, p, d),
              "k_newest: fp16 or bf16 [rows, 2, kv_heads, P, D] expected")
        _need(v_newest.dtype == k_newest.dtype and v_newest.shape == (m, 2, h, p // 4, d, 4),
              "v_newest: k_newest's type, [rows, 2, kv_heads, P/4, D, 4] expected")
        _need(table.dtype == torch.int32 and table.dim() == 2, "table: int32 [batch, blocks] expected")
        b, w = table.shape
        _need(1 <= b <= MAX_BATCH and w >= 1 and n >= 1 and m >= 1, f"batch 1 to {MAX_BATCH}, at least one page, row and block")
        _need(rows is not None or m >= b, "fewer rows of newest blocks than sequences")
        if rows is not None:
            _index(rows, b, "rows")
        for t in (k_pages, v_pages, k_scale, v_scale, k_newest, v_newest, table):
            _need(t.is_contiguous(), "cache tensors must be contiguous")
        self.device = k_pages.device
        _on_device(self.device, k_pages, v_pages, k_scale, v_scale, k_newest, v_newest, table, rows)
        self.tensors = (k_pages, v_pages, k_scale, v_scale, k_newest, v_newest, table, rows)
        self.kv_heads, self.page_size, self.head_dim, self.dtype, self.batch = h, p, d, k_newest.dtype, b
        self._c = rt.KvCache8(
            k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k_newest.data_ptr(),
            v_newest.data_ptr(), table.data_ptr(), None if rows is None else rows.data_ptr(), n, h, p, d, m, w, b,
            int(self.dtype == torch.bfloat16))

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
        d, width = self.head_dim, (heads + 2 * self.kv_heads) * self.head_dim
        _need(heads > 0 and heads % self.kv_heads == 0, f"heads {heads}: a multiple of {self.kv_heads} expected")
        _need(qkv.dim() == 2 and qkv.shape[1] == width and qkv.dtype == self.dtype,
              f"qkv: {self.dtype} [tokens, {width}] expected")
        _need(qkv.stride(1) == 1 and qkv.stride(0) % 8 == 0 or qkv.shape[0] <= 1, "qkv: rows must be dense and start 16-byte aligned")
        n = qkv.shape[0]
        _index(cu, self.batch + 1, "cu")
        _index(start, self.batch, "start")
        _need((cos is None) == (sin is None), "cos and sin go together")
        rot = turns = 0
        if cos is not None:
            _need(cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32 and
                  cos.is_contiguous() and sin.is_contiguous(), "cos, sin: contiguous fp32 [positions, rot / 2] expected")
            turns, rot = cos.shape[0], 2 * cos.shape[1]
            _need(turns > 0 and rot > 0 and rot % 16 == 0 and rot <= d, f"rotated channels {rot}: a multiple of 16 up to {d} expected")
        if out is None:
            out = torch.empty(n, heads, d, dtype=self.dtype, device=self.device)
        _need(out.shape == (n, heads, d) and out.dtype == self.dtype and out.is_contiguous(),
              f"out: contiguous {self.dtype} [{n}, {heads}, {d}] expected")
        _on_device(self.device, qkv, cu, start, cos, sin, out)
        rt.check(rt.lib().b200_kv8_append(
            self._c, qkv.data_ptr(), max(qkv.stride(0), width) if n <= 1 else qkv.stride(0), out.data_ptr(), cu.data_ptr(),
            start.data_ptr(), None if cos is None else cos.data_ptr(), None if sin is None else sin.data_ptr(), rot,
            int(interleaved), turns, n, heads, rt._stream()), "b200_kv8_append")
        return out

    def read(self, cu: Tensor, start: Tensor, lens: Tensor, *, total: int) -> Tuple[Tensor, Tensor]:
        """Keys and values as attention sees them, [total, kv_heads, D] each: row cu[b] + i is token
        start[b] + i of sequence b, of which lens[b] tokens are cached."""
        _index(cu, self.batch + 1, "cu")
        _index(start, self.batch, "start")
        _index(lens, self.batch, "lens")
        _need(total >= 0, "total: the number of rows expected")
        _on_device(self.device, cu, start, lens)
        k = torch.empty(total, self.kv_heads, self.head_dim, dtype=self.dtype, device=self.device)
        v = torch.empty_like(k)
        rt.check(rt.lib().b200_kv8_read(self._c, cu.data_ptr(), start.data_ptr(), lens.data_ptr(), k.data_ptr(),
                                        v.data_ptr(), total, rt._stream()), "b200_kv8_read")
        return k, v

    def attend(self, q: Tensor, cu: Tensor, lens: Tensor, *, max_q_len: int, scale: Optional[float] = None,
               out: Optional[Tensor] = None) -> Tensor:
        """Attention of the newest tokens over the cache, [tokens, heads, D] like ``q``.

        Row cu[b] + i of ``q`` is the token at position lens[b] - n + i of sequence b (n = cu[b+1] -
        cu[b] <= ``max_q_len``), appended already; it sees the keys up to its own.  A row with no key
        gives zeros.  ``scale`` defaults to 1 / sqrt(D).  The same inputs give the same bits."""
        d = self.head_dim
        _need(q.dim() == 3 and q.shape[2] == d and q.dtype == self.dtype, f"q: {self.dtype} [tokens, heads, {d}] expected")
        n, heads = q.shape[0], q.shape[1]
        _need(heads > 0 and heads % self.kv_heads == 0, f"heads {heads}: a multiple of {self.kv_heads} expected")
        _need(max_q_len >= 1 or n == 0, "max_q_len: at least 1 expected")
        _index(cu, self.batch + 1, "cu")
        _index(lens, self.batch, "lens")
        if out is None:
            out = torch.empty(n, heads, d, dtype=self.dtype, device=self.device)
        _need(out.shape == q.shape and out.dtype == q.dtype, "out: q's shape and type expected")
        for t in (q, out):
            _need(t.stride(2) == 1 and (heads == 1 or t.stride(1) == d) and (n <= 1 or t.stride(0) % 8 == 0),
                  "q, out: the heads of a token must be dense and rows start 16-byte aligned")
        _on_device(self.device, q, cu, lens, out)
        lib = rt.lib()
        need = lib.b200_kv8_attention_workspace_bytes(self.batch, heads, self.kv_heads, d, max(1, max_q_len))
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        width = heads * d
        rt.check(lib.b200_kv8_attention(
            self._c, q.data_ptr(), q.stride(0) if n > 1 else width, out.data_ptr(), out.stride(0) if n > 1 else width,
            cu.data_ptr(), lens.data_ptr(), n, heads, max_q_len, 1 / math.sqrt(d) if scale is None else scale,
            ws.data_ptr(), need, rt._stream()), "b200_kv8_attention")
        return out


# ------------------------------------------------------------------ int8 linear
def quantize_weight(w: Tensor) -> Tuple[Tensor, Tensor]:
    """w [n, k] (fp16, bf16 or fp32) -> int8 codes [n, k rounded up to 16] and fp32 scale [n] (largest magnitude / 127)."""
    _need(w.dim() == 2 and w.dtype in _TYPES and w.shape[1] > 0, "w: fp16, bf16 or fp32 [n, k] expected")
    _need(w.stride(1) == 1 or w.shape[1] == 1, "w: rows must be dense")
    _on_device(w.device, w)
    n, k = w.shape
    codes = torch.zeros(n, (k + 15) // 16 * 16, dtype=torch.int8, device=w.device)
    scale = torch.empty(n, device=w.device)
    rt.check(rt.lib().b200_quantize_rows_i8(w.data_ptr(), _TYPES[w.dtype], max(w.stride(0), k), codes.data_ptr(),
                                            codes.shape[1], scale.data_ptr(), n, k, rt._stream()), "b200_quantize_rows_i8")
    return codes, scale


def linear_int8(x: Tensor, w: Tensor, w_scale: Tensor, bias: Optional[Tensor] = None, *, gelu: bool = False,
                resid: Optional[Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                out: Optional[Tensor] = None) -> Tensor:
    """epi((round(x / sx) @ w.T) * sx * w_scale + bias), sx = each row's largest magnitude / 127.

    ``x`` [m, k] fp16, bf16 or fp32 (rows may be strided); ``w`` int8 [n, pitch], pitch a multiple
    of 16, at least k (``quantize_weight``); ``w_scale`` and ``bias`` fp32 [n].  With ``gelu`` the
    exact GELU follows.  ``resid`` fp32 [m, n] is added last: the result is fp32, and ``out`` may be
    ``resid`` itself.  Without it the result has ``out_dtype`` (default: x's type)."""
    _need(x.dim() == 2 and x.dtype in _TYPES, "x: fp16, bf16 or fp32 [m, k] expected")
    m, k = x.shape
    _need(k > 0 and (x.stride(1) == 1 or k == 1), "x: rows must be dense")
    _need(w.dim() == 2 and w.dtype == torch.int8 and w.shape[1] >= k and w.stride(1) == 1 and w.stride(0) % 16 == 0,
          f"w: int8 [n, >= {k}] with a row pitch that is a multiple of 16 expected")
    _need(w.shape[1] < k + 16, f"w has {w.shape[1]} columns for x's {k}")
    n = w.shape[0]
    for t, name in ((w_scale, "w_scale"), (bias, "bias")):
        if t is not None:
            _need(t.dtype == torch.float32 and t.shape == (n,) and t.is_contiguous(), f"{name}: contiguous fp32 [{n}] expected")
    _need(resid is None or not gelu, "gelu and resid exclude each other")
    if resid is not None:
        _need(resid.dtype == torch.float32 and resid.shape == (m, n) and (resid.stride(1) == 1 or n == 1),
              f"resid: fp32 [{m}, {n}] expected")
        _need(out_dtype in (None, torch.float32), "with resid the result is fp32")
        out_dtype = torch.float32
    dt = x.dtype if out_dtype is None else out_dtype
    _need(dt in _TYPES, "out_dtype: fp16, bf16 or fp32 expected")
    if out is None:
        out = torch.empty(m, n, dtype=dt, device=x.device)
    _need(out.shape == (m, n) and out.dtype == dt and (out.stride(1) == 1 or n == 1), f"out: {dt} [{m}, {n}] expected")
    _on_device(x.device, x, w, w_scale, bias, resid, out)
    lib = rt.lib()
    need = lib.b200_linear_i8_workspace_bytes(m, k)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)
    a = rt.LinearI8Args(x.data_ptr(), w.data_ptr(), w_scale.data_ptr(), None if bias is None else bias.data_ptr(),
                        None if resid is None else resid.data_ptr(), out.data_ptr(), max(x.stride(0), k), w.stride(0),
                        n if resid is None else max(resid.stride(0), n), max(out.stride(0), n), m, n, k,
                        _TYPES[x.dtype], _TYPES[dt], int(gelu), ws.data_ptr(), need)
    rt.check(lib.b200_linear_i8(ctypes.byref(a), rt._stream()), "b200_linear_i8")
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
        _on_device(self.dev, x)
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
