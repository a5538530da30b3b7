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
behind it.  The operators' row counts and lengths are device tensors (int32), so
that a step written with them can be captured in a CUDA graph and replayed with
other values in them (``Int8Decoder`` counts on the host, and is not captured).
All of it is for inference: results carry no autograd graph, whatever the inputs.
"""

from __future__ import annotations

import importlib.util
import os
from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from . import build as _build
from . import runtime as rt

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _on_device(t: Tensor) -> None:
    if not t.is_cuda or t.device.index != torch.cuda.current_device():
        raise RuntimeError("libb200block kernels take CUDA tensors on the current device only (no CPU fallback)")


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


_module = None


def _native():
    """The calls' C++ side (csrc/serving_binding.cpp); raises if it has not been built."""
    global _module
    if _module is None:
        rt.lib()
        path = _build.BINDING_PATH
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is missing: build it with `python {_build.__file__}`")
        spec = importlib.util.spec_from_file_location("b200serving", path)
        _module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_module)
    return _module


def _done(result, what: str):
    """A call's result; a launcher's status raises."""
    if type(result) is int:
        rt.check(result, what)
    return result


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
    may go back to the first token of the newest two blocks it has had since it was empty (a slot
    keeps the latest block that was written to it: shortening a sequence does not bring back the
    block before)."""

    def __init__(self, k_pages: Tensor, v_pages: Tensor, k_scale: Tensor, v_scale: Tensor, k_newest: Tensor,
                 v_newest: Tensor, table: Tensor, rows: Optional[Tensor] = None):
        self._c = _native().cache(k_pages, v_pages, k_scale, v_scale, k_newest, v_newest, table, rows)
        self.tensors = (k_pages, v_pages, k_scale, v_scale, k_newest, v_newest, table, rows)

    @property
    def batch(self) -> int:
        return self.tensors[6].shape[0]

    @property
    def kv_heads(self) -> int:
        return self.tensors[0].shape[1]

    @property
    def page_size(self) -> int:
        return self.tensors[0].shape[2]

    @property
    def head_dim(self) -> int:
        return self.tensors[0].shape[3]

    @property
    def dtype(self) -> torch.dtype:
        return self.tensors[4].dtype

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
        channels of a head turn in pairs (i, i + rot/2), or (2i, 2i + 1) if ``interleaved``.  ``out``
        may not overlap qkv."""
        return _done(_module.append(self._c, qkv, cu, start, heads, cos, sin, interleaved, out), "b200_kv8_append")

    def read(self, cu: Tensor, start: Tensor, lens: Tensor, *, total: int) -> Tuple[Tensor, Tensor]:
        """Keys and values as attention sees them, [total, kv_heads, D] each: row cu[b] + i is token
        start[b] + i of sequence b, of which lens[b] tokens are cached."""
        return _done(_module.read(self._c, cu, start, lens, total), "b200_kv8_read")

    def attend(self, q: Tensor, cu: Tensor, lens: Tensor, *, max_q_len: int, scale: Optional[float] = None,
               out: Optional[Tensor] = None) -> Tensor:
        """Attention of the newest tokens over the cache, [tokens, heads, D] like ``q``.

        Row cu[b] + i of ``q`` is the token at position lens[b] - n + i of sequence b (n = cu[b+1] -
        cu[b] <= ``max_q_len``), appended already; it sees the keys up to its own.  A row with no key
        gives zeros.  Weights are rounded to fp16 before they meet V (2^-11 of each), scores, maxima and
        sums are fp32.  ``scale`` defaults to 1 / sqrt(D).  ``out`` may be q itself, and not overlap it
        otherwise.  The same inputs give the same bits."""
        return _done(_module.attend(self._c, q, cu, lens, max_q_len, scale, out), "b200_kv8_attention")


# ------------------------------------------------------------------ int8 linear
def quantize_weight(w: Tensor) -> Tuple[Tensor, Tensor]:
    """w [n, k] (fp16, bf16 or fp32) -> int8 codes [n, k rounded up to 16] and fp32 scale [n] (largest magnitude / 127)."""
    _need(w.dim() == 2 and w.dtype in _TYPES and w.shape[1] > 0, "w: fp16, bf16 or fp32 [n, k] expected")
    _need(w.stride(1) == 1 or w.shape[1] == 1, "w: rows must be dense")
    _on_device(w)
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
    of 16, at least k (``quantize_weight``); ``w_scale`` and ``bias`` fp32 [n].  With ``gelu``
    the erf form of GELU follows (fp32 results: to fp32; 16-bit ones: within 2e-6).  ``resid`` fp32 [m, n] is added last: the result is fp32, and ``out`` may be
    ``resid`` itself; it may not overlap what is read otherwise.  Without it the result has ``out_dtype`` (default: x's type)."""
    return _done(_native().linear_i8(x, w, w_scale, bias, gelu, resid, out_dtype, out), "b200_linear_i8")


# ------------------------------------------------------------------ a block stack served in 8 bits
class Int8Decoder:
    """Serves a ``UserOptimizedTransformer`` token by token with 8-bit weights and cache.

    ``open()`` gives a sequence id; ``forward(x, seqs, counts)`` appends counts[i] tokens to sequence
    seqs[i] and returns their outputs: a prompt, a chunk of one, drafted tokens or one token a
    sequence, mixed at will.  ``rewind(seq, n)`` drops the last n tokens (of the newest two blocks
    that the sequence has had, as far as PagedKV8 keeps them), ``close(seq)`` frees a sequence's pages.  ``rope_base`` turns on the position rotation (the
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
        self.kept = [0] * max_sequences   # first token that the slots of the newest blocks still hold
        self.pages: List[List[int]] = [[] for _ in range(max_sequences)]
        self.spare = list(range(pages - 1, -1, -1))

    def open(self) -> int:
        seq = self.lens.index(-1) if -1 in self.lens else -1
        _need(seq >= 0, "every sequence is in use")
        self.lens[seq] = self.kept[seq] = 0
        return seq

    def _open_length(self, seq: int) -> int:
        _need(0 <= seq < len(self.lens) and self.lens[seq] >= 0, f"sequence {seq} is not open")
        return self.lens[seq]

    def close(self, seq: int) -> None:
        self._open_length(seq)
        self.spare += reversed(self.pages[seq])
        self.pages[seq], self.lens[seq] = [], -1

    def rewind(self, seq: int, n: int) -> None:
        """Drop the last n tokens of a sequence."""
        length = self._open_length(seq)
        _need(0 <= n <= length and (n == 0 or length - n >= self.kept[seq]),
              "rewind reaches back to the first token of the newest two blocks the sequence has had")
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
        _on_device(x)
        _need(all(self.lens[s] + c <= self.table.shape[1] * p for s, c in zip(seqs, counts)), "a sequence over max_tokens")
        _need(all(c == 0 or self.lens[s] >= self.kept[s] for s, c in zip(seqs, counts)),
              "a step of this sequence raised after it had overwritten what the sequence goes on from: close it")
        if total == 0:
            return torch.empty_like(x)
        new = [0] * n
        grown, pages = [], []  # sequences that need pages and how many; the pages
        for s, c in zip(seqs, counts):
            new[s] = c
            more = (self.lens[s] + c + p - 1) // p - len(self.pages[s])
            if more > 0:
                grown.append((s, more))
                end = len(self.spare) - len(pages)
                pages += self.spare[end - more:end][::-1]
        start = [max(0, length) for length in self.lens]
        cu = [0]
        for c in new:
            cu.append(cu[-1] + c)
        # one copy from pinned memory, which the allocator keeps until the copy has run: nothing waits for the device
        meta = torch.tensor(cu + start + [a + b for a, b in zip(start, new)] + pages, dtype=torch.int32,
                            pin_memory=self.dev.type == "cuda").to(self.dev, non_blocking=True)
        cu_t, start_t, lens_t, pages_t = meta.split([n + 1, n, n, len(pages)])
        at = 0
        for s, more in grown:
            had = len(self.pages[s])
            self.table[s, had:had + more] = pages_t[at:at + more]
            self.pages[s] += pages[at:at + more]
            del self.spare[-more:]
            at += more
        for s, c in zip(seqs, counts):
            self.kept[s] = max(self.kept[s], ((self.lens[s] + c - 1) // p - 1) * p)
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
