"""Int8Decoder's bookkeeping (lengths, pages, how far a sequence may be shortened), its kernels replaced by fakes."""

import pytest
import torch


class FakeCache:
    """Stands in for PagedKV8: keeps which block each of a sequence's two slots holds, and up to which token."""

    def __init__(self, page, table):
        self.page, self.table = page, table
        self.slots = [[(-1, 0), (-1, 0)] for _ in range(table.shape[0])]

    def append(self, qkv, cu, start, heads, cos=None, sin=None):
        for b, first in enumerate(start.tolist()):
            n = int(cu[b + 1] - cu[b])
            if n and first % self.page:  # the block's earlier tokens must be there
                block, upto = self.slots[b][first // self.page % 2]
                assert block == first // self.page and upto >= first % self.page, "a block that was not kept"
            for t in range(first, first + n):
                self.slots[b][t // self.page % 2] = (t // self.page, t % self.page + 1)
        return torch.zeros(qkv.shape[0], heads, qkv.shape[1] // (3 * heads))

    def attend(self, q, cu, lens, max_q_len):
        for b, n in enumerate(lens.tolist()):
            if n % self.page and cu[b + 1] > cu[b]:
                block, upto = self.slots[b][n // self.page % 2]
                assert block == n // self.page and upto >= n % self.page, "a block that was not kept"
        return q


@pytest.fixture
def decoder(tt, monkeypatch):
    sv = tt.serving
    cfg = tt.TransformerConfig(2, 8, 64, 2, 128, 1, True)
    model = tt.UserOptimizedTransformer(cfg)
    monkeypatch.setattr(sv, "_on_device", lambda t: None)
    monkeypatch.setattr(sv, "quantize_weight", lambda w: (w, torch.ones(w.shape[0])))
    monkeypatch.setattr(sv.rt, "layernorm", lambda x, g, b, out, eps: out)
    monkeypatch.setattr(sv, "linear_int8", lambda x, w, ws, bias, gelu=False, resid=None, out=None: x.new_zeros(x.shape[0], w.shape[0]))
    monkeypatch.setattr(sv.PagedKV8, "allocate", classmethod(lambda cls, pages, heads, page, dim, table: FakeCache(page, table)))
    dec = sv.Int8Decoder(model, max_sequences=3, max_tokens=256, page_size=16)
    dec.step = lambda seq, n: dec.forward(torch.zeros(n, 64), [seq], [n])
    return dec


def test_rewinding_twice_stays_within_what_is_kept(decoder):
    s = decoder.open()
    decoder.step(s, 33)  # blocks 0, 1, 2: the slots hold 2 and 1
    with pytest.raises(ValueError):
        decoder.rewind(s, 18)  # into block 0
    decoder.rewind(s, 1)       # 32
    with pytest.raises(ValueError):
        decoder.rewind(s, 17)  # 15, into block 0: its slot still holds block 2
    decoder.rewind(s, 16)      # 16: block 1's first token
    with pytest.raises(ValueError):
        decoder.rewind(s, 1)
    decoder.step(s, 3)         # 19
    with pytest.raises(ValueError):
        decoder.rewind(s, 4)   # appending did not bring block 0 back
    decoder.step(s, 30)        # 49: blocks 3 and 2
    with pytest.raises(ValueError):
        decoder.rewind(s, 18)
    decoder.rewind(s, 17)      # 32
    decoder.step(s, 1)


def test_a_sequence_that_was_closed_starts_afresh(decoder):
    s = decoder.open()
    decoder.step(s, 100)
    decoder.close(s)
    assert decoder.open() == s
    decoder.step(s, 5)
    decoder.rewind(s, 5)
    decoder.step(s, 40)


def test_a_step_that_failed(tt, decoder, monkeypatch):
    """A step that raises half way has stored tokens already: it may be repeated where the slots still hold what
    it starts from, and is refused where they do not."""
    sv = tt.serving
    good = sv.linear_int8
    a, b = decoder.open(), decoder.open()
    decoder.step(a, 20)
    decoder.step(b, 20)

    def broken(x, w, *args, resid=None, **kw):
        if resid is not None:  # after the append and attention
            raise RuntimeError("out of memory")
        return good(x, w, *args, resid=resid, **kw)

    for seq, n in ((a, 10), (b, 40)):
        monkeypatch.setattr(sv, "linear_int8", broken)
        with pytest.raises(RuntimeError):
            decoder.step(seq, n)
        monkeypatch.setattr(sv, "linear_int8", good)
    assert decoder.lens[a] == decoder.lens[b] == 20
    decoder.step(a, 10)
    with pytest.raises(ValueError):
        decoder.step(b, 40)  # the slot of block 1, whose first four tokens it needs, holds block 3
    with pytest.raises(ValueError):
        decoder.forward(torch.zeros(2, 64), [a, b], [1, 1])
    decoder.step(a, 1)
    decoder.close(b)
    assert decoder.open() == b
    decoder.step(b, 60)


def test_ids_that_are_no_sequence_are_refused(decoder):
    ids = [decoder.open() for _ in range(3)]
    for s in ids:
        decoder.step(s, 5)
    for bad in (-1, -3, 3, 100):
        for call in (lambda: decoder.rewind(bad, 1), lambda: decoder.close(bad), lambda: decoder.step(bad, 1)):
            with pytest.raises(ValueError):
                call()
    assert decoder.lens == [5, 5, 5]
    decoder.close(2)
    with pytest.raises(ValueError):
        decoder.close(2)
