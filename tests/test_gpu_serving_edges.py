"""Corners of the 8-bit serving operators, on a B200: sequences shortened more than once, values and scales at the
ends of their ranges, arguments that overlap or wrap, shapes that take the kernels' longer paths."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sv(tt):
    return tt.serving


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def starts(counts):
    return i32([0] + torch.tensor(counts).cumsum(0).tolist())


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
