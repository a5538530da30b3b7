"""Serve a block stack in 8 bits: prompts, then one token a sequence a step.

    python examples/serve_int8.py [--sequences 8] [--prompt 500] [--steps 64] [--d-model 1024] [--heads 16] ...

Each sequence's "next token" is the model's output for its last one (the stack has no vocabulary).  Prints the
time of the prompts and of a step, and how far the 8-bit outputs of the prompts are from the fp16 forward.
"""

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import torch_transformer_benchmark as T  # noqa: E402


def timed(f):
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    out = f()
    end.record()
    torch.cuda.synchronize()
    return out, begin.elapsed_time(end)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--sequences", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--d-model", type=int, default=1024)
    ap.add_argument("--heads", type=int, default=16)
    ap.add_argument("--ffn-dim", type=int, default=4096)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args()
    cfg = T.TransformerConfig(a.sequences, a.prompt, a.d_model, a.heads, a.ffn_dim, a.layers, True)
    torch.manual_seed(0)
    model = T.UserOptimizedTransformer(cfg).cuda().eval()
    x = torch.randn(a.sequences, a.prompt, a.d_model, device="cuda")
    with torch.inference_mode():
        dec = T.serving.Int8Decoder(model, a.sequences, a.prompt + a.steps, page_size=64, rope_base=None)
        seqs = [dec.open() for _ in range(a.sequences)]
        y, ms = timed(lambda: dec.forward(x.view(-1, a.d_model), seqs, [a.prompt] * a.sequences))
        want = model(x)
        far = ((y.view_as(want) - want).norm() / want.norm()).item()
        print(f"prompts: {a.sequences} x {a.prompt} tokens in {ms:.2f} ms; {100 * far:.2f} % from the fp16 forward (2-norm)")
        last = y.view(a.sequences, a.prompt, -1)[:, -1].contiguous()
        for _ in range(8 if a.steps > 16 else 0):
            last = dec.forward(last, seqs, [1] * a.sequences)

        def steps():
            t = last
            for _ in range(a.steps - (8 if a.steps > 16 else 0)):
                t = dec.forward(t, seqs, [1] * a.sequences)
            return t

        _, ms = timed(steps)
        n = a.steps - (8 if a.steps > 16 else 0)
        print(f"steps: {1e3 * ms / n:.0f} us for {a.sequences} tokens, {a.layers} layers ({n} steps)")
    err = T._pkg.runtime.device_error()
    if err:
        raise SystemExit(f"device error word {err}")


if __name__ == "__main__":
    main()
