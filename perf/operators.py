"""Cases that measure the 8-bit serving operators: what they take, compute and return.

Three operators make up one decoding step in 8 bits:

* ``append``: the fused QKV rows of new tokens are rotated by position; q is returned, k and v go to a paged
  cache (whole blocks of tokens in 8 bits with one scale a block and key head, the last block in 16 bits), and
  the blocks that were touched are read back as the values that attention sees;
* ``attend``: attention of one or more new tokens of each sequence over such a cache;
* ``linear``: rows quantized to 8 bits with a scale each, times an 8-bit weight with a scale a channel, with
  bias, GELU or a residual.

``run`` computes them with the framework's kernels where ``own`` is true, and with elementary torch operations
in 32 bits where it is not.  ``exact`` restates them in 64 bits, sequence by sequence.

Cache layout (page size P tokens, D channels a head), shared by all the forms:

* ``k_pages`` uint8 [pages, kv_heads, P, D], ``v_pages`` uint8 [pages, kv_heads, P/4, D, 4] (four tokens of a
  channel side by side), a code c standing for (c - 128) * scale; ``k_scale``, ``v_scale`` fp32 [pages, kv_heads];
* ``k_tail`` [rows, 2, kv_heads, P, D], ``v_tail`` [rows, 2, kv_heads, P/4, D, 4], 16 bits: the newest two
  blocks of each sequence, block j in slot j % 2; a block that is not full is read from here;
* ``table`` int32 [batch, blocks]: the page of each block.
"""

import math

import torch

own = False

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of one sequence: the latency of a step for a single user (16 heads of 64, as in the
        # framework's 1024-wide blocks)
        {"name": "append 1 token", "op": "append", "dtype": "float16", "batch": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 700,
         "ctx_hi": 1300, "heads": 16, "kv_heads": 16, "dim": 64, "rot": 0, "page": 64},
        # a decoding step of many users with grouped heads: one token each at ragged lengths
        {"name": "append 1 token x 128", "op": "append", "dtype": "bfloat16", "batch": 128, "new_lo": 1, "new_hi": 1,
         "ctx_lo": 0, "ctx_hi": 8000, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "page": 32},
        # prompts of ragged lengths entering an empty cache
        {"name": "append prompts", "op": "append", "dtype": "float16", "batch": 6, "new_lo": 500, "new_hi": 9001,
         "ctx_lo": 0, "ctx_hi": 0, "heads": 16, "kv_heads": 16, "dim": 64, "rot": 64, "page": 64},
        # a step for a single user over a short context
        {"name": "attend 1 token", "op": "attend", "dtype": "float16", "batch": 1, "q_len": 1, "len_lo": 700, "len_hi": 1300,
         "heads": 16, "kv_heads": 16, "dim": 64, "page": 64},
        # a decoding step of many users at ragged lengths, grouped heads
        {"name": "attend 1 token x 64", "op": "attend", "dtype": "bfloat16", "batch": 64, "q_len": 1, "len_lo": 1,
         "len_hi": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "page": 32},
        # one user deep in a long document
        {"name": "attend 1 token, long", "op": "attend", "dtype": "bfloat16", "batch": 1, "q_len": 1, "len_lo": 130001,
         "len_hi": 131071, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128},
        # several drafted tokens a user are checked at once; some sequences are shorter than the draft
        {"name": "attend 5 drafted x 33", "op": "attend", "dtype": "float16", "batch": 33, "q_len": 5, "len_lo": 3,
         "len_hi": 3000, "heads": 24, "kv_heads": 4, "dim": 64, "page": 16},
        # a chunk of a prompt over what is cached already
        {"name": "attend chunk", "op": "attend", "dtype": "float16", "batch": 1, "q_len": 2048, "len_lo": 16001,
         "len_hi": 18431, "heads": 16, "kv_heads": 16, "dim": 64, "page": 64},
        # the FFN's first product for one token
        {"name": "linear 1 row", "op": "linear", "dtype": "float16", "rows": 1, "k": 1024, "n": 4096, "epi": "gelu"},
        # the FFN's second product for a step of 64 users, added to the residual stream
        {"name": "linear 64 rows", "op": "linear", "dtype": "float16", "rows": 64, "k": 4096, "n": 1024, "epi": "resid"},
        # sizes that fill no tile
        {"name": "linear odd", "op": "linear", "dtype": "bfloat16", "rows": 333, "k": 1001, "n": 1030, "epi": "bias"},
        # the FFN's first product for a batch of prompts
        {"name": "linear 32768 rows", "op": "linear", "dtype": "float16", "rows": 32768, "k": 1024, "n": 4096, "epi": "gelu"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["append", "attend", "attend", "linear"])
        if op == "linear":
            case = {"op": op, "dtype": rng.choice(["float16", "bfloat16", "float32"]), "rows": _log(rng, 1, 32768),
                    "k": _log(rng, 64, 8192), "n": _log(rng, 64, 8192), "epi": rng.choice(["bias", "gelu", "resid"])}
            if rng.random() < 0.6:  # widths of models are mostly round
                case["k"], case["n"] = max(64, case["k"] // 64 * 64), max(64, case["n"] // 64 * 64)
            if 3072 in (case["k"], case["n"], case["rows"]):
                continue
        else:
            dim = rng.choice([32, 64, 128])
            kv = rng.choice([1, 2, 4, 8, 16])
            case = {"op": op, "dtype": rng.choice(["float16", "bfloat16"]), "batch": _log(rng, 1, 128)}
            if op == "append":
                new = _log(rng, 2, 8192) if rng.random() < 0.6 else 1
                ctx = 0 if new > 16 else _log(rng, 1, 16384)  # long pieces enter an empty cache
                case |= {"new_lo": (new + 1) // 2, "new_hi": new, "ctx_lo": 0, "ctx_hi": ctx}
            else:
                q_len = 1 if rng.random() < 0.5 else _log(rng, 2, 16) if rng.random() < 0.6 else _log(rng, 17, 2048)
                most_len = _log(rng, q_len, 131071)
                case |= {"q_len": q_len, "len_lo": max(1, most_len // 8), "len_hi": most_len}
            case |= {"heads": kv * rng.choice([1, 1, 2, 3, 4, 6, 8]), "kv_heads": kv, "dim": dim}
            if op == "append":
                case["rot"] = rng.choice([0, dim // 2, dim, dim])
            case["page"] = rng.choice([16, 32, 64, 128])
            # the plain forms spread the cache out in 32 bits
            rows = case["batch"] * (case["new_hi"] if op == "append" else case["len_hi"])
            if rows * kv * dim > 64 * 8192 * 8 * 128:
                continue
            if op == "attend" and case["batch"] * case["heads"] * case["q_len"] * case["len_hi"] > 16 * 2048 * 18431:
                continue
        if _cost(case) <= most:
            return case


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 200


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        out = 4 if case["epi"] == "resid" else size
        return {"bytes": m * k * size + n * k + 8 * n + m * n * (out + (4 if case["epi"] == "resid" else 0)), "flops": 2 * m * n * k}
    h, kv, d, p, b = case["heads"], case["kv_heads"], case["dim"], case["page"], case["batch"]
    if case["op"] == "append":
        new, ctx = _spread(case, "new"), _spread(case, "ctx")
        t, was = sum(new), sum(x % p for x in ctx)
        done = sum((x + y) // p - x // p for x, y in zip(ctx, new)) * p
        wrote = done * (1 + 4 / (p * d)) + min(t, 2 * p * b) * 2  # codes and scales, and the newest blocks in 16 bits
        return {"bytes": t * (h + 2 * kv) * d * 2 + t * case["rot"] * 4 + t * h * d * 2 + 2 * kv * d * (was * 2 + wrote + (t + was) * 2),
                "flops": 3 * t * (h + kv) * case["rot"] + 6 * done * kv * d}
    lens, q = _spread(case, "len"), case["q_len"]
    seen = sum(q * n - q * (q - 1) // 2 if n >= q else n * (n + 1) // 2 for n in lens)
    cache = sum(n // p * (p * d + 4) + n % p * d * 2 for n in lens) * kv * 2
    return {"bytes": cache + 2 * b * q * h * d * 2, "flops": 4 * d * h * seen}


def _spread(case, what):
    """Ragged whole numbers, one a sequence, from the case's own numbers (the seed changes their order only)."""
    lo, hi, n = case[what + "_lo"], case[what + "_hi"], case["batch"]
    return [lo + (hi - lo) * ((i * 7919 + 5) % 104729 * 31337 % 104729) // 104728 if n > 1 else (lo + hi) // 2 | (hi > lo) for i in range(n)]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def whole(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    t = TYPES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        x = normal(m, k)
        x *= torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 8.0, 1.0)  # a few loud channels
        if m > 2:
            x[m // 2] = 0  # a padded row
        pitch = (k + 15) // 16 * 16  # rows of a weight start on 16 bytes
        w = torch.zeros(n, pitch, dtype=torch.int8, device="cuda")
        w[:, :k] = (normal(n, k) * 36).round_().clamp_(-127, 127).to(torch.int8)
        return {"case": case, "x": x.to(t), "w": w, "w_scale": (0.5 + torch.rand(n, generator=g, device="cuda")) / (36 * math.sqrt(k)),
                "bias": normal(n) * 0.1, "resid": normal(m, n) if case["epi"] == "resid" else None}

    b, kv, d, p = case["batch"], case["kv_heads"], case["dim"], case["page"]
    order = torch.randperm(b, generator=g, device="cuda").tolist()
    if case["op"] == "append":
        new, start = ([_spread(case, w)[i] for i in order] for w in ("new", "ctx"))
        lens = [x + y for x, y in zip(start, new)]
    else:
        lens = [_spread(case, "len")[i] for i in order]
        new, start = [case["q_len"]] * b, None
    blocks = [(x + p - 1) // p for x in lens]
    wide, pages = max(blocks), sum(blocks)
    spot = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(b, wide, dtype=torch.int32, device="cuda")
    table[torch.arange(wide, device="cuda")[None] < whole(blocks)[:, None]] = spot
    # the last page and the last row of the newest blocks belong to no sequence: the plain form drops values there
    s = {"case": case, "table": table, "lens": whole(lens), "cu": whole([0] + torch.tensor(new).cumsum(0).tolist()), "max_new": max(new)}
    for name, shape in (("k", (p, d)), ("v", (p // 4, d, 4))):
        s[name + "_pages"] = torch.empty(pages + 1, kv, *shape, dtype=torch.uint8, device="cuda")
        for i in range(0, pages + 1, 4096):
            part = s[name + "_pages"][i:i + 4096]
            part.copy_((normal(*part.shape) * 36).round_().clamp_(-127, 127).add_(128))
        s[name + "_scale"] = (0.5 + torch.rand(pages + 1, kv, generator=g, device="cuda") * 1.5) / 36
        s[name + "_tail"] = normal(b + 1, 2, kv, *shape).to(t)
    if case["op"] == "attend":
        s["q"] = (normal(sum(new), case["heads"], d) * 1.5).to(t)
        return s
    x = normal(sum(new), case["heads"] + 2 * kv, d)
    x *= torch.where(torch.rand(case["heads"] + 2 * kv, d, generator=g, device="cuda") < 0.02, 6.0, 1.0)
    s["qkv"] = x.view(sum(new), -1).to(t)
    s["start"] = whole(start)
    s["read_start"] = whole([x // p * p for x in start])
    s["read_cu"] = whole([0] + torch.tensor([x % p + y for x, y in zip(start, new)]).cumsum(0).tolist())
    s["read_total"] = sum(x % p + y for x, y in zip(start, new))
    s["cos"] = s["sin"] = None
    if case["rot"]:
        turn = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        s["cos"], s["sin"] = turn.cos().float(), turn.sin().float()
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "linear": _own_linear}[op](s)
    return {"append": _plain_append, "attend": _plain_attend, "linear": _plain_linear}[op](s)


def _serving():
    import torch_transformer_benchmark

    return torch_transformer_benchmark.serving


def _own_cache(s):
    return _serving().PagedKV8(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["k_tail"], s["v_tail"], s["table"])


def _own_append(s):
    cache = _own_cache(s)
    q = cache.append(s["qkv"], s["cu"], s["start"], heads=s["case"]["heads"], cos=s["cos"], sin=s["sin"])
    k, v = cache.read(s["read_cu"], s["read_start"], s["lens"], total=s["read_total"])
    return {"q": q, "k": k, "v": v}


def _own_attend(s):
    return _own_cache(s).attend(s["q"], s["cu"], s["lens"], max_q_len=s["max_new"])


def _own_linear(s):
    return _serving().linear_int8(s["x"], s["w"], s["w_scale"], s["bias"], gelu=s["case"]["epi"] == "gelu", resid=s["resid"])


def _plain_rotate(x, cos, sin):
    half = cos.shape[-1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _plain_codes(x):
    """x [.., heads, tokens, channels] in blocks -> whole numbers in [-127, 127] and the scale of each block and head."""
    top = x.abs().amax((-2, -1))
    scale = torch.where(top.isfinite(), top * (1 / 127), torch.nan)
    codes = torch.where(scale[..., None, None] > 0, x / scale[..., None, None], 0).round().clamp(-127, 127)
    return codes, scale


def _plain_append(s):
    c, t = s["case"], s["qkv"].dtype
    h, kv, d, p, b = c["heads"], c["kv_heads"], c["dim"], c["page"], c["batch"]
    new = s["qkv"].shape[0]
    at = torch.arange(new, device="cuda")
    seq = torch.searchsorted(s["cu"][1:], at, right=True)
    pos = s["start"][seq] + at - s["cu"][seq]
    x = s["qkv"].float().view(new, h + 2 * kv, d)
    q, k, v = x[:, :h], x[:, h:h + kv], x[:, h + kv:]
    if s["cos"] is not None:
        cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
        q, k = _plain_rotate(q, cos, sin), _plain_rotate(k, cos, sin)
    q, k, v = q.to(t), k.to(t), v.to(t)
    # the touched blocks of each sequence, what was there before included
    nb = (s["max_new"] + p - 1) // p + 1
    first = s["start"] // p
    blk = first[:, None] + torch.arange(nb, device="cuda")
    full = (blk + 1) * p <= s["lens"][:, None]
    page = torch.where(full, s["table"].gather(1, blk.clamp(max=s["table"].shape[1] - 1).long()), s["k_pages"].shape[0] - 1)
    row = torch.arange(b, device="cuda")
    keep = pos // p >= ((s["lens"] - 1) // p - 1)[seq]
    to = torch.where(keep, seq, b)
    for name, val in (("k", k), ("v", v)):
        old = s[name + "_tail"][row, first % 2]
        if name == "v":
            old = old.transpose(-1, -2).reshape(b, kv, p, d)
        win = torch.zeros(b, nb * p, kv, d, dtype=t, device="cuda")
        win[:, :p] = old.transpose(1, 2)
        win[seq, pos - (first * p)[seq]] = val
        codes, scale = _plain_codes(win.view(b, nb, p, kv, d).transpose(2, 3).float())
        codes = (codes + 128).to(torch.uint8)
        if name == "v":
            codes = codes.view(b, nb, kv, p // 4, 4, d).transpose(-1, -2)
            s["v_tail"][to, pos // p % 2, :, pos % p // 4, :, pos % 4] = val
        else:
            s["k_tail"][to, pos // p % 2, :, pos % p] = val
        s[name + "_pages"][page] = codes
        s[name + "_scale"][page] = scale
    # what attention sees of these blocks
    at = torch.arange(s["read_total"], device="cuda")
    seq = torch.searchsorted(s["read_cu"][1:], at, right=True)
    pos = s["read_start"][seq] + at - s["read_cu"][seq]
    blk = pos // p
    page = s["table"][seq, blk]
    full = ((blk + 1) * p <= s["lens"][seq])[:, None, None]
    ks = torch.where(full, (s["k_pages"][page, :, pos % p].float() - 128) * s["k_scale"][page][..., None],
                     s["k_tail"][seq, blk % 2, :, pos % p].float())
    vs = torch.where(full, (s["v_pages"][page, :, pos % p // 4, :, pos % 4].float() - 128) * s["v_scale"][page][..., None],
                     s["v_tail"][seq, blk % 2, :, pos % p // 4, :, pos % 4].float())
    return {"q": q, "k": ks.to(t), "v": vs.to(t)}


def _plain_attend(s):
    c, t = s["case"], s["q"].dtype
    h, kv, d, p, b, n = c["heads"], c["kv_heads"], c["dim"], c["page"], c["batch"], c["q_len"]
    wide = s["table"].shape[1]
    row = torch.arange(b, device="cuda")
    last = s["lens"] // p
    part = (torch.arange(wide, device="cuda")[None] == last[:, None])[:, :, None, None, None]
    k = torch.where(part, s["k_tail"][row, last % 2][:, None].float(),
                    (s["k_pages"][s["table"]].float() - 128) * s["k_scale"][s["table"]][..., None, None])
    k = k.permute(0, 2, 1, 3, 4).reshape(b, kv, wide * p, d)
    v = torch.where(part[..., None], s["v_tail"][row, last % 2][:, None].float(),
                    (s["v_pages"][s["table"]].float() - 128) * s["v_scale"][s["table"]][..., None, None, None])
    v = v.permute(0, 2, 1, 3, 5, 4).reshape(b, kv, wide * p, d)
    at = torch.arange(wide * p, device="cuda")
    v = torch.where((at < s["lens"][:, None])[:, None, :, None], v, 0)  # what lies past the end is never summed
    q = s["q"].float().view(b, n, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b, kv, n * (h // kv), d)
    w = (q * (1 / math.sqrt(d))) @ k.transpose(-1, -2)
    pos = s["lens"][:, None] - n + torch.arange(n * (h // kv), device="cuda") // (h // kv)  # of each row's token
    seen = (at <= pos[:, :, None])[:, None]
    w = torch.where(seen, w, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top == -math.inf, 0, top))
    total = w.sum(-1, keepdim=True)
    out = torch.where(pos[:, None, :, None] >= 0, (w @ v) / total, 0)
    return out.view(b, kv, n, h // kv, d).permute(0, 2, 1, 3, 4).reshape(b * n, h, d).to(t)


def _plain_linear(s):
    c = s["case"]
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) * (1 / 127)
    codes = torch.where(scale > 0, x / scale, 0).round().clamp(-127, 127)
    y = (codes @ s["w"][:, :c["k"]].float().T) * scale * s["w_scale"] + s["bias"]
    if c["epi"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * (1 / math.sqrt(2))))
    if c["epi"] == "resid":
        return s["resid"] + y
    return y.to(s["x"].dtype)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "linear": _exact_linear}[case["op"]](s, case)


def _exact_quantized(x):
    """x [tokens, heads, channels] of one whole block, fp64 -> the values its codes stand for."""
    step = x.abs().amax((0, 2), keepdim=True) / 127
    return torch.where(step > 0, (x / step).round() * step, 0)


def _exact_append(s, c):
    h, kv, d, p, t = c["heads"], c["kv_heads"], c["dim"], c["page"], s["qkv"].dtype
    lens, start, cu = s["lens"].tolist(), s["start"].tolist(), s["cu"].tolist()
    qs, ks, vs = [], [], []
    for i in range(c["batch"]):
        x = s["qkv"][cu[i]:cu[i + 1]].double().view(-1, h + 2 * kv, d)
        q, k, v = x.split([h, kv, kv], 1)
        if c["rot"]:
            # the tables are inputs: their values as given
            turn = torch.complex(s["cos"][start[i]:lens[i]].double(), s["sin"][start[i]:lens[i]].double())[:, None]
            half = c["rot"] // 2
            turned = []
            for y in (q, k):
                z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
                turned.append(torch.cat([z.real, z.imag, y[..., 2 * half:]], -1))
            q, k = turned
        qs.append(q)
        first, before = start[i] // p, start[i] % p
        for name, new, to in (("k", k, ks), ("v", v, vs)):
            old = s[name + "_tail"][i, first % 2]
            if name == "v":
                old = old.permute(0, 1, 3, 2).reshape(kv, p, d)
            y = torch.cat([old[:, :before].transpose(0, 1).double(), new.to(t).double()])
            whole = y.shape[0] // p * p
            z = y[:whole].view(-1, p, kv, d).transpose(0, 1).reshape(p, -1, d)  # every block and head has its own step
            to.append(_exact_quantized(z).view(p, -1, kv, d).transpose(0, 1).reshape(whole, kv, d) if whole else y[:0])
            to.append(y[whole:])
    return {"q": torch.cat(qs), "k": torch.cat(ks), "v": torch.cat(vs)}


def _exact_attend(s, c):
    kv, d, p, n = c["kv_heads"], c["dim"], c["page"], c["q_len"]
    g = c["heads"] // kv
    if 16 * d * c["heads"] * n * sum(s["lens"].tolist()) > 1e13:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(s["lens"].tolist()):
        page = s["table"][i, :length // p].long()
        for j in range(kv):
            k = ((s["k_pages"][page, j].double() - 128) * s["k_scale"][page, j].double()[:, None, None]).reshape(-1, d)
            v = ((s["v_pages"][page, j].double() - 128) * s["v_scale"][page, j].double()[:, None, None, None])
            v = v.transpose(-1, -2).reshape(-1, d)
            slot = length // p % 2
            k = torch.cat([k, s["k_tail"][i, slot, j, :length % p].double()])
            v = torch.cat([v, s["v_tail"][i, slot, j].transpose(-1, -2).reshape(p, d)[:length % p].double()])
            for r in range(max(0, n - length), n, 256):  # tokens that see nothing keep their zeros
                e = min(n, r + 256)
                q = s["q"][i * n + r:i * n + e, j * g:(j + 1) * g].double()
                w = torch.einsum("qgd,kd->qgk", q, k) / math.sqrt(d)
                later = torch.arange(length, device="cuda") > torch.arange(length - n + r, length - n + e, device="cuda")[:, None]
                w.masked_fill_(later[:, None], -math.inf)
                out[i * n + r:i * n + e, j * g:(j + 1) * g] = torch.softmax(w, -1) @ v
    return out


def _exact_linear(s, c):
    outs = []
    w = s["w"][:, :c["k"]].double() * s["w_scale"].double()[:, None]
    for i in range(0, c["rows"], 4096):
        x = s["x"][i:i + 4096].double()
        step = x.abs().amax(1, keepdim=True) / 127
        y = (torch.where(step > 0, (x / step).round(), 0) @ w.T) * step + s["bias"].double()
        if c["epi"] == "gelu":
            y = torch.nn.functional.gelu(y)
        outs.append(y + s["resid"][i:i + 4096].double() if c["epi"] == "resid" else y)
    return torch.cat(outs)
