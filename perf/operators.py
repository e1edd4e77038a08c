"""What is measured of the text encoder's operators, with their plain forms in torch.

Three operators of a decoder-only text encoder that feeds the denoiser, as a server of prompts calls them:

norm    residual addition and root-mean-square norm, written in 32 or 16 bits, or in 8 bits (e4m3) with scales
rotary  rotary positions of the new queries and keys, and the append of keys and values to a paged cache
attend  causal attention of a chunk of new tokens (or of single tokens) over a paged cache, with an optional
        sliding window, first tokens that stay visible (sinks) and a soft cap on the scores

``listed()`` gives the cases, ``draw()`` more of the same ranges, ``prepare()`` what a program holds before the call,
``run()`` one pass, ``work()`` what a pass cannot do without and ``exact()`` the result in 64 bits.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
SCALE_FLOOR = 2.0 ** -100  # smallest scale of an 8-bit group: its reciprocal stays finite
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "bf16": 2, "e4m3": 1}


# --- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new token of one sequence: the smallest norm of a decoding step (2304 channels: the encoder's hidden size)
        {"name": "norm one token", "op": "norm", "rows": 1, "channels": 2304, "x": "bf16", "residual": "f32", "out": "bf16",
         "group": 0, "offset": 1.0},
        # odd sizes in the 32-bit check mode
        {"name": "norm odd f32", "op": "norm", "rows": 777, "channels": 1153, "x": "f32", "residual": "f32", "out": "f32",
         "group": 0, "offset": 0.0},
        # 128 sequences (64 prompt pairs) of 300 tokens, 8-bit operand of the next product, a scale per 128 channels
        {"name": "norm pairs 8 bit", "op": "norm", "rows": 38400, "channels": 2304, "x": "bf16", "residual": "f32",
         "out": "e4m3", "group": 128, "offset": 1.0},
        # a decoding step of 64 sequences far into their caches, half layout, whole head
        {"name": "rotary decode", "op": "rotary", "dtype": "bf16", "sequences": 64, "new_lo": 1, "new_hi": 1, "past_lo": 100,
         "past_hi": 130000, "heads": 8, "kv_heads": 4, "head_dim": 256, "rotated": 256, "interleaved": False,
         "stretch": 8.0, "page": 64, "cache": 2000},
        # prompts of 8 to 120 tokens behind a shared prefix, interleaved layout, half of the head, 32-bit check mode
        {"name": "rotary prompts f32", "op": "rotary", "dtype": "f32", "sequences": 16, "new_lo": 8, "new_hi": 120,
         "past_lo": 211, "past_hi": 211, "heads": 12, "kv_heads": 3, "head_dim": 96, "rotated": 48, "interleaved": True,
         "stretch": 1.0, "page": 16, "cache": 1000},
        # 128 sequences of up to 512 new tokens
        {"name": "rotary chunks", "op": "rotary", "dtype": "bf16", "sequences": 128, "new_lo": 200, "new_hi": 512,
         "past_lo": 0, "past_hi": 3000, "heads": 16, "kv_heads": 4, "head_dim": 128, "rotated": 128, "interleaved": False,
         "stretch": 4.0, "page": 16, "cache": 30000},
        # the smallest attention: one token of one sequence over a prompt's cache
        {"name": "attend one token", "op": "attend", "dtype": "bf16", "sequences": 1, "new_lo": 1, "new_hi": 1,
         "past_lo": 299, "past_hi": 299, "heads": 8, "kv_heads": 4, "head_dim": 256, "window": 0, "sinks": 0, "cap": 50.0,
         "page": 16},
        # a decoding step of 64 sequences of very different lengths
        {"name": "attend decode batch", "op": "attend", "dtype": "bf16", "sequences": 64, "new_lo": 1, "new_hi": 1,
         "past_lo": 100, "past_hi": 16000, "heads": 16, "kv_heads": 4, "head_dim": 128, "window": 0, "sinks": 0, "cap": 0.0,
         "page": 16},
        # one long sequence: the cache's axis has to be split to fill the card
        {"name": "attend decode long", "op": "attend", "dtype": "bf16", "sequences": 1, "new_lo": 1, "new_hi": 1,
         "past_lo": 131071, "past_hi": 131071, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0, "sinks": 0,
         "cap": 0.0, "page": 64},
        # 32-bit check mode: short prompts, odd page and head sizes
        {"name": "attend prompts f32", "op": "attend", "dtype": "f32", "sequences": 4, "new_lo": 8, "new_hi": 120,
         "past_lo": 100, "past_hi": 180, "heads": 6, "kv_heads": 2, "head_dim": 72, "window": 0, "sinks": 0, "cap": 0.0,
         "page": 24},
        # 64 prompts of up to 300 tokens behind an instruction prefix
        {"name": "attend prompts", "op": "attend", "dtype": "bf16", "sequences": 64, "new_lo": 8, "new_hi": 300,
         "past_lo": 211, "past_hi": 211, "heads": 8, "kv_heads": 4, "head_dim": 256, "window": 0, "sinks": 0, "cap": 50.0,
         "page": 16},
        # a chunk of 4096 tokens late in a long document, sliding window with sinks
        {"name": "attend chunk window", "op": "attend", "dtype": "bf16", "sequences": 2, "new_lo": 4000, "new_hi": 4096,
         "past_lo": 12288, "past_hi": 28672, "heads": 16, "kv_heads": 4, "head_dim": 128, "window": 8192, "sinks": 4,
         "cap": 0.0, "page": 64},
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "attend", "attend"])
    if op == "norm":
        channels = rng.choice([_between(rng, 64, 8192), 8 * _between(rng, 8, 1024), 2304])
        out = rng.choice(["f32", "bf16", "bf16", "e4m3", "e4m3"])
        return {"op": "norm", "rows": _between(rng, 1, max(2, 80_000_000 // channels)), "channels": channels,
                "x": rng.choice(["f32", "bf16", "bf16"]), "residual": rng.choice(["f32", "bf16"]), "out": out,
                "group": rng.choice([0, 64, 128]) if out == "e4m3" else 0, "offset": rng.choice([0.0, 1.0])}
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    head_dim = rng.choice([64, 72, 96, 128, 128, 256])
    c = {"op": op, "dtype": rng.choice(["bf16", "bf16", "bf16", "f32"])}
    group = rng.choice([1, 2, 3, 4, 8])
    if op == "rotary":
        c |= {"sequences": _between(rng, 1, 128)}
        new_hi = rng.choice([1, _between(rng, 2, 512)])
        past_hi = _between(rng, 1, 130000)
        c |= {"new_lo": rng.randint(1, new_hi), "new_hi": new_hi, "past_lo": rng.randint(0, past_hi), "past_hi": past_hi,
              "heads": kv_heads * min(group, 4), "kv_heads": min(kv_heads, 4), "head_dim": min(head_dim, 128)}
        c["heads"] = c["kv_heads"] * min(group, 4)
        c |= {"rotated": rng.choice([c["head_dim"], c["head_dim"] // 2]), "interleaved": rng.random() < 0.5,
              "stretch": rng.choice([1.0, 4.0, 8.0]), "page": rng.choice([16, 24, 64, 128])}
        c["cache"] = 2 * (c["sequences"] * (new_hi // c["page"] + 2)) + rng.randint(1, 99)
        return c
    kind = rng.choice(["decode", "prompts", "chunk"])
    if kind == "decode":
        sequences = _between(rng, 1, 96)
        past_hi = _between(rng, 16, max(17, min(131000, 500_000_000 // (sequences * kv_heads * head_dim * 4))))
        new_hi = rng.choice([1, 1, 2, 4])
    elif kind == "prompts":
        sequences, new_hi, past_hi = _between(rng, 1, 48), rng.randint(9, 300), rng.choice([0, 64, 211, 500])
    else:
        sequences, new_hi, past_hi = rng.randint(1, 2), _between(rng, 512, 3000), _between(rng, 16, 12000)
    if c["dtype"] == "f32":  # the check mode runs short sequences
        sequences, new_hi, past_hi = min(sequences, 8), min(new_hi, 150), min(past_hi, 600)
    windowed = rng.random() < 0.4
    return c | {"sequences": sequences, "new_lo": rng.randint(max(1, new_hi // 3), new_hi), "new_hi": new_hi,
                "past_lo": rng.randint(past_hi // 3, past_hi), "past_hi": past_hi, "heads": kv_heads * group,
                "kv_heads": kv_heads, "head_dim": head_dim, "window": _between(rng, 8, 5000) if windowed else 0,
                "sinks": rng.choice([0, 1, 4]) if windowed else 0, "cap": rng.choice([0.0, 0.0, 50.0]),
                "page": rng.choice([16, 16, 24, 32, 64, 128])}


def _lengths(case):
    """(new tokens, tokens before them) of each sequence: spread evenly over their ranges, in no order."""
    n = case["sequences"]
    new = [case["new_hi"] if i == 0 else case["new_lo"] + int((case["new_hi"] - case["new_lo"] + 1) * (i * 0.6180339887 % 1.0))
           for i in range(n)]
    past = [case["past_hi"] if i == 0 else case["past_lo"] + int((case["past_hi"] - case["past_lo"] + 1) * (i * 0.7548776662 % 1.0))
            for i in range(n)]
    return new, past


# --- inputs ----------------------------------------------------------------------------------------------------------

def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _frequencies(case):
    """Angles per position of the rotated pairs, in 64 bits: base 10000; the pairs that turn less than once over 4096
    positions are slowed by `stretch`, those that turn more than 32 times are left, and between the two it goes over evenly."""
    n = case["rotated"] // 2
    f = 10000.0 ** (-torch.arange(n, dtype=torch.float64) / n)
    keep = ((4096.0 * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return (f * keep + f / case["stretch"] * (1.0 - keep)).cuda()


def _paged(case, gen):
    """The batch's bookkeeping on the device: rows, lengths and page numbers. Pages are handed out in no order. The append
    touches the pages of new tokens alone: there the table's other entries stay zero, and the pool holds no pages for them."""
    new, past = _lengths(case)
    page = case["page"]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    kv = [n + p for n, p in zip(new, past)]
    first = [p // page if case["op"] == "rotary" else 0 for p in past]
    need = [-(-k // page) for k in kv]
    total = sum(n - f for n, f in zip(need, first))
    pages = max(total, case.get("cache", 0))
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(new), max(need), dtype=torch.int32)
    at, spans = 0, []
    for n, f in zip(need, first):
        spans.append((f, n, at))
        at += n - f
    order = order.cpu()
    for s, (f, n, a) in enumerate(spans):
        table[s, f:n] = order[a:a + n - f]
    to = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"row_start": to(starts), "kv_len": to(kv), "page_table": table.cuda(), "max_new": max(new), "max_kv": max(kv),
            "rows": starts[-1], "pages": pages}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": dict(case)}
    if case["op"] == "norm":
        rows, c = case["rows"], case["channels"]
        s["x"] = _normal(gen, (rows, c), DTYPES[case["x"]])
        s["residual"] = _normal(gen, (rows, c), DTYPES[case["residual"]], 3.0)
        s["weight"] = _normal(gen, (c,), torch.float32, 0.2) + (1.0 - case["offset"])
        return s
    dtype, d = DTYPES[case["dtype"]], case["head_dim"]
    s |= _paged(case, gen)
    pool = (s["pages"], case["page"], case["kv_heads"], d)
    s["k_cache"], s["v_cache"] = _normal(gen, pool, dtype), _normal(gen, pool, dtype)
    s["q"] = _normal(gen, (s["rows"], case["heads"], d), dtype, 1.0 if case["op"] == "rotary" else 2.0)
    if case["op"] == "rotary":
        s["k"], s["v"] = (_normal(gen, (s["rows"], case["kv_heads"], d), dtype) for _ in range(2))
        s["frequencies"] = _frequencies(case)
    return s


# --- one pass --------------------------------------------------------------------------------------------------------

_handles = {}


def _handle():
    """The framework's handle of this process, on the stream that torch works on."""
    if not _handles:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.getcwd(), "sana.cpp_b200"))
        from sana_b200 import SanaCuda
        g = SanaCuda(torch.cuda.current_device())
        g.set_stream(torch.cuda.current_stream().cuda_stream or 1)  # 1: CUDA's legacy default stream
        _handles["g"] = g
    return _handles["g"]


def run(state):
    return {"norm": _norm, "rotary": _rotary, "attend": _attend}[state["case"]["op"]](state)


def _norm(s):
    case = s["case"]
    if own:
        return _handle().add_rms_norm_device(s["x"], s["residual"], s["weight"], eps=1e-6, weight_offset=case["offset"],
                                             out_dtype=DTYPES[case["out"]], group=case["group"])
    h = (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)  # the stream is held in the residual's type
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * (s["weight"] + case["offset"])
    if case["out"] != "e4m3":
        return y.to(DTYPES[case["out"]]), h
    rows, c = y.shape
    g = case["group"] or c
    n = -(-c // g)
    z = torch.nn.functional.pad(y, (0, n * g - c)).view(rows, n, g)
    scale = (z.abs().amax(-1) / E4M3_MAX).clamp(min=SCALE_FLOOR)
    q = (z / scale[..., None]).view(rows, n * g)[:, :c].to(torch.float8_e4m3fn)
    return q, scale, h


def _places(s):
    """For each row its sequence, and its position in that sequence."""
    row = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["row_start"][1:].contiguous(), row, right=True)
    return seq, (s["kv_len"] - s["row_start"][1:])[seq] + row


def _turn(x, cos, sin, rotated, interleaved):
    x = x.float()
    r, rest = x[..., :rotated], x[..., rotated:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :rotated // 2], r[..., rotated // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((r, rest), -1)


def _rotary(s):
    case = s["case"]
    if own:
        q = _handle().rotary_append_device(s["q"], s["k"], s["v"], s["frequencies"], s["k_cache"], s["v_cache"], s["row_start"],
                                           s["kv_len"], s["page_table"], s["max_new"], interleaved=case["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    seq, pos = _places(s)
    angle = pos.double()[:, None, None] * s["frequencies"]  # 64 bits: far positions lose the angle in 32
    cos, sin = angle.cos().float(), angle.sin().float()
    page = case["page"]
    at = s["page_table"][seq, torch.div(pos, page, rounding_mode="floor").long()].long(), (pos % page).long()
    s["k_cache"][at] = _turn(s["k"], cos, sin, case["rotated"], case["interleaved"]).to(s["k"].dtype)
    s["v_cache"][at] = s["v"]
    return _turn(s["q"], cos, sin, case["rotated"], case["interleaved"]).to(s["q"].dtype), s["k_cache"], s["v_cache"]


def _attend(s):
    case = s["case"]
    if own:
        return _handle().paged_attention_device(s["q"], s["k_cache"], s["v_cache"], s["row_start"], s["kv_len"], s["page_table"],
                                                s["max_new"], s["max_kv"], window=case["window"], sinks=case["sinks"],
                                                softcap=case["cap"])
    n, h, hk, d = case["sequences"], case["heads"], case["kv_heads"], case["head_dim"]
    new, kv = s["max_new"], s["max_kv"]
    row = (s["row_start"][:-1, None] + torch.arange(new, device="cuda")).clamp(max=s["rows"] - 1)
    pos = (s["kv_len"] - s["row_start"].diff())[:, None] + torch.arange(new, device="cuda")  # [n, new]
    q = s["q"][row].float().view(n, new, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(n, hk, h // hk * new, d)
    k, v = (c[s["page_table"].long()].flatten(1, 2)[:, :kv].permute(0, 2, 1, 3).float() for c in (s["k_cache"], s["v_cache"]))
    key = torch.arange(kv, device="cuda")
    v = v.masked_fill((key >= s["kv_len"][:, None])[:, None, :, None], 0.0)  # behind the last token: anything
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(d ** -0.5)
    del k
    if case["cap"]:
        score = score.div_(case["cap"]).tanh_().mul_(case["cap"])
    seen = key <= pos[..., None]
    if case["window"]:
        seen &= (key > pos[..., None] - case["window"]) | (key < case["sinks"])
    score = score.view(n, hk, h // hk, new, kv).masked_fill_(~seen[:, None, None], -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(n, hk, -1, kv), v).view(n, hk, h // hk, new, d) / total.clamp(min=1e-30)
    seq, at = _places(s)
    at = at - pos[:, 0][seq]
    return o[seq, :, :, at].flatten(1, 2).to(s["q"].dtype)


# --- what a pass cannot do without -----------------------------------------------------------------------------------

def _seen(case, new, past):
    """(pairs of a new token and a token that it sees, tokens of the cache that some new token sees) of one sequence."""
    w, k = case["window"], case["sinks"]
    pairs = 0
    if not w:
        return new * past + new * (new + 1) // 2, past + new
    for p in range(past, past + new):
        lo = max(0, p - w + 1)
        pairs += p + 1 - lo + min(k, lo)
    lo = max(0, past - w + 1)
    return pairs, past + new - lo + min(k, lo)


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["channels"]
        scales = case["rows"] * (-(-case["channels"] // (case["group"] or case["channels"]))) * 4 if case["out"] == "e4m3" else 0
        return {"bytes": n * (BYTES[case["x"]] + 2 * BYTES[case["residual"]] + BYTES[case["out"]]) + scales + 4 * case["channels"],
                "flops": 6 * n}
    new, past = _lengths(case)
    rows, d, size = sum(new), case["head_dim"], BYTES[case["dtype"]]
    if case["op"] == "rotary":
        n = rows * d * (case["heads"] + 2 * case["kv_heads"])
        return {"bytes": 2 * n * size, "flops": 3 * rows * case["rotated"] * (case["heads"] + case["kv_heads"])}
    seen = [_seen(case, n, p) for n, p in zip(new, past)]
    return {"bytes": (2 * rows * case["heads"] + 2 * sum(k for _, k in seen) * case["kv_heads"]) * d * size,
            "flops": 4 * case["heads"] * d * sum(p for p, _ in seen)}


# --- the result in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = (s["x"].double() + s["residual"].double()).to(s["residual"].dtype)
        z = h.double()
        y = z / (z.pow(2).sum(-1, keepdim=True) / z.shape[-1] + 1e-6).sqrt() * (s["weight"].double() + case["offset"])
        if case["out"] != "e4m3":
            return y, z
        parts = y.split(case["group"] or y.shape[-1], dim=-1)
        scales = [(p.abs().max(-1, keepdim=True).values / E4M3_MAX).clamp_min(SCALE_FLOOR) for p in parts]
        q = torch.cat([(p / t).float().to(torch.float8_e4m3fn).double() for p, t in zip(parts, scales)], -1)
        return q, torch.cat(scales, -1), z
    new, past = _lengths(case)
    page, d, hk = case["page"], case["head_dim"], case["kv_heads"]
    table = s["page_table"].long()
    row = 0
    if case["op"] == "rotary":
        kc, vc, qo = s["k_cache"].double(), s["v_cache"].double(), s["q"].double()
        half = case["rotated"] // 2
        first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        for i, (n, p) in enumerate(zip(new, past)):
            pos = torch.arange(p, p + n, device="cuda")
            turn = torch.polar(torch.ones(n, 1, half, dtype=torch.float64, device="cuda"),
                               pos.double()[:, None, None] * s["frequencies"])
            page_of, slot = table[i, pos // page], pos % page
            for x, to in ((s["q"], None), (s["k"], kc)):
                x = x[row:row + n].double()
                z = torch.complex(x[..., first], x[..., second]) * turn
                x[..., first], x[..., second] = z.real, z.imag
                if to is None:
                    qo[row:row + n] = x
                else:
                    to[page_of, slot] = x
            vc[page_of, slot] = s["v"][row:row + n].double()
            row += n
        return qo, kc, vc
    if work(case)["flops"] > 4e12:
        return None
    out = torch.zeros(s["rows"], case["heads"], d, dtype=torch.float64, device="cuda")
    g = case["heads"] // hk
    for i, (n, p) in enumerate(zip(new, past)):
        at = table[i, :-(-(n + p) // page)]
        k, v = (c[at].reshape(-1, hk, d)[:n + p].double() for c in (s["k_cache"], s["v_cache"]))
        me, key = torch.arange(p, p + n, device="cuda")[:, None], torch.arange(n + p, device="cuda")
        hidden = key > me
        if case["window"]:
            hidden |= (key <= me - case["window"]) & (key >= case["sinks"])
        for h in range(case["heads"]):
            t = s["q"][row:row + n, h].double() @ k[:, h // g].T / math.sqrt(d)
            if case["cap"]:
                t = case["cap"] * torch.tanh(t / case["cap"])
            t[hidden] = -math.inf
            out[row:row + n, h] = torch.softmax(t, -1) @ v[:, h // g]
        row += n
    return out
