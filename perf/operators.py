"""Cases and plain forms of the paged 8-bit KV cache operators.

Four operators make one serving step over a cache whose keys and values are
held in 8 bits:

  rope     rotary positions: interleaved or half layout, the whole head or a
           part of it, frequencies as trained or scaled for long contexts, and
           the transposed map (its gradient)
  pages    block tables, slot maps and row positions of one step from request
           lengths, with pages taken from and returned to a free list
  append   rows quantised into their pages under one scale per page and head,
           pages requantised when their scale grows, and rows read back
  attend   grouped-query causal attention over the pages: one query per
           sequence (decode) or many (prompt chunks)

The cache: codes [n_pages][n_kv][page][d] (signed bytes or e4m3), scales
[n_pages][n_kv] in fp32; token t of a sequence lies in page table[t / page] at
t % page.  A value is code * scale.

`run` computes an operator with elementary torch operations, or (`own`) with
the library's entry points.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
LLAMA3 = {"factor": 32.0, "low": 1.0, "high": 4.0, "original": 8192}
YARN = {"factor": 4.0, "fast": 32.0, "slow": 1.0, "original": 8192}
CODE_MAX = {"i8": 127.0, "e4m3": 448.0}


# ------------------------------------------------------------------- cases

def listed():
    return [
        # One decode step of 64 sequences: query and key heads of a token side by side.
        {"name": "rope-decode", "op": "rope", "rows": 64, "heads": 40, "d": 64, "rot": 64, "layout": "interleaved",
         "scaling": "llama3", "type": "f32", "far": 131072, "transpose": False},
        # A prompt batch in half precision, half layout.
        {"name": "rope-prompt", "op": "rope", "rows": 16384, "heads": 40, "d": 64, "rot": 64, "layout": "half",
         "scaling": "llama3", "type": "f16", "far": 131072, "transpose": False},
        # The gradient of a partly rotated wide head with stretched frequencies.
        {"name": "rope-grad-part", "op": "rope", "rows": 2047, "heads": 40, "d": 128, "rot": 96, "layout": "half",
         "scaling": "yarn", "type": "f32", "far": 32768, "transpose": True},
        # The bookkeeping of one decode step: 64 sequences, one token each.
        {"name": "pages-decode", "op": "pages", "n": 64, "hi": 2048, "new": 1, "ended": 2, "page": 32, "ragged": 3},
        # A large mixed step: prompts arriving, sequences growing and ending.
        {"name": "pages-mixed", "op": "pages", "n": 1777, "hi": 4096, "new": 100, "ended": 90, "page": 16,
         "ragged": 5},
        # 64 sequences add one token each, fp32 rows as the engine makes them.
        {"name": "append-decode", "op": "append", "n": 64, "hi": 2048, "new": 1, "kv": 8, "d": 64, "page": 32,
         "fmt": "i8", "type": "f32", "ragged": 7},
        # Ragged prompt chunks written at once.
        {"name": "append-prompt", "op": "append", "n": 24, "hi": 1000, "new": 1365, "kv": 8, "d": 64, "page": 32,
         "fmt": "e4m3", "type": "f16", "ragged": 8},
        # One long conversation: a single query over 128 Ki positions.
        {"name": "attend-long", "op": "attend", "n": 1, "lo": 131071, "hi": 131071, "new": 1, "heads": 32, "kv": 8,
         "d": 64, "page": 64, "fmt": "i8", "type": "f32", "ragged": 11},
        # Serving: 64 sequences of very different lengths.
        {"name": "attend-serve", "op": "attend", "n": 64, "lo": 1, "hi": 8191, "new": 1, "heads": 32, "kv": 8,
         "d": 64, "page": 32, "fmt": "i8", "type": "f32", "ragged": 12},
        # Many short sequences of a wider model, e4m3 codes, half precision rows.
        {"name": "attend-short-wide", "op": "attend", "n": 200, "lo": 0, "hi": 333, "new": 1, "heads": 32, "kv": 8,
         "d": 128, "page": 16, "fmt": "e4m3", "type": "f16", "ragged": 13},
        # Prompt chunks of a few sequences over what they hold already.
        {"name": "attend-chunks", "op": "attend", "n": 6, "lo": 500, "hi": 4000, "new": 333, "heads": 32, "kv": 8,
         "d": 64, "page": 32, "fmt": "i8", "type": "f16", "ragged": 14},
        # One long prompt in fp32.
        {"name": "attend-prompt", "op": "attend", "n": 1, "lo": 4096, "hi": 4096, "new": 4096, "heads": 32, "kv": 8,
         "d": 64, "page": 32, "fmt": "i8", "type": "f32", "ragged": 15},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "pages", "append", "attend", "attend", "attend"])
    ragged = rng.randrange(1 << 20)
    if op == "rope":
        d = rng.choice([64, 128])
        return {"op": op, "rows": _log(rng, 1, 16384 * 64 // d // 2), "heads": rng.choice([8, 9, 32, 40]), "d": d,
                "rot": rng.choice([d, d, d // 2, d * 3 // 4]), "layout": rng.choice(["interleaved", "half"]),
                "scaling": rng.choice(["none", "linear", "llama3", "yarn"]), "type": rng.choice(["f32", "f16"]),
                "far": _log(rng, 16, 1 << 20), "transpose": rng.random() < 0.3}
    if op == "pages":
        n = _log(rng, 1, 1777)
        return {"op": op, "n": n, "hi": _log(rng, 1, 4096), "new": _log(rng, 1, 100),
                "ended": rng.randint(0, n // 8), "page": rng.choice([16, 32, 64, 128]), "ragged": ragged}
    if op == "append":
        n = _log(rng, 1, 256)
        return {"op": op, "n": n, "hi": _log(rng, 1, 2048), "new": _log(rng, 1, max(1, 16384 // n)),
                "kv": rng.choice([1, 4, 8]), "d": rng.choice([64, 128]), "page": rng.choice([16, 32, 64, 128]),
                "fmt": rng.choice(["i8", "e4m3"]), "type": rng.choice(["f32", "f16"]), "ragged": ragged}
    kv, group = rng.choice([(8, 4), (8, 4), (8, 3), (4, 8), (8, 1), (2, 6)])
    c = {"op": op, "heads": kv * group, "kv": kv, "d": rng.choice([64, 64, 128]),
         "page": rng.choice([16, 32, 64, 128]), "fmt": rng.choice(["i8", "e4m3"]),
         "type": rng.choice(["f32", "f16"]), "ragged": ragged}
    if rng.random() < 0.6:  # decode
        n = _log(rng, 1, 200)
        hi = _log(rng, 1, min(131072, 262144 // n) * 64 // c["d"])
        return {**c, "n": n, "lo": rng.choice([0, 1, hi]) if hi > 1 else hi, "hi": hi, "new": rng.choice([1, 1, 1, 2])}
    n = _log(rng, 1, 24)
    new = _log(rng, 3, 4096 // n)
    pairs = 4096 * 2048 * 32 // c["heads"] * 64 // c["d"]  # of the largest listed case
    return {**c, "n": n, "lo": 0, "hi": _log(rng, min(new, pairs // (n * new)), min(16384, pairs // (n * new))), "new": new}


def _lengths(case):
    """(tokens held, tokens added) of each sequence; -1 added: the sequence ends.  From the case alone."""
    r = random.Random(case["ragged"])
    n, hi, new = case["n"], case["hi"], case["new"]
    if case["op"] == "attend":  # lengths count the step's own tokens
        total = [r.randint(case["lo"], hi) for _ in range(n)]
        add = [new if new <= 2 or n == 1 else r.randint(1, 2 * new - 1) for _ in range(n)]
        return [max(0, t - a) for t, a in zip(total, add)], [min(a, t) if new > 2 else a for t, a in zip(total, add)]
    held = [r.randint(0, hi) for _ in range(n)]
    add = [new if new <= 2 else r.randint(0, 2 * new) for _ in range(n)]
    for s in r.sample(range(n), case.get("ended", 0)):
        add[s] = -1
    return held, add


def _elem(case):
    return 2 if case.get("type") == "f16" else 4


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["rows"] * case["heads"] * case["d"]
        return {"bytes": 2.0 * n * _elem(case) + 4.0 * case["rows"],
                "flops": 3.0 * case["rows"] * case["heads"] * case["rot"]}
    held, add = _lengths(case)
    page = case["page"]
    if op == "pages":
        tokens = sum(max(0, a) for a in add)
        fresh = sum(-(-(h + a) // page) - -(-h // page) for h, a in zip(held, add) if a > 0)
        back = sum(-(-h // page) for h, a in zip(held, add) if a < 0)
        return {"bytes": 4.0 * (4 * len(held) + 4 * tokens + 2 * fresh + 2 * back), "flops": 0}
    kv, d = case["kv"], case["d"]
    if op == "append":
        tokens = sum(add)
        back = sum(h + a - h // page * page for h, a in zip(held, add) if a > 0)
        pages = sum(-(-(h + a) // page) - h // page for h, a in zip(held, add) if a > 0)
        # rows in; the touched tokens' codes out once and in once; rows read back
        return {"bytes": 2.0 * kv * d * (tokens * _elem(case) + back * 2 + back * 4) + 16.0 * pages * kv,
                "flops": 4.0 * kv * d * tokens}
    heads = case["heads"]
    rows = sum(add) if case["new"] > 2 else case["new"] * case["n"]
    total = sum(h + a for h, a in zip(held, add)) if case["new"] > 2 else sum(_attend_lens(case)[0])
    pairs = sum(sum(max(0, t - q + j + 1) for j in range(q)) for t, q in zip(*_attend_lens(case)))
    return {"bytes": 2.0 * total * kv * d + 8.0 * total / page * kv + 2.0 * rows * heads * d * _elem(case),
            "flops": 4.0 * d * heads * pairs}


def _attend_lens(case):
    """(positions held once the step's tokens are in, queries) of each sequence."""
    r = random.Random(case["ragged"])
    n, new = case["n"], case["new"]
    total = [r.randint(case["lo"], case["hi"]) for _ in range(n)]
    q = [new if new <= 2 or n == 1 else r.randint(1, 2 * new - 1) for _ in range(n)]
    if new > 2:
        q = [min(a, t) for a, t in zip(q, total)]
    return total, q


# ------------------------------------------------------------------ inputs

def _dtype(case):
    return torch.float16 if case["type"] == "f16" else torch.float32


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _codes(shape, fmt, g):
    """Codes as values of a bell with the page's largest value near the end of the range."""
    x = torch.randn(shape, device=DEV, generator=g) * (CODE_MAX[fmt] / 3.5)
    if fmt == "i8":
        return x.round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    return x.clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _tables(totals, page, slack, g):
    """A random placement of pages: table [n][stride], the number of pages, and the pages left over."""
    need = [-(-t // page) for t in totals]
    n_pages = sum(need) + slack
    perm = torch.randperm(n_pages, generator=g).to(torch.int32)
    stride = max(1, max(need))
    table = np.full((len(totals), stride), -1, np.int32)
    at, p = 0, perm.numpy()
    for s, k in enumerate(need):
        table[s, :k] = p[at:at + k]
        at += k
    return torch.from_numpy(table).to(DEV), n_pages, perm[at:].contiguous().to(DEV)


def _pool(n_pages, case, g):
    kv, page, d, fmt = case["kv"], case["page"], case["d"], case["fmt"]
    pool = {}
    for name in ("k", "v"):
        pool[name] = _codes((n_pages, kv, page, d), fmt, g)
        pool[name + "_scale"] = (3.5 / CODE_MAX[fmt]) * torch.exp(0.3 * torch.randn(n_pages, kv, device=DEV, generator=g))
    return pool


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    gc = torch.Generator().manual_seed(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "rope":
        shape = (case["rows"], case["heads"], case["d"])
        s["x"] = torch.randn(shape, device=DEV, generator=g).to(_dtype(case))
        s["y"] = torch.zeros_like(s["x"])
        s["pos"] = torch.randint(0, case["far"], (case["rows"],), dtype=torch.int32, device=DEV, generator=g)
        return s
    if op == "attend":
        totals, q = _attend_lens(case)
        held, add = totals, q
    else:
        held, add = _lengths(case)
        totals = [h + max(0, a) for h, a in zip(held, add)]
    page = case["page"]
    if op == "pages":
        table, n_pages, rest = _tables(held, page, sum(-(-t // page) for t in totals) + 3, gc)
        stride = max(1, max(-(-t // page) for t in totals)) + 1
        wide = torch.full((case["n"], stride), -1, dtype=torch.int32, device=DEV)
        wide[:, :table.shape[1]] = table
        tokens = sum(max(0, a) for a in add)
        cap = tokens + 5  # a padded batch
        free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
        free[:len(rest)] = rest
        new = {k: torch.zeros(c, dtype=torch.int32, device=DEV) for k, c in
               (("lens_out", case["n"]), ("q_start", case["n"] + 1), ("slots", cap), ("positions", cap),
                ("seq_ids", cap), ("free_count_out", 1), ("status", 2))}
        return {**s, "lens": _ints(held), "n_new": _ints(add), "table": wide, "free_list": free,
                "free_count": _ints([len(rest)]), "n_pages": n_pages, **new}
    table, n_pages, _ = _tables(totals, page, 7, gc)
    s |= {"table": table, "n_pages": n_pages, **_pool(n_pages, case, g)}
    if op == "append":
        kv, d = case["kv"], case["d"]
        tab = table.cpu().numpy()
        slot = lambda i, t: tab[i, t // page].astype(np.int64) * page + t % page  # noqa: E731
        spans = [(i, h, h + a) for i, (h, a) in enumerate(zip(held, add)) if a > 0]
        at = [slot(i, np.arange(b, e)) for i, b, e in spans] or [np.zeros(0, np.int64)]
        back = [slot(i, np.arange(b // page * page, e)) for i, b, e in spans] or [np.zeros(0, np.int64)]
        s["slots"], s["back"] = _ints(np.concatenate(at)), _ints(np.concatenate(back))
        for name in ("k", "v"):
            x = torch.randn(len(s["slots"]), kv, d, device=DEV, generator=g)
            # keys have a few channels that are much larger than the rest
            x[:, :, : d // 16] *= 4.0
            s[name + "_rows"] = x.to(_dtype(case))
            s[name + "_back"] = torch.zeros(len(s["back"]), kv, d, device=DEV)
        return s
    # attend: what lies behind a sequence's end in its last page is never read as a value
    if case["fmt"] == "e4m3":
        last = [(int(table[i, t // page]), t % page) for i, t in enumerate(totals) if t % page]
        if last:
            behind = torch.arange(page, device=DEV)[None, :] >= _ints([o for _, o in last])[:, None]
            for name in ("k", "v"):
                p = s[name][_ints([a for a, _ in last]).long()]
                s[name][_ints([a for a, _ in last]).long()] = torch.where(behind[:, None, :, None], torch.full_like(p, 0x7F), p)
    rows = sum(q)
    s["q_start"] = _ints([0] + list(np.cumsum(q)))
    s["kv_lens"] = _ints(totals)
    s["max_q"], s["max_len"] = max(1, max(q)), max(1, max(totals))
    s["q"] = (1.5 * torch.randn(rows, case["heads"], case["d"], device=DEV, generator=g)).to(_dtype(case))
    s["out"] = torch.zeros_like(s["q"])
    return s


# ------------------------------------------------------------- plain forms

def _frequencies(case):
    """Radians per position of each rotated pair, 64 bits, and the factor on the rotated values."""
    rot = case["rot"]
    f = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "llama3":
        c = LLAMA3
        waves = c["original"] * f / (2 * math.pi)  # turns within the trained length
        keep = ((waves - c["low"]) / (c["high"] - c["low"])).clamp(0, 1)
        return keep * f + (1 - keep) * f / c["factor"], 1.0
    if case["scaling"] == "yarn":
        c = YARN
        at = lambda turns: rot * math.log(c["original"] / (turns * 2 * math.pi)) / (2 * math.log(500000.0))  # noqa: E731
        low, high = max(math.floor(at(c["fast"])), 0), min(math.ceil(at(c["slow"])), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64, device=DEV) - low) / max(high - low, 0.001)).clamp(0, 1)
        return ramp * f / c["factor"] + (1 - ramp) * f, 0.1 * math.log(c["factor"]) + 1.0
    return f, 1.0


def _plain_rope(s):
    case = s["case"]
    f, m = _frequencies(case)
    angle = s["pos"].double()[:, None] * f
    cos, sin = (angle.cos() * m).float()[:, None], (angle.sin() * m).float()[:, None]
    if case["transpose"]:
        sin = -sin
    x, rot = s["x"].float(), case["rot"]
    y = x.clone()
    if case["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return y.to(s["x"].dtype)


def _plain_pages(s):
    page, cap = s["case"]["page"], s["slots"].shape[0]
    lens, new, table, free = s["lens"].long(), s["n_new"].long(), s["table"], s["free_list"]
    ended = new < 0
    add = new.clamp(min=0)
    before = (lens + page - 1) // page
    after = torch.where(ended, before, (lens + add + page - 1) // page)
    back = torch.where(ended, before, torch.zeros_like(before))
    cols = torch.arange(table.shape[1], device=DEV)[None]
    returned = table[ended[:, None] & (cols < before[:, None])]
    stack = torch.cat([free[:int(s["free_count"])], returned])
    taken = (cols >= before[:, None]) & (cols < after[:, None])
    n_taken = int(taken.sum())
    table[taken] = stack[len(stack) - n_taken:].flip(0)
    left = len(stack) - n_taken
    free[:left] = stack[:left]
    q_start = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), add.cumsum(0)])
    tokens = int(q_start[-1])
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), add)
    pos = lens[seq] + torch.arange(tokens, device=DEV) - q_start[seq]
    slot = table[seq, pos // page].long() * page + pos % page
    pad = torch.full((cap - tokens,), -1, dtype=torch.int64, device=DEV)
    return {"table": table, "lens": torch.where(ended, torch.zeros_like(lens), lens + add).int(),
            "q_start": q_start.int(), "slots": torch.cat([slot, pad]).int(), "positions": torch.cat([pos, pad]).int(),
            "seq_ids": torch.cat([seq, pad]).int(), "free_list": free,
            "free_count": torch.full((1,), left, dtype=torch.int32, device=DEV),
            "status": torch.zeros(2, dtype=torch.int32, device=DEV)}


def _decode(codes, fmt):
    """Bytes -> the values their codes stand for, fp32."""
    return codes.view(torch.int8).float() if fmt == "i8" else codes.view(torch.float8_e4m3fn).float()


def _encode(x, fmt):
    """Quotients in 64 bits -> bytes, to the nearest code, ties to the even one."""
    if fmt == "i8":
        return x.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return ((x / step).round() * step).clamp(-448, 448).float().to(torch.float8_e4m3fn).view(torch.uint8)


def _over(x, scale):
    """x / scale in 64 bits, 0 where the scale is 0."""
    return torch.where(scale > 0, x.double() / scale.double(), torch.zeros((), dtype=torch.float64, device=DEV))


def _plain_append(s):
    case = s["case"]
    page, fmt = case["page"], case["fmt"]
    slots, back = s["slots"].long(), s["back"].long()
    at = slots // page
    first = torch.ones_like(at, dtype=torch.bool)
    first[1:] = at[1:] != at[:-1]
    mine, which = at[first], first.long().cumsum(0) - 1  # touched pages, and each row's place among them
    old_tokens = (slots % page)[first]                   # tokens that each page held
    got = []
    for name in ("k", "v"):
        rows, codes, scale = s[name + "_rows"].float(), s[name], s[name + "_scale"]
        old = torch.where((old_tokens > 0)[:, None], scale[mine], torch.zeros_like(scale[mine]))
        top = torch.zeros_like(old).scatter_reduce_(0, which[:, None].expand(-1, old.shape[1]), rows.abs().amax(-1), "amax")
        now = torch.maximum(old, top / torch.full_like(top, CODE_MAX[fmt]))
        grown = (now > old)[:, :, None, None] & (torch.arange(page, device=DEV) < old_tokens[:, None])[:, None, :, None]
        held = codes[mine]
        again = _encode(_over(_decode(held, fmt).double() * old[:, :, None, None].double(), now[:, :, None, None]), fmt)
        codes[mine] = torch.where(grown, again, held)
        codes[at, :, slots % page] = _encode(_over(rows, now[which][:, :, None]), fmt)
        scale[mine] = now
        got.append(_decode(codes[back // page, :, back % page], fmt) * scale[back // page][:, :, None])
    return {"k": got[0], "v": got[1]}


def _plain_attend(s):
    case = s["case"]
    page, fmt, kv, d = case["page"], case["fmt"], case["kv"], case["d"]
    group, top, max_q = case["heads"] // kv, s["max_len"], s["max_q"]
    lens, start = s["kv_lens"].long(), s["q_start"].long()
    n, count = len(lens), start[1:] - start[:-1]
    t = torch.arange(top, device=DEV)
    there = t[None] < lens[:, None]
    at = torch.where(there, s["table"].long()[:, t // page], 0)
    k = _decode(s["k"][at, :, t % page], fmt) * s["k_scale"][at][..., None]
    v = _decode(s["v"][at, :, t % page], fmt) * s["v_scale"][at][..., None]
    v = torch.where(there[:, :, None, None], v, 0.0)
    j = torch.arange(max_q, device=DEV)
    mine = j[None] < count[:, None]
    row = torch.where(mine, start[:-1, None] + j, 0)
    q = s["q"].float()[row].view(n, max_q, kv, group, d).permute(0, 2, 3, 1, 4).reshape(n, kv, group * max_q, d)
    score = torch.matmul(q, k.permute(0, 2, 3, 1)).view(n, kv, group, max_q, top) / math.sqrt(d)
    seen = t[None, None] <= (lens - count)[:, None, None] + j[None, :, None]
    score = torch.where(seen[:, None, None], score, -math.inf)
    high = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(high > -math.inf, high, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(n, kv, group * max_q, top), v.permute(0, 2, 1, 3)).view(n, kv, group, max_q, d)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(n, max_q, kv * group, d)[mine].to(s["q"].dtype)


# ----------------------------------------------------------- the library's

_kept = {}


def _library():
    """The library's kernels on one accelerator, as a program keeps them."""
    if not _kept:
        import os
        import sys
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama3-java-hat_b200"))
        import llamahat
        f, acc = llamahat.CudaKernelFactory(), llamahat.Accelerator(0)
        _kept.update(lib=llamahat, acc=acc, rope=f.createRoPE(acc), pages=f.createPages(acc))
    return _kept


def _rope_config(lib, case):
    a = {"head_dim": case["d"], "rot_dim": case["rot"], "layout": case["layout"], "scaling": case["scaling"],
         "theta": 500000.0}
    if case["scaling"] == "linear":
        a |= {"factor": 4.0}
    if case["scaling"] == "llama3":
        a |= {"factor": LLAMA3["factor"], "low_freq_factor": LLAMA3["low"], "high_freq_factor": LLAMA3["high"],
              "original_max_pos": LLAMA3["original"]}
    if case["scaling"] == "yarn":
        a |= {"factor": YARN["factor"], "beta_fast": YARN["fast"], "beta_slow": YARN["slow"],
              "original_max_pos": YARN["original"]}
    return lib.RopeConfig(**a)


def _own(s):
    own_, case = _library(), s["case"]
    lib, op = own_["lib"], case["op"]
    if op == "rope":
        if "config" not in s:
            s["config"] = _rope_config(lib, case)
        own_["rope"].apply_scaled(s["x"], s["y"], s["pos"], s["config"], transpose=case["transpose"])
        return s["y"]
    if op == "pages":
        own_["pages"].step(s["lens"], s["n_new"], s["table"], s["free_list"], s["free_count"], case["page"],
                           s["lens_out"], s["q_start"], s["slots"], s["positions"], s["seq_ids"],
                           s["free_count_out"], s["status"])
        return {"table": s["table"], "lens": s["lens_out"], "q_start": s["q_start"], "slots": s["slots"],
                "positions": s["positions"], "seq_ids": s["seq_ids"], "free_list": s["free_list"],
                "free_count": s["free_count_out"], "status": s["status"]}
    if "cache" not in s:
        s["cache"] = lib.PagedKV8(s["k"], s["v"], s["k_scale"], s["v_scale"], format=case["fmt"], acc=own_["acc"])
    if op == "append":
        s["cache"].append(s["k_rows"], s["v_rows"], s["slots"])
        s["cache"].read(s["k_back"], s["v_back"], s["back"])
        return {"k": s["k_back"], "v": s["v_back"]}
    s["cache"].attention(s["q"], s["out"], s["q_start"], s["kv_lens"], s["table"], max_q=s["max_q"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "pages": _plain_pages, "append": _plain_append,
            "attend": _plain_attend}[state["case"]["op"]](state)


# -------------------------------------------------------------- definitions

def _exact_rope(case, s):
    """Each pair as a complex number times m * e^(i p f); the transposed map is the conjugate."""
    rot = case["rot"]
    f = np.array([500000.0 ** (-2.0 * j / rot) for j in range(rot // 2)])
    m = 1.0
    if case["scaling"] == "linear":
        f = f / 4.0
    elif case["scaling"] == "llama3":
        wave = 2 * np.pi / f
        smooth = (LLAMA3["original"] / wave - LLAMA3["low"]) / (LLAMA3["high"] - LLAMA3["low"])
        f = np.where(wave < LLAMA3["original"] / LLAMA3["high"], f,
                     np.where(wave > LLAMA3["original"] / LLAMA3["low"], f / LLAMA3["factor"],
                              (1 - smooth) * f / LLAMA3["factor"] + smooth * f))
    elif case["scaling"] == "yarn":
        dim = [rot * np.log(YARN["original"] / (b * 2 * np.pi)) / (2 * np.log(500000.0)) for b in (YARN["fast"], YARN["slow"])]
        low, high = max(np.floor(dim[0]), 0), min(np.ceil(dim[1]), rot - 1)
        own_part = 1 - np.clip((np.arange(rot // 2) - low) / max(high - low, 0.001), 0, 1)
        f = f / YARN["factor"] * (1 - own_part) + f * own_part
        m = 0.1 * np.log(YARN["factor"]) + 1
    turn = torch.polar(torch.full((case["rows"], rot // 2), m, dtype=torch.float64, device=DEV),
                       torch.outer(s["pos"].double(), torch.from_numpy(f).to(DEV)))
    turn = (turn.conj() if case["transpose"] else turn)[:, None]
    x = s["x"].double()
    part = x[..., :rot]
    pair = part.unflatten(-1, (2, -1)).transpose(-1, -2) if case["layout"] == "half" else part.unflatten(-1, (-1, 2))
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    z = (z.transpose(-1, -2) if case["layout"] == "half" else z).flatten(-2)
    return torch.cat([z, x[..., rot:]], -1)


def _exact_pages(case, s):
    page = case["page"]
    lens, new, count = s["lens"].tolist(), s["n_new"].tolist(), int(s["free_count"])
    table, free = s["table"].cpu().numpy().copy(), s["free_list"].cpu().numpy().copy()
    stack = free[:count].tolist()
    for i, (h, a) in enumerate(zip(lens, new)):
        if a < 0:
            stack += table[i, :-(-h // page)].tolist()
    slots, positions, ids, start, out = [], [], [], [0], []
    for i, (h, a) in enumerate(zip(lens, new)):
        for p in range(-(-h // page), -(-(h + a) // page)) if a > 0 else ():
            table[i, p] = stack.pop()
        for t in range(h, h + max(0, a)):
            slots.append(int(table[i, t // page]) * page + t % page)
            positions.append(t)
            ids.append(i)
        start.append(len(slots))
        out.append(0 if a < 0 else h + a)
    free[:len(stack)] = stack
    pad = [-1] * (s["slots"].shape[0] - len(slots))
    return {"table": torch.from_numpy(table), "lens": torch.tensor(out, dtype=torch.int32),
            "q_start": torch.tensor(start, dtype=torch.int32), "slots": torch.tensor(slots + pad, dtype=torch.int32),
            "positions": torch.tensor(positions + pad, dtype=torch.int32),
            "seq_ids": torch.tensor(ids + pad, dtype=torch.int32), "free_list": torch.from_numpy(free),
            "free_count": torch.tensor([len(stack)], dtype=torch.int32), "status": torch.zeros(2, dtype=torch.int32)}


def _nearest(x, fmt):
    """The nearest code value to each quotient, from the sorted list of all of them; ties to the even code."""
    if fmt == "i8":
        values = np.arange(-127, 128, dtype=np.float64)
        even = np.arange(-127, 128) % 2 == 0
    else:
        pos = torch.arange(0, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
        values = np.concatenate([-pos[:0:-1], pos])
        even = np.concatenate([np.arange(0x7E, 0, -1) % 2 == 0, np.arange(0x7F) % 2 == 0])
    hi = np.clip(np.searchsorted(values, x), 1, len(values) - 1)
    lo = hi - 1
    up, down = values[hi] - x, x - values[lo]
    return np.where((up < down) | ((up == down) & even[hi]), values[hi], values[lo])


def _exact_append(case, s):
    """Page by page, on the host: the running largest scale, every held value to its nearest code."""
    page, fmt = case["page"], case["fmt"]
    slots, back = s["slots"].cpu().numpy().astype(np.int64), s["back"].cpu().numpy().astype(np.int64)
    got = {}
    for name in ("k", "v"):
        rows = s[name + "_rows"].double().cpu().numpy()
        held = {}
        order = np.argsort(slots // page, kind="stable")
        touched, begin = np.unique((slots // page)[order], return_index=True)
        old_codes = _decode(s[name][torch.from_numpy(touched).to(DEV)], fmt).double().cpu().numpy()
        old_scale = s[name + "_scale"].cpu().numpy()
        for i, p in enumerate(touched):
            r = order[begin[i]:begin[i + 1] if i + 1 < len(touched) else None]
            off = slots[r] % page
            before = old_scale[p] if off.min() > 0 else np.zeros_like(old_scale[p])
            top = np.abs(rows[r]).max((0, 2)).astype(np.float32)
            now = np.maximum(before, top / np.float32(CODE_MAX[fmt])).astype(np.float64)[:, None, None]
            safe = np.where(now > 0, now, 1.0)
            values = old_codes[i].copy()
            again = _nearest(values * before.astype(np.float64)[:, None, None] / safe, fmt)
            grown = now > before.astype(np.float64)[:, None, None]
            values = np.where(grown, again, values)
            values[:, off] = _nearest(rows[r].transpose(1, 0, 2) / safe, fmt)
            held[int(p)] = values * now
        got[name] = torch.from_numpy(np.stack([held[int(b // page)][:, b % page] for b in back])) if len(back) else torch.zeros(0, case["kv"], case["d"], dtype=torch.float64)
    return got


def _exact_attend(case, s):
    """Sequence by sequence and head by head in 64 bits."""
    page, fmt, group, d = case["page"], case["fmt"], case["heads"] // case["kv"], case["d"]
    start, lens, table = s["q_start"].tolist(), s["kv_lens"].tolist(), s["table"].long()
    q = s["q"].double()
    out = torch.zeros_like(q)
    for i, length in enumerate(lens):
        b, e = start[i], start[i + 1]
        if length == 0 or e == b:
            continue
        mine = table[i, :-(-length // page)]
        at = torch.arange(length, device=DEV)
        for h in range(case["kv"]):
            k = (_decode(s["k"][mine, h], fmt).double() * s["k_scale"][mine, h].double()[:, None, None]).reshape(-1, d)[:length]
            v = (_decode(s["v"][mine, h], fmt).double() * s["v_scale"][mine, h].double()[:, None, None]).reshape(-1, d)[:length]
            limit = torch.arange(length - (e - b), length, device=DEV)
            hidden = at[None] > limit[:, None]
            for x in range(h * group, (h + 1) * group):
                score = (q[b:e, x] @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
                w = torch.softmax(score, -1).masked_fill(hidden, 0.0)
                out[b:e, x] = torch.where((limit >= 0)[:, None], w @ v, 0.0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "pages": _exact_pages, "append": _exact_append,
            "attend": _exact_attend}[case["op"]](case, s)
