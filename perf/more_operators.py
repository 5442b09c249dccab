"""Cases and plain forms of the 4-bit weights and of the log probabilities.

Three operators of the last step of an answer, and of the products before it:

  quantize  rows of weights to 4-bit codes under one scale (and one zero point)
            per group of columns, and back to values
  product   y = x W^T (+ a residual) with such weights: one row of x (decode),
            a batch, a prompt
  logprobs  from rows of logits: the log probability and rank of one given
            token, the entropy, and the best alternatives with theirs

A value is scale * (code - zero): codes 0..15, fp16 scales [rows][groups],
zero points 0..15 [rows][groups] or 8 throughout; the last group of a row may
be short.

`run` computes an operator with elementary torch operations, or (`own`) with
the library's entry points.
"""
import math
import random

import torch

own = False

DEV = "cuda"
LOWEST = {"f32": -3.4028234663852886e38, "f16": -65504.0}
TYPES = {"f32": torch.float32, "f16": torch.float16}


# ------------------------------------------------------------------- cases

def listed():
    return [
        # The down projection of a layer, quantised at load: fp16 rows, no zero points.
        {"name": "quantize-down", "op": "quantize", "rows": 2048, "cols": 8192, "group": 128, "zeros": False,
         "type": "f16"},
        # A vocabulary of odd size with a ragged last group: fp32 rows, zero points.
        {"name": "quantize-vocabulary", "op": "quantize", "rows": 32003, "cols": 2085, "group": 32, "zeros": True,
         "type": "f32"},
        # The output projection of attention for one token: the smallest call of a decode step.
        {"name": "product-o", "op": "product", "rows": 2048, "cols": 2048, "batch": 1, "group": 128, "zeros": False,
         "type": "f32", "residual": True, "pad": 0},
        # The lm_head for one token: the largest matrix that a decode step reads.
        {"name": "product-lm-head", "op": "product", "rows": 128256, "cols": 2048, "batch": 1, "group": 64,
         "zeros": False, "type": "f32", "residual": False, "pad": 0},
        # The down projection of 8 sequences, fine groups with zero points, added to the residual stream.
        {"name": "product-down-8", "op": "product", "rows": 2048, "cols": 8192, "batch": 8, "group": 32, "zeros": True,
         "type": "f32", "residual": True, "pad": 0},
        # Odd sizes and strides: a shard of a matrix, 5 sequences in half precision.
        {"name": "product-odd", "op": "product", "rows": 1777, "cols": 2085, "batch": 5, "group": 64, "zeros": True,
         "type": "f16", "residual": False, "pad": 3},
        # Gate and up of 64 sequences in one step.
        {"name": "product-gate-64", "op": "product", "rows": 16384, "cols": 2048, "batch": 64, "group": 128,
         "zeros": False, "type": "f32", "residual": False, "pad": 0},
        # Gate and up of a prompt.
        {"name": "product-prompt", "op": "product", "rows": 16384, "cols": 2048, "batch": 2048, "group": 128,
         "zeros": True, "type": "f16", "residual": False, "pad": 0},
        # The token that one sequence has just chosen, with 20 alternatives.
        {"name": "logprobs-one", "op": "logprobs", "rows": 1, "vocab": 128256, "top": 20, "type": "f32", "pad": 0,
         "masked": 0.0, "scale": 1.0},
        # 64 sequences under a grammar: most logits masked, by -inf or by the lowest value; a row may be empty.
        {"name": "logprobs-masked", "op": "logprobs", "rows": 64, "vocab": 128256, "top": 5, "type": "f32", "pad": 0,
         "masked": 0.9, "scale": 1.25},
        # Scoring prompts: log probability, rank and entropy of each position.
        {"name": "logprobs-score", "op": "logprobs", "rows": 2048, "vocab": 128256, "top": 0, "type": "f16", "pad": 0,
         "masked": 0.0, "scale": 1.0},
        # An odd vocabulary, rows at a larger odd stride, the most alternatives.
        {"name": "logprobs-odd", "op": "logprobs", "rows": 333, "vocab": 32003, "top": 32, "type": "f16", "pad": 8,
         "masked": 0.0, "scale": 0.7},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["quantize", "product", "product", "product", "logprobs", "logprobs"])
    kind = rng.choice(["f32", "f16"])
    if op == "logprobs":
        vocab = _log_int(rng, 1000, 128256)
        return {"op": op, "vocab": vocab, "rows": _log_int(rng, 1, min(2048, 2048 * 128256 // vocab)),
                "top": rng.choice([0, 1, 5, 20, 32]), "type": kind, "pad": rng.choice([0, 0, 1, 8]),
                "masked": rng.choice([0.0, 0.0, 0.5, 0.9]), "scale": rng.choice([1.0, 0.7, 1.25])}
    case = {"op": op, "cols": _log_int(rng, 128, 8192), "group": rng.choice([32, 64, 128]),
            "zeros": rng.random() < 0.5, "type": kind}
    if rng.random() < 0.6:  # most widths are multiples of 128
        case["cols"] = max(128, case["cols"] // 128 * 128)
    if op == "quantize":
        return case | {"rows": _log_int(rng, 64, min(131072, 32003 * 2085 // case["cols"]))}
    rows = _log_int(rng, 64, min(131072, 128256 * 2048 // case["cols"]))
    most = min(2048, (1 << 25) // rows, 16384 * 2048 * 2048 // (rows * case["cols"]))
    return case | {"rows": rows, "batch": _log_int(rng, 1, max(1, most)), "residual": rng.random() < 0.3,
                   "pad": rng.choice([0, 0, 3, 8])}


# ------------------------------------------------------------------ inputs

def _rows(x, pad):
    """x at a row stride of its width plus `pad` elements."""
    held = torch.zeros(x.shape[0], x.shape[1] + pad, dtype=x.dtype, device=DEV)
    held[:, :x.shape[1]] = x
    return held[:, :x.shape[1]]


def _weights(gen, rows, cols):
    """Trained weights look like this: normal, columns of unlike size, a few far outliers."""
    w = torch.randn(rows, cols, generator=gen, device=DEV) * 0.02
    w *= torch.exp(0.3 * torch.randn(cols, generator=gen, device=DEV))
    far = torch.randint(0, rows * cols, (rows * cols // 5000 + 1,), generator=gen, device=DEV)
    w.view(-1)[far] *= 12.0
    return w


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind, s = TYPES[case["type"]], {"case": case}
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn(rows, vocab, generator=gen, device=DEV)
        x *= 2.0 + torch.rand(rows, 1, generator=gen, device=DEV)
        each = torch.arange(rows, device=DEV)
        peak = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)  # sure rows and unsure ones
        x[each, peak] += 16.0 * torch.rand(rows, generator=gen, device=DEV)
        given = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
        given = torch.where(torch.rand(rows, generator=gen, device=DEV) < 0.7, peak, given)
        if case["masked"]:
            gone = torch.rand(rows, vocab, generator=gen, device=DEV) < case["masked"]
            gone[each, given] = False  # what was chosen was allowed
            x = torch.where(gone, torch.where(torch.rand(rows, 1, generator=gen, device=DEV) < 0.5, -math.inf,
                                              LOWEST[case["type"]]), x)
            if rows >= 8:
                x[rows // 2] = -math.inf  # a row that allows nothing
        if rows >= 8:
            given[rows // 3] = -1  # a padded position
        s |= {"logits": _rows(x.to(kind), case["pad"]), "tokens": given.int(),
              "logprob": torch.empty(rows, device=DEV), "rank": torch.empty(rows, dtype=torch.int32, device=DEV),
              "entropy": torch.empty(rows, device=DEV)}
        if case["top"]:
            s |= {"top_ids": torch.empty(rows, case["top"], dtype=torch.int32, device=DEV),
                  "top_logprobs": torch.empty(rows, case["top"], device=DEV)}
        if own:
            s["lib"] = _library()["logprobs"]
        return s
    rows, cols = case["rows"], case["cols"]
    w = _weights(gen, rows, cols).to(kind)
    if case["op"] == "quantize":
        s |= {"w": w, "back": torch.empty_like(w)}
        if own:
            s["weights"] = _library()["Weights4"].empty(rows, cols, case["group"], case["zeros"],
                                                       acc=_library()["acc"])
        return s
    batch = case["batch"]
    x = torch.randn(batch, cols, generator=gen, device=DEV)
    x[:, torch.randint(0, cols, (3,), generator=gen, device=DEV)] *= 20.0  # loud channels
    s |= {"x": _rows(x.to(kind), case["pad"]), "residual": None,
          "y": _rows(torch.empty(batch, rows, dtype=kind, device=DEV), case["pad"])}
    if case["residual"]:
        s["residual"] = _rows(torch.randn(batch, rows, generator=gen, device=DEV).to(kind), case["pad"])
    # What a checkpoint holds: two codes to a byte, the lower column in the low half.
    code, scale, zero = _quantize(w, case["group"], case["zeros"])
    code = torch.cat([code, torch.zeros(rows, cols % 2, dtype=torch.uint8, device=DEV)], 1)
    s |= {"codes": code[:, ::2] | code[:, 1::2] << 4, "scales": scale, "zeros": zero}
    if own:
        # Weights are laid out once, when a model is loaded; the library's stream does not wait for torch's.
        torch.cuda.synchronize()
        s["weights"] = _library()["Weights4"].empty(rows, cols, case["group"], case["zeros"], acc=_library()["acc"])
        s["weights"].pack(s["codes"], scale, zero)
        _library()["acc"].synchronize()
    return s


# ------------------------------------------------------------- plain forms

def _grouped(w, group, fill):
    """[rows][cols] -> [rows][groups][group], the last group filled up."""
    rows, cols = w.shape
    room = -cols % group
    w = torch.cat([w, torch.full((rows, room), fill, dtype=w.dtype, device=DEV)], 1) if room else w
    return w.view(rows, -1, group)


def _quantize(w, group, zeros):
    """Codes [rows][cols], scales, zero points (None: 8), quotients in 64 bits."""
    cols = w.shape[1]
    g = _grouped(w.float(), group, 0.0)
    if zeros:
        low, high = g.amin(-1).clamp(max=0).double(), g.amax(-1).clamp(min=0).double()
        scale = ((high - low) / 15).clamp(max=65504.0).half()
        step = scale.double()
        zero = torch.where(step > 0, -low / step, 0.0).round().clamp(0, 15)
        q = torch.where(step[..., None] > 0, g.double() / step[..., None], 0.0).round()
        code = (q + zero[..., None]).clamp(0, 15)
    else:
        scale = (g.abs().amax(-1).double() / 7).clamp(max=65504.0).half()
        step = scale.double()
        zero = None
        code = torch.where(step[..., None] > 0, g.double() / step[..., None], 0.0).round().clamp(-7, 7) + 8
    return (code.to(torch.uint8).view(w.shape[0], -1)[:, :cols].contiguous(), scale,
            None if zero is None else zero.to(torch.uint8))


def _values(code, scale, zero, group):
    """The values that codes [rows][cols] stand for, fp32."""
    cols = code.shape[1]
    z = 8.0 if zero is None else zero.float()[..., None]
    return ((_grouped(code, group, 0).float() - z) * scale.float()[..., None]).reshape(code.shape[0], -1)[:, :cols]


def _plain_quantize(s):
    group = s["case"]["group"]
    code, scale, zero = _quantize(s["w"], group, s["case"]["zeros"])
    return {"values": _values(code, scale, zero, group).to(s["w"].dtype)}


def _plain_product(s):
    case = s["case"]
    code = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(case["rows"], -1)[:, :case["cols"]]
    y = s["x"].float() @ _values(code, s["scales"], s["zeros"], case["group"]).t()
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(s["x"].dtype)}


def _plain_logprobs(s):
    case = s["case"]
    rows, vocab = s["logits"].shape
    x = s["logits"].float() + 0.0  # no negative zeros: equal logits go by their index
    high = x.amax(1, keepdim=True)
    empty = high == -math.inf
    t = torch.where(x > -math.inf, (x - torch.where(empty, 0.0, high)) * case["scale"], -math.inf)
    e = torch.exp(t)
    total = e.sum(1, keepdim=True)
    log_total = torch.where(empty, 0.0, torch.log(total))
    entropy = log_total - torch.where(e > 0, e * t, 0.0).sum(1, keepdim=True) / torch.where(empty, 1.0, total)
    given = s["tokens"].long()
    there = (given >= 0) & (given < vocab)
    at = torch.where(there, given, 0)[:, None]
    mine = x.gather(1, at)
    before = (x > mine) | ((x == mine) & (torch.arange(vocab, device=DEV)[None] < at))
    out = {"logprob": torch.where(there, (t.gather(1, at) - log_total)[:, 0], 0.0),
           "rank": torch.where(there, before.sum(1), -1).int(), "entropy": entropy[:, 0]}
    if case["top"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :case["top"]]
        out |= {"top_ids": ids.int(), "top_logprobs": t.gather(1, ids) - log_total}
    return out


# ------------------------------------------------------------- the library

_made = {}


def _library():
    if not _made:
        import os
        import sys
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama3-java-hat_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import llamahat
        acc = llamahat.Accelerator(torch.cuda.current_device())
        _made.update(acc=acc, Weights4=llamahat.Weights4, logprobs=llamahat.CudaKernelFactory().createLogProbs(acc))
    return _made


def _own(s):
    op = s["case"]["op"]
    if op == "quantize":
        s["weights"].quantize(s["w"])
        s["weights"].read(s["back"])
        return {"values": s["back"]}
    if op == "product":
        s["weights"].apply(s["x"], s["y"], residual=s["residual"])
        return {"y": s["y"]}
    s["lib"].apply(s["logits"], s["tokens"], s["logprob"], s["rank"], s["entropy"], s.get("top_ids"),
                   s.get("top_logprobs"), scale=s["case"]["scale"])
    return {k: s[k] for k in ("logprob", "rank", "entropy", "top_ids", "top_logprobs") if k in s}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "quantize":
        return _plain_quantize(state)
    return _plain_product(state) if op == "product" else _plain_logprobs(state)


# -------------------------------------------------------- work, and 64 bits

def work(case):
    size = 4 if case["type"] == "f32" else 2
    rows = case["rows"]
    if case["op"] == "logprobs":
        n = rows * case["vocab"]
        return {"bytes": n * size + rows * (16 + 8 * case["top"]), "flops": 6 * n}
    cols, groups = case["cols"], -(-case["cols"] // case["group"])
    held = rows * cols / 2 + rows * groups * (2.5 if case["zeros"] else 2)
    if case["op"] == "quantize":  # values in, codes and values out
        return {"bytes": int(2 * rows * cols * size + held), "flops": 6 * rows * cols}
    batch = case["batch"]
    return {"bytes": int(held + batch * cols * size + batch * rows * size * (2 if case["residual"] else 1)),
            "flops": 2 * rows * cols * batch}


def _exact_quantize(case, s):
    """Group by group of columns; the nearest whole quotient from its remainder."""
    x, g = s["w"].double(), case["group"]
    parts = []
    for c in range(0, case["cols"], g):
        part = x[:, c:c + g]
        if case["zeros"]:
            low, high = part.min(1, keepdim=True)[0].clamp(max=0), part.max(1, keepdim=True)[0].clamp(min=0)
            scale = ((high - low) / 15).clamp(max=65504.0).half().double()
        else:
            scale = (part.abs().max(1, keepdim=True)[0] / 7).clamp(max=65504.0).half().double()
        one = torch.where(scale > 0, scale, 1.0)

        def nearest(v):
            down = torch.floor(v / one)
            rest = v / one - down
            return down + ((rest > 0.5) | ((rest == 0.5) & (down % 2 != 0)))

        if case["zeros"]:
            zero = nearest(-low).clamp(0, 15)
            steps = (nearest(part) + zero).clamp(0, 15) - zero
        else:
            steps = nearest(part).clamp(-7, 7)
        parts.append(steps * scale)
    return {"values": torch.cat(parts, 1)}


def _exact_product(case, s):
    y = torch.zeros(case["batch"], case["rows"], dtype=torch.float64, device=DEV)
    g = case["group"]
    for i in range(-(-case["cols"] // g)):
        held = s["codes"][:, i * g // 2:(i + 1) * g // 2].double()
        high = torch.floor(held / 16)
        codes = torch.stack([held - 16 * high, high], 2).flatten(1)
        codes -= 8.0 if s["zeros"] is None else s["zeros"][:, i:i + 1].double()
        x = s["x"][:, i * g:(i + 1) * g].double()
        y += (x @ codes[:, :x.shape[1]].T) * s["scales"][:, i].double()
    return {"y": y if s["residual"] is None else y + s["residual"].double()}


def _exact_logprobs(case, s):
    out = {"logprob": [], "rank": None, "entropy": []}
    if case["top"]:
        out |= {"top_ids": None, "top_logprobs": []}
    for at in range(0, case["rows"], 128):
        x, given = s["logits"][at:at + 128].double() * case["scale"], s["tokens"][at:at + 128].long()
        lp = torch.log_softmax(x, 1)
        lp = torch.where((x == -math.inf).all(1, keepdim=True), -math.inf, lp)
        p = torch.exp(lp)
        out["entropy"].append(-torch.where(p > 0, p * lp, 0.0).sum(1))
        mine = lp[torch.arange(len(x), device=DEV), given.clamp(min=0)]
        out["logprob"].append(torch.where(given >= 0, mine, 0.0))
        if case["top"]:
            out["top_logprobs"].append(torch.topk(lp, case["top"], dim=1)[0])
    out = {k: torch.cat(v) if v else None for k, v in out.items()}
    beyond = torch.finfo(torch.float32).min  # what fp32 cannot hold
    return {k: v if v is None else torch.where(v < beyond, -math.inf, v) for k, v in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"quantize": _exact_quantize, "product": _exact_product, "logprobs": _exact_logprobs}[case["op"]](case, s)
