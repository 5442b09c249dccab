"""Plain 64-bit references of the paged 8-bit cache operators (numpy)."""
import math

import numpy as np

LIMIT = {"i8": 127.0, "e4m3": 448.0}


# --------------------------------------------------------------- rotary

def rope_frequencies(cfg):
    """Radians per position of each pair and the factor on cos and sin."""
    rot = cfg.head_dim if cfg.rot_dim is None else cfg.rot_dim
    out, mult = [], 1.0
    low = high = 0.0
    if cfg.scaling == "yarn":
        dim = lambda turns: rot * math.log(cfg.original_max_pos / (turns * 2 * math.pi)) / (2 * math.log(cfg.theta))  # noqa: E731
        low, high = max(math.floor(dim(cfg.beta_fast)), 0), min(math.ceil(dim(cfg.beta_slow)), rot - 1)
        mult = cfg.attn_factor or 0.1 * math.log(cfg.factor) + 1.0
    for j in range(rot // 2):
        f = cfg.theta ** (-2.0 * j / rot)
        if cfg.scaling == "linear":
            f /= cfg.factor
        elif cfg.scaling == "llama3":
            wave = 2 * math.pi / f
            if wave > cfg.original_max_pos / cfg.low_freq_factor:
                f /= cfg.factor
            elif wave > cfg.original_max_pos / cfg.high_freq_factor:
                k = (cfg.original_max_pos / wave - cfg.low_freq_factor) / (cfg.high_freq_factor - cfg.low_freq_factor)
                f = (1 - k) * f / cfg.factor + k * f
        elif cfg.scaling == "yarn":
            r = min(max((j - low) / max(high - low, 0.001), 0.0), 1.0)
            f = r * f / cfg.factor + (1 - r) * f
        out.append(f)
    return np.array(out), mult


def rope(x, pos, cfg, transpose=False):
    """x [rows, heads, head_dim] -> float64 rotation; rows at pos < 0 come back unchanged."""
    x = x.astype(np.float64)
    f, m = rope_frequencies(cfg)
    half = len(f)
    y = x.copy()
    for i, p in enumerate(pos):
        if p < 0:
            continue
        c, s = m * np.cos(p * f), m * np.sin(p * f) * (-1 if transpose else 1)
        for j in range(half):
            a, b = (j, j + half) if cfg.layout == "half" else (2 * j, 2 * j + 1)
            u, v = x[i, :, a], x[i, :, b]
            y[i, :, a], y[i, :, b] = u * c[j] - v * s[j], u * s[j] + v * c[j]
    return y


# ---------------------------------------------------------------- pages

def pages_step(lens, n_new, page, table, free, capacity):
    """lens, n_new, free: lists; table: array, updated.  None where the step
    cannot be done, else (lens, q_start, slots, positions, seq_ids, free)."""
    ceil = lambda t: -(-t // page)  # noqa: E731
    stack = list(free)
    for s, (h, a) in enumerate(zip(lens, n_new)):
        if a < 0:
            stack += [int(p) for p in table[s, :ceil(h)]]
    need = sum(ceil(h + a) - ceil(h) for h, a in zip(lens, n_new) if a > 0)
    if need > len(stack) or any(ceil(h + max(a, 0)) > table.shape[1] for h, a in zip(lens, n_new)):
        return None
    if sum(max(a, 0) for a in n_new) > capacity:
        return None
    slots, positions, ids, start, out = [], [], [], [0], []
    for s, (h, a) in enumerate(zip(lens, n_new)):
        for p in range(ceil(h), ceil(h + max(a, 0))):
            table[s, p] = stack.pop()
        for t in range(h, h + max(a, 0)):
            slots.append(int(table[s, t // page]) * page + t % page)
            positions.append(t)
            ids.append(s)
        start.append(len(slots))
        out.append(h + a if a >= 0 else 0)
    pad = [-1] * (capacity - len(slots))
    return out, start, slots + pad, positions + pad, ids + pad, stack


# ---------------------------------------------------------------- codes

def e4m3_values():
    """Value of every e4m3 byte (NaN at 0x7f and 0xff)."""
    out = np.zeros(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[b] = math.nan if (b & 0x7F) == 0x7F else (-v if b & 0x80 else v)
    return out


E4M3 = e4m3_values()


def decode(codes, fmt):
    return codes.view(np.int8).astype(np.float64) if fmt == "i8" else E4M3[codes]


def encode(q, fmt):
    """Nearest code of each quotient (float64), ties to the even code, ends saturate."""
    q = np.clip(q, -LIMIT[fmt], LIMIT[fmt])
    if fmt == "i8":
        return np.rint(q).astype(np.int8).view(np.uint8)
    pos = E4M3[:0x7F]
    x = np.abs(q)
    hi = np.clip(np.searchsorted(pos, x), 1, 0x7E)
    lo = hi - 1
    up, down = pos[hi] - x, x - pos[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo).astype(np.uint8)
    return code | (np.signbit(q).astype(np.uint8) << 7)


def append(codes, scales, rows, slots, fmt):
    """codes [n_pages, n_kv, page, d] and scales [n_pages, n_kv] updated in
    place with rows [n, n_kv, d] at slots."""
    page, total = codes.shape[2], codes.shape[0] * codes.shape[2]
    i = 0
    while i < len(slots):
        first = int(slots[i])
        if first < 0 or first >= total:
            i += 1
            continue
        n = 1
        while i + n < len(slots) and slots[i + n] == first + n and (first + n) % page:
            n += 1
        p, off = first // page, first % page
        x = rows[i:i + n].astype(np.float64)
        fine = np.where(np.isfinite(x), np.abs(x), 0.0).max((0, 2)).astype(np.float32)
        old = scales[p].copy() if off else np.zeros_like(scales[p])
        now = np.maximum(old, fine / np.float32(LIMIT[fmt]))
        for h in range(codes.shape[1]):
            s = float(now[h])
            if now[h] > old[h] and off:
                codes[p, h, :off] = encode(decode(codes[p, h, :off], fmt) * float(old[h]) / s, fmt)
            q = x[:, h] / s if s > 0 else np.zeros_like(x[:, h])
            codes[p, h, off:off + n] = encode(np.where(np.isnan(q), 0.0, q), fmt)
        scales[p] = now
        i += n


# ------------------------------------------------------------ attention

def attention(q, q_start, lens, table, k, v, k_scale, v_scale, fmt, scale, out, terms=None):
    """out [rows, n_heads, d] (float64) filled for the rows of the sequences.
    terms: a dict that receives per (row, head) the largest sum |q k| scale
    and sum p |v| that error bounds need."""
    page, n_kv = k.shape[2], k.shape[1]
    group = q.shape[1] // n_kv
    for s, length in enumerate(lens):
        b, e = (q_start[s], q_start[s + 1]) if q_start is not None else (s, s + 1)
        for j in range(b, e):
            seen = length - (e - b) + (j - b) + 1
            for h in range(q.shape[1]):
                out[j, h] = 0.0
                if seen <= 0:
                    continue
                t = np.arange(seen)
                pg = table[s, t // page]
                keep = (pg >= 0) & (pg < k.shape[0])
                t, pg = t[keep], pg[keep]
                if not len(t):
                    continue
                g = h // group
                kk = decode(k[pg, g, t % page], fmt) * k_scale[pg, g].astype(np.float64)[:, None]
                vv = decode(v[pg, g, t % page], fmt) * v_scale[pg, g].astype(np.float64)[:, None]
                x = kk @ q[j, h].astype(np.float64) * scale
                w = np.exp(x - x.max())
                w /= w.sum()
                out[j, h] = w @ vv
                if terms is not None:
                    terms[j, h] = ((np.abs(kk) @ np.abs(q[j, h].astype(np.float64))).max() * scale, w @ np.abs(vv), len(t))
    return out
