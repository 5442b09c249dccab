"""Plain 64-bit references of the 4-bit weights and of the log probabilities,
on the CPU, and what their tests share."""
import numpy as np

# A rounding to the type is off by at most half a step.
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25}
NP = {"f32": np.float32, "f16": np.float16}


def _groups(x, group, fill):
    room = -x.shape[1] % group
    x = np.concatenate([x, np.full((x.shape[0], room), fill, x.dtype)], 1)
    return x.reshape(x.shape[0], -1, group)


def _f16(q):
    with np.errstate(over="ignore"):
        return np.minimum(q, 65504.0).astype(np.float32).astype(np.float16)


def quantize(x, group, zeros):
    """Codes [rows, cols] (uint8), scales [rows, groups] (float16), zero points or None."""
    g = _groups(x.astype(np.float64), group, 0.0)
    g = np.where(np.isnan(g), 0.0, g)
    fine = np.where(np.isfinite(g), g, 0.0)
    low, high = np.minimum(fine.min(-1), 0.0), np.maximum(fine.max(-1), 0.0)
    scale = _f16((high - low) / 15.0 if zeros else np.maximum(-low, high) / 7.0)
    s = scale.astype(np.float64)
    one = np.where(s > 0, s, 1.0)[..., None]
    q = np.where(s[..., None] > 0, np.rint(np.clip(g, -1e300, 1e300) / one), 0.0)
    zero = np.clip(np.where(s > 0, np.rint(-low / one[..., 0]), 0.0), 0, 15) if zeros else None
    code = np.clip(q + zero[..., None], 0, 15) if zeros else np.clip(q, -7, 7) + 8
    code = code.astype(np.uint8).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return code, scale, None if zero is None else zero.astype(np.uint8)


def steps(code, zero, group):
    """code - zero point, whole numbers."""
    z = 8.0 if zero is None else np.repeat((zero & 15).astype(np.float64), group, 1)[:, :code.shape[1]]
    return code.astype(np.float64) - z


def values(code, scale, zero, group):
    return steps(code, zero, group) * np.repeat(scale.astype(np.float64), group, 1)[:, :code.shape[1]]


def two_to_a_byte(code):
    code = np.concatenate([code, np.zeros((code.shape[0], code.shape[1] % 2), np.uint8)], 1)
    return np.ascontiguousarray(code[:, ::2] | code[:, 1::2] << 4)


def product(x, code, scale, zero, group, residual=None):
    """y in 64 bits, and the sum of sizes that bounds of its error go by: the
    code and the zero point of a weight count apart, for they may enter so."""
    x = x.astype(np.float64)
    y = x @ values(code, scale, zero, group).T
    z = np.full(scale.shape, 8.0) if zero is None else (zero & 15).astype(np.float64)
    size = (code + np.repeat(z, group, 1)[:, :code.shape[1]]) * np.repeat(np.abs(scale.astype(np.float64)), group, 1)[:, :code.shape[1]]
    terms = np.abs(x) @ size.T
    far = np.abs(x).max(1, keepdims=True) * size.sum(1)[None]  # what a row's largest element stands for
    if residual is not None:
        y = y + residual
        terms = terms + np.abs(residual)
    return y, terms, far


def product_bound(y, terms, far, groups, kind):
    """Elements of x as two f16 under a row scale: off by 2^-22 of themselves and
    2^-39 of the row's largest.  A group's sum takes up to 9 additions of one
    instruction each, of which tensor cores may drop up to two units of the last
    place (2^-23) of the largest operand; then one rounding per group, scale and join.
    At the end one rounding to the type."""
    held = terms * (2.0 ** -22 + 9 * 2.0 ** -22 + (groups + 24) * 2.0 ** -24) + far * 2.0 ** -39
    return held + HALF[kind] * (np.abs(y) + held) + TINY[kind]


def order(x):
    """Indexes by logit, largest first, equal ones by index; NaN counts as -inf."""
    return np.argsort(-np.where(np.isnan(x), -np.inf, x), kind="stable")


def logprobs(x, scale):
    """ln p [vocab], entropy and the mean size of t under p, of one row, in 64 bits."""
    x = x.astype(np.float64)
    if np.isnan(x).any() or (x == np.inf).any():
        return np.full(len(x), np.nan), np.nan, 0.0
    high = x.max()
    if high == -np.inf:
        return np.full(len(x), -np.inf), 0.0, 0.0
    t = (x - high) * scale
    e = np.exp(t)
    total = e.sum()
    there = e > 0
    mean = (e[there] * t[there]).sum() / total
    return t - np.log(total), np.log(total) - mean, -mean


def logprobs_bound(t, mean, vocab):
    """How far ln p of an element t below the largest logit may be off.  Each t is
    rounded twice and its exponential is good to 2^-21, t itself in the unit of
    a power of two once more; a thread adds at most 64 + vocab / 128 of them in
    fp32 before sums are joined."""
    total = 2.0 ** -21 * (2 + mean) + (64 + vocab / 128) * 2.0 ** -24
    return total + 2.0 ** -23 * (np.abs(t) + 4)
