"""Paged 8-bit cache operators against plain 64-bit references: rotary
positions, page bookkeeping, quantised append and read, attention over the
pages, and a serving loop of all of them."""
import ctypes

import numpy as np
import pytest

import paged_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

NP = {"f32": np.float32, "f16": np.float16}
# A rounding to the type is off by at most half a step.
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11}
TINY = {"f32": 0.0, "f16": 2.0 ** -25}  # half a subnormal step of half precision


class Ordered:
    """The library's calls run on the context's stream, torch's on its own:
    every call waits for what torch has queued."""

    def __init__(self, inner):
        self.inner = inner

    def __getattr__(self, name):
        fn = getattr(self.inner, name)

        def call(*a, **k):
            torch.cuda.synchronize()
            return fn(*a, **k)
        return call


@pytest.fixture(scope="module")
def lib():
    import llamahat
    acc = llamahat.Accelerator(0)
    f = llamahat.CudaKernelFactory()
    return llamahat, acc, Ordered(f.createRoPE(acc)), Ordered(f.createPages(acc))


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def sync():
    torch.cuda.synchronize()


# ------------------------------------------------------------------ rotary

CONFIGS = [
    dict(head_dim=64),
    dict(head_dim=64, layout="half", scaling="llama3", factor=32.0),
    dict(head_dim=128, rot_dim=96, scaling="yarn", factor=4.0),
    dict(head_dim=128, rot_dim=64, layout="half", scaling="linear", factor=4.0),
    dict(head_dim=20, rot_dim=6, layout="half", theta=10000.0),
    dict(head_dim=18, rot_dim=18, theta=10000.0, scaling="yarn", factor=8.0, attn_factor=1.25),
    dict(head_dim=16, rot_dim=0),
    dict(head_dim=512, layout="half", scaling="llama3", factor=8.0),
]


def rope_tolerance(x, cfg, kind):
    """A pair's cos and sin: the angle is held to 2^-26 of a turn (1e-7), the
    function to 2 units of the last place and the factor's product to one
    rounding, 2^-21 in all; the two products and their sum add three
    roundings of (|a| + |b|) m, and the result one of its own type."""
    m = ref.rope_frequencies(cfg)[1] if (cfg.rot_dim or cfg.head_dim) else 1.0
    size = 2 * np.abs(x.astype(np.float64)).max() * m
    return size * (2.0 ** -21 + 3 * 2.0 ** -24 + HALF[kind]) + TINY[kind]


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("transpose", [False, True])
@pytest.mark.parametrize("spec", CONFIGS)
@pytest.mark.parametrize("rows,heads", [(1, 1), (37, 5), (300, 8)])
def test_rope(lib, kind, transpose, spec, rows, heads):
    L, acc, rope, _ = lib
    cfg = L.RopeConfig(**spec)
    rng = np.random.default_rng(rows + heads)
    x = rng.standard_normal((rows, heads, cfg.head_dim)).astype(NP[kind])
    pos = rng.integers(0, 131072, rows).astype(np.int32)
    pos[0] = 2 ** 31 - 1 if rows > 1 else 0
    if rows > 2:
        pos[1], pos[2] = -1, 0
    want = ref.rope(x, pos, cfg, transpose)
    xt, out = dev(x), torch.full((rows, heads, cfg.head_dim), 7.0, dtype=dev(x).dtype, device="cuda")
    rope.apply_scaled(xt, out, dev(pos), cfg, transpose)
    sync()
    got = out.cpu().numpy().astype(np.float64)
    live = pos >= 0
    assert np.all(got[~live] == 7.0)  # rows at negative positions are left as they are
    assert np.abs(got - want)[live].max() <= rope_tolerance(x, cfg, kind)
    rot = cfg.head_dim if cfg.rot_dim is None else cfg.rot_dim
    assert np.array_equal(got[live][..., rot:], x.astype(np.float64)[live][..., rot:])
    # in place, from host memory and into strided rows: the same bits
    rope.apply_scaled(xt, xt, dev(pos), cfg, transpose)
    sync()
    assert np.array_equal(xt.cpu().numpy()[live], out.cpu().numpy()[live])
    assert np.array_equal(xt.cpu().numpy()[~live], x[~live])
    host = np.full_like(x, 7.0)
    rope.apply_scaled(x, host, pos, cfg, transpose)
    assert np.array_equal(host, out.cpu().numpy())
    wide = torch.full((rows, heads * cfg.head_dim + 3), 7.0, dtype=xt.dtype, device="cuda")
    wide[:, 1:-2] = dev(x).view(rows, -1)
    rope.apply_scaled(wide[:, 1:-2], wide[:, 1:-2], dev(pos), cfg, transpose)
    sync()
    assert np.array_equal(wide[:, 1:-2].cpu().numpy()[live], out.view(rows, -1).cpu().numpy()[live])
    assert bool((wide[:, 0] == 7).all()) and bool((wide[:, -2:] == 7).all())


def test_rope_is_its_transpose_by_differences(lib):
    """<R x, g> = <x, R^T g> for random x and g, and the difference quotient of
    a linear map is the map itself: (R(x + h) - R x) = R h."""
    L, acc, rope, _ = lib
    cfg = L.RopeConfig(head_dim=64, rot_dim=48, layout="half", scaling="yarn", factor=4.0)
    rng = np.random.default_rng(5)
    x, g = (dev(rng.standard_normal((23, 3, 64)).astype(np.float32)) for _ in range(2))
    pos = dev(rng.integers(0, 9000, 23).astype(np.int32))
    y, b, shifted = (torch.empty_like(x) for _ in range(3))
    rope.apply_scaled(x, y, pos, cfg)
    rope.apply_scaled(g, b, pos, cfg, transpose=True)
    rope.apply_scaled(x + g, shifted, pos, cfg)
    sync()
    m = ref.rope_frequencies(cfg)[1]
    left, right = (y.double() * g.double()).sum(), (x.double() * b.double()).sum()
    size = float((x.double().abs() * g.double().abs()).sum()) * 2 * m
    assert abs(float(left - right)) <= 2 * size * 2.0 ** -20
    forward = torch.empty_like(x)
    rope.apply_scaled(g, forward, pos, cfg)
    sync()
    tol = 3 * rope_tolerance((x.abs() + g.abs()).cpu().numpy(), cfg, "f32")
    assert float((shifted.double() - y.double() - forward.double()).abs().max()) <= tol


def test_rope_unscaled_agrees_with_rope_rows(lib):
    """Near positions, where the fp32 angle of lc_rope_rows is good to p f 2^-24."""
    L, acc, rope, _ = lib
    rng = np.random.default_rng(6)
    x = rng.standard_normal((33, 4, 64)).astype(np.float32)
    pos = np.arange(33, dtype=np.int32)
    a, b = dev(x), dev(x)
    rope.apply_rows(a, dev(pos), 33, 4, 64, 500000.0)
    rope.apply_scaled(b, b, dev(pos), L.RopeConfig())
    sync()
    tol = 2 * np.abs(x).max() * (2.0 ** -20 + 2 * 33 * 2.0 ** -24)
    assert float((a - b).abs().max()) <= tol


# ------------------------------------------------------------------- pages

def pages_case(rng, n, hi, new, page, ended, slack, stride_extra=0):
    lens = rng.integers(0, hi + 1, n)
    add = rng.integers(0, new + 1, n)
    add[rng.permutation(n)[:ended]] = -1
    need = -(-lens // page)
    want = -(-(lens + np.maximum(add, 0)) // page)
    n_pages = int(want.sum()) + int(need.sum()) + slack
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n, max(1, int(want.max())) + stride_extra), -1, np.int32)
    at = 0
    for s in range(n):
        table[s, :need[s]] = perm[at:at + need[s]]
        at += need[s]
    return lens.astype(np.int32), add.astype(np.int32), table, perm[at:], n_pages


def run_pages(pages, lens, add, table, free, n_pages, page, cap, in_place=False, host=False):
    to = (lambda x: np.array(x)) if host else dev
    new = (lambda n: np.full(n, -9, np.int32)) if host else (lambda n: torch.full((n,), -9, dtype=torch.int32, device="cuda"))
    fl = np.full(n_pages, -1, np.int32)
    fl[:len(free)] = free
    d = {"lens": to(lens), "add": to(add), "table": to(table), "free": to(fl), "count": to(np.array([len(free)], np.int32))}
    o = {k: new(m) for k, m in (("lens", len(lens)), ("q_start", len(lens) + 1), ("slots", cap), ("positions", cap),
                                ("ids", cap), ("count", 1), ("status", 2))}
    if in_place:
        o["lens"], o["count"] = d["lens"], d["count"]
    pages.step(d["lens"], d["add"], d["table"], d["free"], d["count"], page, o["lens"], o["q_start"], o["slots"],
               o["positions"], o["ids"], o["count"], o["status"])
    sync()
    get = lambda x: x if host else x.cpu().numpy()  # noqa: E731
    return {k: get(v) for k, v in o.items()} | {"table": get(d["table"]), "free": get(d["free"])}


@pytest.mark.parametrize("n,hi,new,page,ended", [(1, 0, 1, 16, 0), (1, 100, 4096, 16, 0), (7, 50, 3, 32, 2),
                                                 (64, 300, 1, 64, 5), (300, 40, 90, 128, 30), (1023, 200, 33, 16, 100),
                                                 (4096, 60, 20, 16, 500), (5, 64, 0, 32, 0), (6, 90, 9, 16, 6)])
@pytest.mark.parametrize("in_place", [False, True])
def test_pages_step(lib, n, hi, new, page, ended, in_place):
    pages = lib[3]
    rng = np.random.default_rng(n * 7 + new)
    lens, add, table, free, n_pages = pages_case(rng, n, hi, new, page, ended, 3)
    cap = int(np.maximum(add, 0).sum()) + 3
    want_table = table.copy()
    want = ref.pages_step(lens.tolist(), add.tolist(), page, want_table, free.tolist(), cap)
    got = run_pages(pages, lens, add, table, free, n_pages, page, cap, in_place)
    assert got["status"].tolist() == [0, 0]
    assert np.array_equal(got["table"], want_table)
    for key, value in zip(("lens", "q_start", "slots", "positions", "ids"), want):
        assert got[key].tolist() == value, key
    assert got["count"][0] == len(want[5])
    assert got["free"][:len(want[5])].tolist() == want[5]
    if n <= 64:
        host = run_pages(pages, lens, add, table, free, n_pages, page, cap, in_place, host=True)
        for key in ("lens", "q_start", "slots", "positions", "ids", "table", "status", "count"):
            assert np.array_equal(host[key], got[key]), key


@pytest.mark.parametrize("what,status", [("short", [1, 2]), ("row", [2, 1]), ("capacity", [3, 40]), ("length", [4, 2]),
                                         ("count", [5, -1]), ("returned", [5, 7])])
def test_pages_step_refuses_and_changes_nothing(lib, what, status):
    pages = lib[3]
    page, lens, add = 16, [5, 30, 16], [20, 3, 17]  # 25 -> 2 pages, 33 -> 3, 33 -> 3: 1 + 1 + 2 new pages
    table = np.array([[0, -1, -1], [1, 2, -1], [3, -1, -1]], np.int32)
    free, n_pages, cap = [4, 5, 6, 7], 8, 64
    if what == "short":
        free = [4, 5]
    if what == "row":
        table = np.ascontiguousarray(table[:, :2])
    if what == "capacity":
        cap = 39
    if what == "length":
        lens = [5, 30, -1]
    if what == "returned":  # ended sequences return more pages than there can be
        add, n_pages, free = [-1, -1, -1], 6, [4, 5, 0]
    lens, add = np.array(lens, np.int32), np.array(add, np.int32)
    if what == "count":
        fl, o = dev(np.array(free, np.int32)), [torch.zeros(k, dtype=torch.int32, device="cuda") for k in (3, 4, cap, cap, cap, 1, 2)]
        t = dev(table)
        pages.step(dev(lens), dev(add), t, fl, dev(np.array([-1], np.int32)), page, *o)
        sync()
        got = dict(zip(("lens", "q_start", "slots", "positions", "ids", "count", "status"), [x.cpu().numpy() for x in o]))
        got |= {"table": t.cpu().numpy(), "free": fl.cpu().numpy()}
        free = [-1] * 0
        assert got["count"][0] == -1
    else:
        got = run_pages(pages, lens, add, table, np.array(free, np.int32), n_pages, page, cap)
        assert got["count"][0] == len(free)
    assert got["status"].tolist() == status
    assert np.array_equal(got["table"], table) and np.array_equal(got["lens"], lens)
    assert not got["q_start"].any()
    for key in ("slots", "positions", "ids"):
        assert (got[key] == -1).all()
    assert got["free"][:len(free)].tolist() == list(free)


# ------------------------------------------------------------ append, read

def make_pool(rng, n_pages, kv, page, d, fmt):
    pool = {}
    for name in ("k", "v"):
        codes = rng.integers(0, 256, (n_pages, kv, page, d)).astype(np.uint8)
        if fmt == "i8":
            codes[codes == 0x80] = 0x81  # -128 is no code
        else:
            codes[(codes & 0x7F) == 0x7F] = 0
        pool[name] = codes
        pool[name + "_scale"] = np.exp(rng.standard_normal((n_pages, kv)) * 0.4 - 4).astype(np.float32)
    return pool


def cache_of(lib, pool, fmt):
    L, acc = lib[:2]
    t = {k: dev(v) for k, v in pool.items()}
    return Ordered(L.PagedKV8(t["k"], t["v"], t["k_scale"], t["v_scale"], format=fmt, acc=acc)), t


def runs(rng, spans, page, n_pages):
    """Slots of (start, count) spans of sequences, each on pages of its own."""
    perm = list(rng.permutation(n_pages))
    out = []
    for start, count in spans:
        ids = [perm.pop() for _ in range(-(-(start + count) // page))]
        out += [int(ids[t // page]) * page + t % page for t in range(start, start + count)]
    return np.array(out, np.int32)


def assert_same_codes(got, want, fmt, what):
    same = got == want
    if got.dtype == np.uint8 and fmt == "e4m3":  # -0.0 and 0.0 of e4m3 are one value
        same |= (got & 0x7F == 0) & (want & 0x7F == 0)
    assert same.all(), (what, np.argwhere(~same)[:4])


SPANS = [[(0, 1)], [(5, 1), (15, 1), (16, 1), (0, 1)], [(0, 16)], [(3, 130), (0, 33), (31, 2)], [(127, 200), (1, 1)]]


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("kv,page,d", [(1, 16, 64), (8, 32, 64), (3, 64, 128), (2, 128, 64)])
@pytest.mark.parametrize("spans", range(len(SPANS)))
def test_append_and_read(lib, kind, fmt, kv, page, d, spans):
    rng = np.random.default_rng(spans * 31 + page + kv)
    n_pages = 40
    pool = make_pool(rng, n_pages, kv, page, d, fmt)
    slots = runs(rng, SPANS[spans], page, n_pages)
    if spans == 3:  # rows without a slot, and slots behind the cache, in between
        slots = np.insert(slots, [0, 7, len(slots)], [-1, -1, n_pages * page])
    n = len(slots)
    rows = {k: (rng.standard_normal((n, kv, d)) * np.exp(rng.standard_normal((n, 1, 1)))).astype(NP[kind]) for k in "kv"}
    if spans == 3:
        rows["k"][3, 0, :3] = [np.nan, np.inf, -np.inf]
        rows["v"][4:8] = 0.0
    cache, t = cache_of(lib, pool, fmt)
    want = {k: v.copy() for k, v in pool.items()}
    for name in "kv":
        ref.append(want[name], want[name + "_scale"], rows[name], slots, fmt)
    cache.append(dev(rows["k"]), dev(rows["v"]), dev(slots))
    sync()
    for name in want:
        got = t[name].cpu().numpy()
        assert_same_codes(got, want[name], fmt, name)
    # A second time: the scales are there, so nothing moves.  Where skipped
    # rows split a page into two runs, the first now meets the second's
    # scale and is rounded once instead of twice.
    before = {k: v.clone() for k, v in t.items()}
    cache.append(dev(rows["k"]), dev(rows["v"]), dev(slots))
    sync()
    for name in "kv":
        ref.append(want[name], want[name + "_scale"], rows[name], slots, fmt)
    for name in want:
        assert_same_codes(t[name].cpu().numpy(), want[name], fmt, name)
        assert spans == 3 or torch.equal(before[name], t[name]), name
    # read back: one rounding of code * scale
    k, v = (torch.full((n, kv, d), 7.0, dtype=dev(rows["k"]).dtype, device="cuda") for _ in "kv")
    cache.read(k, v, dev(slots))
    sync()
    ok = (slots >= 0) & (slots < n_pages * page)
    for name, x in (("k", k), ("v", v)):
        x = x.cpu().numpy().astype(np.float64)
        value = ref.decode(want[name][slots[ok] // page, :, slots[ok] % page], fmt) * want[name + "_scale"][slots[ok] // page].astype(np.float64)[:, :, None]
        assert (np.abs(x[ok] - value) <= np.abs(value) * (2.0 ** -24 + HALF[kind]) + TINY[kind]).all()
        assert (x[~ok] == 7.0).all()
    # strided rows and host rows: the same
    wide = {name: torch.zeros(n, kv * d + 5, dtype=k.dtype, device="cuda") for name in "kv"}
    for name in "kv":
        wide[name][:, 3:-2] = dev(rows[name]).view(n, -1)
    other, u = cache_of(lib, pool, fmt)
    other.append(wide["k"][:, 3:-2], wide["v"][:, 3:-2], dev(slots))
    third, w = cache_of(lib, pool, fmt)
    third.append(rows["k"], rows["v"], slots)
    sync()
    for name in want:
        assert torch.equal(u[name], before[name]) and torch.equal(w[name], before[name]), name


def test_append_rounds_ties_of_the_quotient_only(lib):
    """Scale 3 / 127: quotients that fp32 division rounds onto a tie, and real ties."""
    rng = np.random.default_rng(9)
    for fmt in ("i8", "e4m3"):
        limit = ref.LIMIT[fmt]
        top = np.float32(3.0)
        s = np.float32(top / np.float32(limit))
        grid = np.arange(1, 254, dtype=np.float64) / 2 if fmt == "i8" else (ref.E4M3[:0x7D] + ref.E4M3[1:0x7E]) / 2
        near = (grid * float(s)).astype(np.float32)
        x = np.concatenate([near, np.nextafter(near, np.float32(9)), np.nextafter(near, np.float32(-9)), -near])
        x = np.resize(x, (128, 1, 64)).astype(np.float32)
        x[0, 0, 0] = top
        pool = make_pool(rng, 1, 1, 128, 64, fmt)
        cache, t = cache_of(lib, pool, fmt)
        want = {k: v.copy() for k, v in pool.items()}
        slots = np.arange(128, dtype=np.int32)
        ref.append(want["k"], want["k_scale"], x, slots, fmt)
        cache.append(dev(x), dev(x), dev(slots))
        sync()
        got = t["k"].cpu().numpy()
        assert ((got == want["k"]) | ((got & 0x7F == 0) & (want["k"] & 0x7F == 0))).all()


# --------------------------------------------------------------- attention

def attention_tolerance(terms, kind, d):
    """Error of a row against the exact result.  A score's d products sum in
    fp32, each step at most one unit 2^-23 of the running size, q and the
    scale adding a few more: ds = (d + 16) 2^-23 max_t sum |q k| scale.  The
    weights are then off by a factor exp(+-2 ds) and by the exponential's and
    the running rescale's roundings, 16 units 2^-23; the weighted sum over n
    tokens and its normaliser add n units each.  Half precision rounds each
    weight and the result to its type."""
    x, pv, n = terms
    ds = (d + 16) * 2.0 ** -23 * x
    rel = 2 * ds + (16 + 2 * n) * 2.0 ** -23 + (2 * HALF["f16"] if kind == "f16" else 0.0)
    return pv.max() * rel + (HALF[kind] * pv.max() + TINY[kind])


def attention_case(lib, rng, lens, counts, heads, kv, page, d, fmt, kind, extra_rows=2, scale=None):
    n = len(lens)
    need = [-(-int(t) // page) for t in lens]
    n_pages = sum(need) + 3
    pool = make_pool(rng, n_pages, kv, page, d, fmt)
    for name in ("k_scale", "v_scale"):
        pool[name] = (pool[name] * (1.0 if fmt == "i8" else 0.05)).astype(np.float32)
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n, max(1, max(need))), -1, np.int32)
    at = 0
    for s, k in enumerate(need):
        table[s, :k] = perm[at:at + k]
        at += k
        if fmt == "e4m3" and lens[s] % page:  # NaN behind the end of the last page
            for name in "kv":
                pool[name][table[s, k - 1], :, lens[s] % page:] = 0x7F
    for p in perm[at:]:  # pages that nobody holds
        pool["k_scale"][p] = pool["v_scale"][p] = np.nan
    q_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    rows = int(q_start[-1]) + extra_rows
    q = rng.standard_normal((rows, heads, d)).astype(NP[kind])
    return pool, table, q_start, q


def check_attention(lib, pool, table, q_start, q, lens, fmt, kind, max_q, scale=None, decode=False):
    d = q.shape[2]
    sc = d ** -0.5 if scale is None else scale
    cache, t = cache_of(lib, pool, fmt)
    out = torch.full(q.shape, 7.0, dtype=dev(q).dtype, device="cuda")
    lens = np.asarray(lens, np.int32)
    cache.attention(dev(q), out, None if decode else dev(q_start), dev(lens), dev(table), max_q=max_q, scale=scale)
    sync()
    got = out.cpu().numpy().astype(np.float64)
    terms = {}
    want = ref.attention(q, None if decode else q_start, lens, table, pool["k"], pool["v"], pool["k_scale"],
                         pool["v_scale"], fmt, sc, np.full(q.shape, 7.0), terms)
    for j in range(q.shape[0]):
        for h in range(q.shape[1]):
            if (j, h) in terms:
                off = np.abs(got[j, h] - want[j, h]).max()
                assert off <= attention_tolerance(terms[j, h], kind, d), (j, h, off)
            else:
                assert np.array_equal(got[j, h], want[j, h]), (j, h)
    return got


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,kv,page,d", [(8, 2, 32, 64), (4, 4, 16, 64), (6, 2, 64, 128), (24, 2, 128, 64)])
def test_attention_decode(lib, kind, fmt, heads, kv, page, d):
    rng = np.random.default_rng(heads + page)
    lens = [1, 0, page - 1, page, page + 1, 150, 517, 16, 17]
    counts = [1] * len(lens)
    case = attention_case(lib, rng, lens, counts, heads, kv, page, d, fmt, kind, extra_rows=0)
    a = check_attention(lib, *case, lens, fmt, kind, 1, decode=True)
    b = check_attention(lib, *case, lens, fmt, kind, 1)
    assert np.array_equal(a, b)


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("n,length", [(1, 5000), (3, 2111), (40, 300)])
def test_attention_decode_long(lib, fmt, n, length):
    rng = np.random.default_rng(n)
    lens = [int(x) for x in rng.integers(length // 2, length, n)]
    lens[0] = length
    case = attention_case(lib, rng, lens, [1] * n, 8, 2, 32, 64, fmt, "f32", extra_rows=0)
    check_attention(lib, *case, lens, fmt, "f32", 1, decode=True)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,kv,page,d", [(8, 2, 32, 64), (3, 1, 16, 128), (8, 8, 64, 64), (10, 1, 128, 64)])
@pytest.mark.parametrize("lens,counts", [([2, 40, 0, 33], [2, 2, 2, 2]), ([70, 0, 1, 33], [70, 0, 5, 9]),
                                         ([300, 129], [37, 129]), ([260], [200])])
def test_attention_chunks(lib, kind, fmt, heads, kv, page, d, lens, counts):
    """Chunks that start the cache, continue it, and ask for more positions than it holds."""
    rng = np.random.default_rng(heads + page + len(lens))
    case = attention_case(lib, rng, lens, counts, heads, kv, page, d, fmt, kind)
    check_attention(lib, *case, lens, fmt, kind, max(counts))


def exact_on_gpu(pool, table, q_start, lens, q, fmt, scale):
    """Attention in 64 bits with torch, a sequence and kv head at a time; and
    per row what an error bound needs: max_t sum |q k| scale and sum p |v|."""
    t = {k: dev(v) for k, v in pool.items()}
    page, group = pool["k"].shape[2], q.shape[1] // pool["k"].shape[1]
    values = torch.from_numpy(ref.decode(np.arange(256, dtype=np.uint8), fmt)).cuda()
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    size, weight = (torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda") for _ in range(2))
    x = dev(q).double()
    for s, length in enumerate(lens):
        b, e = int(q_start[s]), int(q_start[s + 1])
        if b == e or length == 0:
            continue
        ids = dev(table[s, : -(-length // page)].astype(np.int64))
        for h in range(pool["k"].shape[1]):
            k, v = ((values[t[n][ids, h].long()] * t[n + "_scale"][ids, h].double()[:, None, None]).reshape(-1, q.shape[2])[:length]
                    for n in "kv")
            hidden = torch.arange(length, device="cuda")[None] > torch.arange(length - (e - b), length, device="cuda")[:, None]
            for a in range(h * group, (h + 1) * group):
                w = torch.softmax((x[b:e, a] @ k.T * scale).masked_fill(hidden, -torch.inf), -1)
                out[b:e, a] = w @ v
                size[b:e, a] = (x[b:e, a].abs() @ k.abs().T * scale).masked_fill(hidden, 0).amax(-1)
                weight[b:e, a] = (w @ v.abs()).amax(-1)
    return out, size, weight


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
@pytest.mark.parametrize("heads,kv,page,d,lens,counts", [
    (32, 8, 32, 64, [937, 3022, 3377, 3170, 2659], [253, 278, 262, 75, 461]),
    (8, 2, 64, 128, [1500, 700], [1400, 333]),
    (24, 8, 16, 64, [2100], [1000]),
    (8, 8, 128, 64, [5000, 300, 64], [20, 300, 64]),
])
def test_attention_prompts_at_length(lib, kind, fmt, heads, kv, page, d, lens, counts):
    """Many units, each over several CTAs: every row, every time, within its bound."""
    rng = np.random.default_rng(heads + page)
    pool, table, q_start, q = attention_case(lib, rng, lens, counts, heads, kv, page, d, fmt, kind, extra_rows=0)
    want, size, weight = exact_on_gpu(pool, table, q_start, lens, q, fmt, d ** -0.5)
    # attention_tolerance with the row's own terms; tokens of a row: at most max(lens)
    rel = 2 * (d + 16) * 2.0 ** -23 * size + (16 + 2 * max(lens)) * 2.0 ** -23 + (2 * HALF["f16"] if kind == "f16" else 0.0)
    bound = weight * rel + HALF[kind] * weight + TINY[kind]
    cache, _ = cache_of(lib, pool, fmt)
    args = dev(q_start), dev(np.array(lens, np.int32)), dev(table)
    first = None
    for _ in range(4):
        out = torch.full(q.shape, 7.0, dtype=dev(q).dtype, device="cuda")
        cache.attention(dev(q), out, *args, max_q=max(counts))
        sync()
        off = (out.double() - want).abs().amax(-1)
        assert bool((off <= bound).all()), (off / bound).max()
        first = out if first is None else first
        assert torch.equal(first, out)


def test_attention_of_a_call_of_seconds(lib):
    """A prompt of 420,000 positions, every query the same (row stride 0): its
    waits have limits of seconds, the call as a whole has none."""
    rng = np.random.default_rng(12)
    n, heads, page, d = 420_000, 32, 128, 64
    pool, table, _, _ = attention_case(lib, rng, [n], [1], 1, 1, page, d, "i8", "f32")
    q = rng.standard_normal((heads, d)).astype(np.float32)
    cache, _ = cache_of(lib, pool, "i8")
    out = torch.full((n, heads, d), 7.0, device="cuda")
    args = dev(np.array([0, n], np.int32)), dev(np.array([n], np.int32)), dev(table)
    cache.attention(dev(q)[None].expand(n, heads, d), out, *args, max_q=n)
    sync()
    assert bool(torch.isfinite(out).all())
    for j in (0, 63, 64, 4095, 211_111, n - 1):
        terms = {}
        want = ref.attention(q[None], np.array([0, 1]), [j + 1], table, pool["k"], pool["v"], pool["k_scale"],
                             pool["v_scale"], "i8", d ** -0.5, np.zeros((1, heads, d)), terms)
        got = out[j].cpu().numpy()
        for h in range(0, heads, 5):
            assert np.abs(got[h] - want[0, h]).max() <= attention_tolerance(terms[0, h], "f32", d), (j, h)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("heads,kv,page,d", [(16, 4, 16, 64), (8, 2, 64, 128)])
def test_attention_of_units_of_one_tile_and_two(lib, kind, heads, kv, page, d):
    """Prompts whose last rows fill one tile, two, or a corner of one, long ones
    among many that end within a step."""
    rng = np.random.default_rng(d)
    counts = np.tile([3, 70, 40, 1, 64, 0, 33, 32, 129, 5], 9)
    lens = counts + np.tile([0, 5, 1200, 0, 0, 700, 61, 0, 30], 10)
    pool, table, q_start, q = attention_case(lib, rng, lens.tolist(), counts.tolist(), heads, kv, page, d, "e4m3", kind, extra_rows=0)
    want, size, weight = exact_on_gpu(pool, table, q_start, lens.tolist(), q, "e4m3", d ** -0.5)
    rel = 2 * (d + 16) * 2.0 ** -23 * size + (16 + 2 * lens.max()) * 2.0 ** -23 + (2 * HALF["f16"] if kind == "f16" else 0.0)
    bound = weight * rel + HALF[kind] * weight + TINY[kind]
    cache, _ = cache_of(lib, pool, "e4m3")
    args = dev(q_start), dev(lens.astype(np.int32)), dev(table)
    first = None
    for _ in range(6):
        out = torch.full(q.shape, 7.0, dtype=dev(q).dtype, device="cuda")
        cache.attention(dev(q), out, *args, max_q=int(counts.max()))
        sync()
        off = (out.double() - want).abs().amax(-1)
        assert bool((off <= bound).all()), (off / bound).max()
        first = out if first is None else first
        assert torch.equal(first, out)


@pytest.mark.parametrize("per", [1, 5])
def test_attention_of_4096_sequences(lib, per):
    """The largest number of sequences: no longer than a page or two each, some empty."""
    rng = np.random.default_rng(per)
    lens = rng.integers(0, 40, 4096)
    counts = np.full(4096, per)
    pool, table, q_start, q = attention_case(lib, rng, lens, counts, 4, 1, 16, 64, "i8", "f32", extra_rows=3)
    cache, _ = cache_of(lib, pool, "i8")
    out = torch.full(q.shape, 7.0, device="cuda")
    cache.attention(dev(q), out, dev(q_start), dev(lens.astype(np.int32)), dev(table), max_q=per)
    sync()
    got = out.cpu().numpy()
    assert (got[-3:] == 7).all()
    some = list(range(0, 4096, 64)) + [4095]
    for s in some:
        rows = slice(q_start[s], q_start[s + 1])
        terms = {}
        want = ref.attention(q[rows], np.array([0, per]), [int(lens[s])], table[s:s + 1], pool["k"], pool["v"],
                             pool["k_scale"], pool["v_scale"], "i8", 0.125, np.zeros((per, 4, 64)), terms)
        for key in np.ndindex(per, 4):
            off = np.abs(got[rows][key] - want[key]).max()
            assert off <= (attention_tolerance(terms[key], "f32", 64) if key in terms else 0.0), (s, key)


def test_append_of_a_padded_batch(lib):
    """Rows without a slot before, between and behind: what is written is what the rows alone give."""
    rng = np.random.default_rng(3)
    pool = make_pool(rng, 9, 2, 32, 64, "i8")
    slots = runs(rng, [(0, 3), (31, 2), (5, 1), (64, 40)], 32, 9)
    rows = rng.standard_normal((len(slots), 2, 64)).astype(np.float32)
    at = np.sort(rng.choice(np.arange(700, 2900), len(slots), replace=False))
    at[1:3] = at[0] + 1 + np.arange(2)  # neighbours too
    at = np.unique(at)
    n = len(at)
    padded = np.full(20000, -1, np.int32)
    padded[at] = slots[:n]
    wide = np.zeros((20000, 2, 64), np.float32)
    wide[at] = rows[:n]
    a, ta = cache_of(lib, pool, "i8")
    want = {k: v.copy() for k, v in pool.items()}
    a.append(dev(wide), dev(wide), dev(padded))
    sync()
    for name in "kv":
        ref.append(want[name], want[name + "_scale"], wide, padded, "i8")
    for name in want:
        assert np.array_equal(ta[name].cpu().numpy(), want[name]), name


@pytest.mark.parametrize("fmt,kind,page,d", [("i8", "f32", 64, 64), ("e4m3", "f16", 128, 64), ("i8", "f16", 64, 128),
                                             ("e4m3", "f32", 128, 128), ("i8", "f32", 32, 128)])
def test_append_of_long_prompts_in_large_pages(lib, fmt, kind, page, d):
    """More rows than there is room for side by side: pages longer than the rows
    that are looked at together, begun in their middle, cut by skipped rows,
    with infinities, and codes below that are rounded anew."""
    rng = np.random.default_rng(page + d)
    spans = [(0, 9000), (37, 5000), (1, 1), (page - 1, 2), (page // 2 + 3, 4000), (0, page), (90, 1400)]
    n_pages = sum(-(-(a + b) // page) for a, b in spans) + 1
    pool = make_pool(rng, n_pages, 1, page, d, fmt)
    slots = runs(rng, spans, page, n_pages)
    slots = np.insert(slots, [5, 6000, 6001, 9003, len(slots)], -1)
    n = len(slots)
    assert n >= 19000
    rows = {k: (rng.standard_normal((n, 1, d)) * np.exp(rng.standard_normal((n, 1, 1)))).astype(NP[kind]) for k in "kv"}
    rows["k"][[3, 8000, 14010], 0, 1:3] = [np.inf, -np.inf]
    rows["v"][4:300] = 0.0
    cache, t = cache_of(lib, pool, fmt)
    want = {k: v.copy() for k, v in pool.items()}
    for name in "kv":
        ref.append(want[name], want[name + "_scale"], rows[name], slots, fmt)
    cache.append(dev(rows["k"]), dev(rows["v"]), dev(slots))
    sync()
    for name in want:
        assert_same_codes(t[name].cpu().numpy(), want[name], fmt, name)


@pytest.mark.parametrize("max_q", [1, 2, 9, 1000])
def test_attention_holds_for_any_max_q(lib, max_q):
    rng = np.random.default_rng(4)
    lens, counts = [61, 200, 7], [3, 50, 1]
    case = attention_case(lib, rng, lens, counts, 8, 2, 32, 64, "i8", "f32")
    check_attention(lib, *case, lens, "i8", "f32", max_q)


@pytest.mark.parametrize("max_q,counts", [(1, [1, 1]), (40, [40, 20])])
def test_attention_scale_large_scores_and_missing_pages(lib, max_q, counts):
    """Scores of a few hundred (the softmax is nearly one-hot), a scale of the
    caller's, and table entries outside the cache, whose tokens are not seen."""
    rng = np.random.default_rng(12)
    lens = [170, 95]
    pool, table, q_start, q = attention_case(lib, rng, lens, counts, 8, 2, 32, 64, "i8", "f32")
    table[0, 1], table[1, 2] = -1, 1 << 20
    check_attention(lib, pool, table, q_start, q * np.float32(20), lens, "i8", "f32", max_q, scale=0.3)
    table[0, :] = -5  # a sequence of which nothing is left
    got = check_attention(lib, pool, table, q_start, q, lens, "i8", "f32", max_q)
    assert not got[:counts[0]].any()


def test_attention_is_the_same_every_time_and_strided(lib):
    rng = np.random.default_rng(8)
    lens = [900, 33, 400]
    for counts, max_q in (([1, 1, 1], 1), ([90, 33, 61], 90)):
        pool, table, q_start, q = attention_case(lib, rng, lens, counts, 8, 2, 32, 64, "i8", "f32", extra_rows=0)
        cache, t = cache_of(lib, pool, "i8")
        rows = q.shape[0]
        wide_q = torch.zeros(rows, 8 * 64 + 8, device="cuda")
        wide_q[:, 4:-4] = dev(q).view(rows, -1)
        first = None
        args = dev(q_start), dev(np.array(lens, np.int32)), dev(table)
        sync()
        for k in range(4):
            out = torch.full((rows, 8 * 64 + 2), 7.0, device="cuda")
            sync()
            cache.attention(wide_q[:, 4:-4], out[:, 1:-1], *args, max_q=max_q)
            sync()
            assert bool((out[:, 0] == 7).all()) and bool((out[:, -1] == 7).all())
            first = out if first is None else first
            assert torch.equal(first, out)
        host = np.zeros_like(q)
        cache.attention(q, host, q_start, np.array(lens, np.int32), table, max_q=max_q)
        assert np.array_equal(host.reshape(rows, -1), first[:, 1:-1].cpu().numpy())


def test_offsets_past_32_bits(lib):
    """The last pages of a cache whose codes reach past byte 2^32."""
    L, acc = lib[:2]
    kv, page, d, n_pages = 64, 128, 128, 4200  # 1 MiB a page: 4.4e9 bytes
    k = torch.zeros(n_pages, kv, page, d, dtype=torch.uint8, device="cuda")
    v = torch.zeros_like(k)
    ks, vs = (torch.zeros(n_pages, kv, device="cuda") for _ in "kv")
    cache = L.PagedKV8(k, v, ks, vs, acc=acc)
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(200, kv, d, device="cuda", generator=g)
    at = torch.arange(200, dtype=torch.int32, device="cuda") + (n_pages - 2) * page
    back_k, back_v, out = torch.zeros_like(rows), torch.zeros_like(rows), torch.zeros(1, kv, d, device="cuda")
    table = torch.tensor([[n_pages - 2, n_pages - 1]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([200], dtype=torch.int32, device="cuda")
    q = torch.randn(1, kv, d, device="cuda", generator=g)
    sync()
    cache.append(rows, rows, at)
    cache.read(back_k, back_v, at)
    cache.attention(q, out, None, lens, table)
    sync()
    # half a code step of the largest value of a page and head
    assert float((back_k - rows).abs().max()) <= float(rows.abs().max()) / 127 * 0.5 * (1 + 2.0 ** -20)
    assert torch.equal(back_k, back_v)
    x = torch.einsum("hd,thd->ht", q[0].double(), back_k.double()) * d ** -0.5
    want = torch.einsum("ht,thd->hd", torch.softmax(x, -1), back_v.double())
    size = float((q.double().abs().amax() * back_k.double().abs().sum(-1)).max()) * d ** -0.5
    assert float((out[0] - want).abs().max()) <= float(rows.abs().max()) * (2 * (d + 16) * size + 16 + 400) * 2.0 ** -23
    assert not k[: n_pages - 2].any()


# -------------------------------------------------------------- the set of them

def serve(lib, steps, page, cfg, rng, graph=False):
    """Sequences of random rows through rope, pages, append and attention;
    returns what every step's attention gave, and all rows by sequence."""
    L, acc = lib[:2]
    rope, pages = (x.inner for x in lib[2:])
    n, heads, kv, d, n_pages = 5, 8, 2, 64, 60
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    t = {name: torch.zeros(n_pages, kv, page, d, dtype=torch.uint8, device="cuda") for name in "kv"}
    sc = {name: torch.zeros(n_pages, kv, device="cuda") for name in "kv"}
    cache = L.PagedKV8(t["k"], t["v"], sc["k"], sc["v"], acc=acc)
    cap = 64
    lens, new, table, free = i32(n), i32(n), i32(n, 12), torch.arange(n_pages, dtype=torch.int32, device="cuda")
    count = torch.full((1,), n_pages, dtype=torch.int32, device="cuda")
    q_start, slots, pos, ids, status = i32(n + 1), i32(cap), i32(cap), i32(cap), i32(2)
    q, k, v = (torch.zeros(cap, h, d, device="cuda") for h in (heads, kv, kv))
    out = torch.zeros(cap, heads, d, device="cuda")
    sync()

    def step():
        pages.step(lens, new, table, free, count, page, lens, q_start, slots, pos, ids, count, status)
        rope.apply_scaled(q, q, pos, cfg)
        rope.apply_scaled(k, k, pos, cfg)
        cache.append(k, v, slots)
        cache.attention(q, out, q_start, lens, table, max_q=cap)

    g = None
    stream = torch.cuda.ExternalStream(acc.stream, device=torch.device("cuda", 0))
    if graph:
        step()  # first use outside the capture
        sync()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step()
        for x in (lens, table, *t.values(), *sc.values()):
            x.zero_()
        free.copy_(torch.arange(n_pages, dtype=torch.int32, device="cuda"))
        count.fill_(n_pages)
    got, rows, held = [], {s: [] for s in range(n)}, [0] * n
    for add in steps:
        total = sum(max(a, 0) for a in add)
        for x in (q, k, v):
            x.zero_()
            x[:total] = dev(rng.standard_normal((total, *x.shape[1:])).astype(np.float32))
        new.copy_(dev(np.array(add, np.int32)))
        fresh = [x[:total].cpu().numpy().copy() for x in (q, k, v)]
        out.fill_(7.0)
        sync()
        if graph:
            with torch.cuda.stream(stream):
                g.replay()
        else:
            step()
        sync()
        assert status.tolist() == [0, 0]
        at, queries = 0, []
        for s, a in enumerate(add):
            if a < 0:
                rows[s], held[s] = [], 0
            for i in range(max(a, 0)):
                rows[s].append((fresh[1][at], fresh[2][at]))
                queries.append((s, held[s] + i, fresh[0][at]))
                at += 1
            held[s] += max(a, 0)
        assert lens.tolist() == held
        got.append((out.cpu().numpy().copy(), queries, {s: list(r) for s, r in rows.items()}))
    return got, (kv, heads, d)


STEPS = [[9, 0, 33, 1, 5], [1, 1, 1, 1, 1], [1, 20, -1, 1, 1], [-1, 1, 7, 1, 1], [30, 1, 1, -1, 1], [1, 1, 1, 1, 1]]


@pytest.mark.parametrize("graph", [False, True])
def test_serving_steps(lib, graph):
    """Every step's attention against exact attention over the rows as given:
    what is left between them is the 8-bit rounding of keys and values."""
    L = lib[0]
    cfg = L.RopeConfig.llama32()
    got, (kv, heads, d) = serve(lib, STEPS, 16, cfg, np.random.default_rng(3), graph)
    for out, queries, rows in got:
        for i, (s, p, q) in enumerate(queries):
            kk = ref.rope(np.stack([r[0] for r in rows[s][:p + 1]]), range(p + 1), cfg)
            vv = np.stack([r[1] for r in rows[s][:p + 1]]).astype(np.float64)
            qq = ref.rope(q[None], [p], cfg)[0]
            for h in range(heads):
                g = h // (heads // kv)
                # A stored value is off by half a code step when it comes, and by half a step
                # again each time its page's scale grows, at most once for every later token
                # of the page, 16 in all: 8 steps of the page's largest value / 127 bound it.
                dk, dv = np.abs(kk).max() / 127 * 8, np.abs(vv).max() / 127 * 8
                x = kk[:, g] @ qq[h] * d ** -0.5
                w = np.exp(x - x.max())
                w /= w.sum()
                ds = dk * np.abs(qq[h]).sum() * d ** -0.5
                assert np.abs(out[i, h] - w @ vv[:, g]).max() <= dv + np.abs(vv).max() * (np.exp(2 * ds) - 1)
        assert (out[len(queries):] == 7.0).all()


def test_serving_steps_captured_and_eager_agree(lib):
    L = lib[0]
    cfg = L.RopeConfig.llama32()
    a, _ = serve(lib, STEPS, 32, cfg, np.random.default_rng(7), False)
    b, _ = serve(lib, STEPS, 32, cfg, np.random.default_rng(7), True)
    for (x, *_), (y, *_) in zip(a, b):
        assert np.array_equal(x, y)


def test_two_contexts_at_once(lib):
    """Calls of two contexts overlap on the GPU: neither sees the other's workspace."""
    L, acc = lib[:2]
    other = L.Accelerator(0)
    rng = np.random.default_rng(2)
    lens = [4000, 3500]
    pool, table, q_start, q = attention_case(lib, rng, lens, [1, 1], 8, 2, 32, 64, "i8", "f32", extra_rows=0)
    caches = [cache_of((L, a), pool, "i8")[0].inner for a in (acc, other)]
    args = dev(np.array(lens, np.int32)), dev(table)
    qs = [dev(q), dev(-q)]
    want = []
    for c, x in zip(caches, qs):
        out = torch.zeros_like(x)
        sync()
        c.attention(x, out, None, *args)
        sync()
        want.append(out)
    outs = [[torch.zeros_like(x) for _ in range(20)] for x in qs]
    sync()
    for k in range(20):
        for c, x, o in zip(caches, qs, outs):
            c.attention(x, o[k], None, *args)
    sync()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)


# -------------------------------------------------------------- refusals of the library

def test_refusals_of_the_library(lib):
    L, acc, rope, pages = lib
    from llamahat import _lib
    x, pos = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (dict(theta=1.0), dict(scaling="linear", factor=0.5), dict(rot_dim=3), dict(rot_dim=66),
                dict(scaling="llama3", factor=8.0, low_freq_factor=4.0), dict(scaling="llama3", original_max_pos=0),
                dict(scaling="yarn", factor=4.0, beta_fast=1.0), dict(theta=float("nan")), dict(theta=float("inf"))):
        with pytest.raises(L.IllegalArgumentError):
            rope.apply_scaled(x, x, pos, L.RopeConfig(**bad))
    with pytest.raises(L.IllegalArgumentError):
        rope.apply_scaled(torch.zeros(4, 1, 514, device="cuda"), torch.zeros(4, 1, 514, device="cuda"), pos, L.RopeConfig(head_dim=514))
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    with pytest.raises(L.LlamaCudaError) as e:
        pages.step(i32(2), i32(2), i32(2, 3), i32(4), i32(1), 24, i32(2), i32(3), i32(5), i32(5), i32(5), i32(1), i32(2))
    assert e.value.code == _lib.LC_ERR_UNSUPPORTED
    with pytest.raises(L.IllegalArgumentError):
        pages.step(i32(4097), i32(4097), i32(4097, 1), i32(4), i32(1), 16, i32(4097), i32(4098), i32(5), i32(5), i32(5), i32(1), i32(2))

    def pool(n=4, kv=2, page=32, d=64, **kw):
        c = lambda: torch.zeros(n, kv, page, d, dtype=torch.uint8, device="cuda")  # noqa: E731
        return L.PagedKV8(c(), c(), torch.zeros(n, kv, device="cuda"), torch.zeros(n, kv, device="cuda"), acc=acc, **kw)

    q, out, table, lens = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 2, 64, device="cuda"), i32(1, 4), i32(1)
    for cache in (pool(page=24), pool(page=256)):
        with pytest.raises(L.LlamaCudaError) as e:
            cache.attention(q, out, None, lens, table)
        assert e.value.code == _lib.LC_ERR_UNSUPPORTED
    with pytest.raises(L.LlamaCudaError):
        pool(d=96).attention(torch.zeros(1, 2, 96, device="cuda"), torch.zeros(1, 2, 96, device="cuda"), None, lens, table)
    cache = pool()
    for kw in (dict(max_q=0), dict(max_q=2), dict(scale=0.0), dict(scale=float("nan")), dict(scale=-1.0)):
        with pytest.raises(L.IllegalArgumentError):
            cache.attention(q, out, None, lens, table, **kw)
    with pytest.raises(L.IllegalArgumentError):  # 3 query heads over 2 kv heads
        cache.attention(torch.zeros(1, 3, 64, device="cuda"), torch.zeros(1, 3, 64, device="cuda"), None, lens, table)
    with pytest.raises(L.IllegalArgumentError):  # without q_start, a row for every sequence
        cache.attention(torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda"), None, lens, table)
    with pytest.raises(L.LlamaCudaError, match="2\\^32 steps"):  # 4096 rows one by one over 2^26 positions
        cache.attention(torch.zeros(4096, 2, 64, device="cuda"), torch.zeros(4096, 2, 64, device="cuda"), i32(2), lens,
                        torch.zeros(1, 1 << 21, dtype=torch.int32, device="cuda"), max_q=1)
    # counts that 32-bit steps would pass: no buffer is looked at
    many, raw, ctx, config = 2 ** 31 - 16, _lib.load(), acc.handle, _lib.LcRopeConfig()
    raw.lc_rope_config_llama32(ctypes.byref(config))
    at = x.data_ptr()
    assert raw.lc_rope_apply(ctx, ctypes.byref(config), at, at, at, many, 1, 64, 64, 0, 0) == _lib.LC_ERR_UNSUPPORTED
    assert raw.lc_rope_apply(ctx, ctypes.byref(config), at, at, at, 1, 2 ** 26, 64, 64, 0, 0) == _lib.LC_ERR_UNSUPPORTED
    assert raw.lc_pages_step(ctx, at, at, 1, 16, at, 1, at, at, 1, many, *[at] * 7) == _lib.LC_ERR_UNSUPPORTED
    kv = _lib.LcKv8(k=at, v=at, k_scale=at, v_scale=at, n_pages=1, page_size=16, n_kv_heads=1, head_dim=64, format=0)
    assert raw.lc_kv8_append(ctx, ctypes.byref(kv), at, at, 64, 0, at, many) == _lib.LC_ERR_UNSUPPORTED
    assert raw.lc_kv8_read(ctx, ctypes.byref(kv), at, at, 64, 0, at, many) == _lib.LC_ERR_UNSUPPORTED
    kv.n_kv_heads = 32768
    assert raw.lc_kv8_read(ctx, ctypes.byref(kv), at, at, 64, 0, at, 1) == _lib.LC_ERR_UNSUPPORTED
    host = L.PagedKV8(torch.zeros(4, 2, 32, 64, dtype=torch.uint8), torch.zeros(4, 2, 32, 64, dtype=torch.uint8),
                      torch.zeros(4, 2), torch.zeros(4, 2), acc=acc)
    with pytest.raises(L.IllegalArgumentError, match="device memory"):
        host.attention(q, out, None, lens, table)
    # nothing to do is no error
    cache.append(torch.zeros(0, 2, 64, device="cuda"), torch.zeros(0, 2, 64, device="cuda"), i32(0))
    cache.attention(torch.zeros(0, 2, 64, device="cuda"), torch.zeros(0, 2, 64, device="cuda"), i32(2), lens, table)
    # the context stays usable
    cache.attention(q, out, None, lens, table)
    sync()
    assert not out.any()
