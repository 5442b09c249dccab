"""Log probabilities, ranks, entropy and alternatives against 64-bit references."""
import numpy as np
import pytest

import w4_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
LOWEST = {"f32": np.finfo(np.float32).min, "f16": np.finfo(np.float16).min}


@pytest.fixture(scope="module")
def L():
    import llamahat
    return llamahat


@pytest.fixture(scope="module")
def acc(L):
    return L.Accelerator(0)


@pytest.fixture(scope="module")
def lp(L, acc):
    return L.CudaKernelFactory().createLogProbs(acc)


def padded(x, pad):
    held = torch.full((x.shape[0], x.shape[1] + pad), float("inf"), dtype=torch.from_numpy(x[:1]).dtype, device="cuda")
    held[:, :x.shape[1]] = torch.from_numpy(x).cuda()
    return held[:, :x.shape[1]]


def run(lp, x, tokens, top, scale=1.0, pad=0):
    """Outputs as numpy arrays, from device memory that holds something else before the call."""
    n = len(x)
    d = padded(x, pad)
    out = [torch.full((n,), 7.0, device="cuda"), torch.full((n,), 7, dtype=torch.int32, device="cuda"),
           torch.full((n,), 7.0, device="cuda"), torch.full((n, top), 7, dtype=torch.int32, device="cuda") if top else None,
           torch.full((n, top), 7.0, device="cuda") if top else None]
    t = torch.from_numpy(np.asarray(tokens, np.int32)).cuda()
    torch.cuda.synchronize()
    lp.apply(d, t, *out, scale=scale)
    lp.acc.synchronize()
    return [None if o is None else o.cpu().numpy() for o in out]


def check(lp, x, tokens, top, scale=1.0, pad=0):
    mine, rank, entropy, ids, best = run(lp, x, tokens, top, scale, pad)
    scale = float(np.float32(scale))
    vocab = x.shape[1]
    for i in range(len(x)):
        p, h, mean = ref.logprobs(x[i], scale)
        order = ref.order(x[i])
        with np.errstate(invalid="ignore"):
            t = p - p.max()
        bound = np.where(np.isfinite(p), ref.logprobs_bound(np.where(np.isfinite(t), t, 0.0), mean, vocab), 0.0)

        def same(got, want, b, what):
            with np.errstate(over="ignore"):
                want32 = np.float32(want)
            if not np.isfinite(want32):
                assert np.array_equal(got, want32, equal_nan=True), f"row {i}: {what} {got}, not {want32}"
            else:
                assert abs(got - want) <= b, f"row {i}: {what} {got}, not {want} within {b:g}"
        if 0 <= tokens[i] < vocab:
            assert rank[i] == np.nonzero(order == tokens[i])[0][0], f"row {i}: rank"
            same(mine[i], p[tokens[i]], bound[tokens[i]], "ln p")
        else:
            assert rank[i] == -1 and mine[i] == 0.0
        same(entropy[i], h, 4 * (1 + mean) * ref.logprobs_bound(0.0, mean, vocab), "entropy")
        if top:
            k = min(top, vocab)
            np.testing.assert_array_equal(ids[i, :k], order[:k], err_msg=f"row {i}")
            for j in range(k):
                same(best[i, j], p[order[j]], bound[order[j]], f"alternative {j}")
            bad = np.isnan(h)
            assert (ids[i, k:] == -1).all() and (np.isnan(best[i, k:]).all() if bad else (best[i, k:] == -np.inf).all())


def logits(rng, rows, vocab, kind):
    x = rng.standard_normal((rows, vocab)) * rng.uniform(0.5, 4.0, (rows, 1))
    x[np.arange(rows), rng.integers(0, vocab, rows)] += rng.uniform(0, 16, rows)
    return x.astype(ref.NP[kind])


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("top", [0, 1, 5, 20, 32])
def test_sizes(lp, top, kind):
    rng = np.random.default_rng(top)
    for vocab in (1, 2, 3, 7, 8, 9, 31, 32, 33, 100, 255, 257, 1000, 2048, 4099, 16384, 32003):
        rows = 3
        check(lp, logits(rng, rows, vocab, kind), rng.integers(0, vocab, rows), top, scale=0.7, pad=vocab % 3)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows,vocab", [(1, 128256), (2, 128256), (5, 100003), (19, 50021), (64, 8192), (150, 1001), (300, 4096),
                                        (700, 515), (500, 9001)])
def test_rows(lp, rows, vocab, kind):
    rng = np.random.default_rng(rows)
    check(lp, logits(rng, rows, vocab, kind), rng.integers(-1, vocab, rows), 20, scale=1.25, pad=rows % 2)
    check(lp, logits(rng, rows, vocab, kind), rng.integers(-1, vocab + 1, rows), 0)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [40, 1000, 40000])
def test_hard_rows(lp, vocab, kind):
    """Masked rows, equal logits, sorted ones, zeros of both signs, NaN and infinities."""
    rng = np.random.default_rng(vocab)
    low = LOWEST[kind]
    x = logits(rng, 24, vocab, kind).astype(np.float64)
    gone = rng.random((24, vocab)) < 0.95
    x[0] = np.where(gone[0], -np.inf, x[0])
    x[1] = np.where(gone[1], low, x[1])
    x[2] = -np.inf
    x[3] = low
    x[4] = -np.inf
    x[4, vocab // 2] = 3.0                 # one allowed token
    x[5] = low
    x[5, vocab - 1] = -5.0
    x[6] = 1.5                             # all equal
    x[7] = np.arange(vocab) / 64.0         # ascending
    x[8] = -np.arange(vocab) / 64.0        # descending
    x[9] = rng.integers(0, 3, vocab)       # many equal ones
    x[10] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    x[11, 5] = np.nan
    x[12, 7] = np.inf
    x[13] = np.nan
    x[14, ::2] = -np.inf
    x[14, 3] = np.nan
    x[15] = -np.finfo(ref.NP[kind]).max / 2
    x[16] = 0.0
    x[16, 9] = 40.0                        # a sure row
    x[17] = np.where(np.arange(vocab) < 3, -np.inf, low)
    x[18, :] = -60000.0
    x[18, 1] = 60000.0
    x[19] = -np.inf
    x[19, 0] = low
    x[20] = np.inf
    x[21, 0] = -np.inf
    with np.errstate(over="ignore"):
        x = x.astype(ref.NP[kind])
    tokens = rng.integers(0, vocab, 24)
    tokens[4], tokens[16], tokens[22], tokens[23] = vocab // 2, 9, -5, vocab + 3
    tokens[11], tokens[13], tokens[10] = 5, 1, 2
    check(lp, x, tokens, 32)
    check(lp, x, tokens, 3, scale=0.5)
    check(lp, x[::-1].copy(), tokens[::-1].copy(), 0, scale=2.0)


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_few_allowed(lp, kind):
    """A grammar: a handful of allowed tokens, next to each other or far apart, or a
    few threads that have all the large ones."""
    rng = np.random.default_rng(8)
    vocab = 50000
    for low in (-np.inf, LOWEST[kind]):
        x = np.full((6, vocab), low)
        x[0, rng.integers(0, vocab, 13)] = rng.standard_normal(13)
        x[1, 777:790] = rng.standard_normal(13)
        x[2, 20000:21000] = rng.standard_normal(1000)
        x[3, ::1024] = rng.standard_normal(len(x[3, ::1024]))
        x[4, :40] = np.arange(40)
        x[5] = rng.standard_normal(vocab)
        x[5, 3000:3400] += 50.0  # all of the best in a few threads
        x = x.astype(ref.NP[kind])
        tokens = x.argmax(1)
        check(lp, x, tokens, 5)
        check(lp, x, rng.integers(0, vocab, 6), 32)
    # Large ones at the stride at which a thread reads: hundreds in one thread.
    n = 16 // np.dtype(ref.NP[kind]).itemsize
    x = rng.standard_normal((1, 256 * n * 120)) * 0.01
    for e in range(n):
        x[0, 5 * n + e::256 * n] += 10.0
    x = np.repeat(x, 400, 0).astype(ref.NP[kind])  # one CTA per row
    x[:, 0] += np.arange(400) % 3
    got = run(lp, x, np.zeros(400), 32)
    check(lp, x[:3], [0, 5 * n, 7], 32)
    for i in range(0, 400, 57):
        np.testing.assert_array_equal(got[3][i], ref.order(x[i])[:32])


@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_many_short_rows(lp, kind):
    """More rows than are resident: the hard ones of them in the CTAs of short rows."""
    rng = np.random.default_rng(18)
    x = logits(rng, 460, 6007, kind)
    x[3], x[7], x[11] = -np.inf, LOWEST[kind], 2.0
    x[20, rng.random(6007) < 0.999] = -np.inf
    x[30] = np.arange(6007) / 16.0
    x[40, 9] = np.nan
    x[50, ::7] = np.inf
    x[60, ::8] += 30.0
    check(lp, x, rng.integers(-1, 6007, 460), 32)
    check(lp, x, rng.integers(-1, 6007, 460), 0, pad=1)


def test_asked_outputs_alone(L, lp):
    """Each output by itself has the same bits as all together; host memory too."""
    rng = np.random.default_rng(2)
    x, tokens = logits(rng, 9, 3001, "f32"), rng.integers(0, 3001, 9).astype(np.int32)
    mine, rank, entropy, ids, best = run(lp, x, tokens, 7, 0.9)
    for name, whole in (("token_logprobs", mine), ("token_ranks", rank), ("entropy", entropy), ("top_ids", ids), ("top_logprobs", best)):
        alone = np.zeros_like(whole)
        lp.apply(x, tokens, **{name: alone}, scale=0.9)
        np.testing.assert_array_equal(alone, whole, err_msg=name)
    alone = np.zeros_like(best)
    lp.apply(x, top_logprobs=alone, scale=0.9)
    np.testing.assert_array_equal(alone, best)
    lp.apply(x[:0], entropy=np.zeros(0, np.float32))


def test_captured(L, acc, lp):
    rng = np.random.default_rng(3)
    st, graph = torch.cuda.ExternalStream(acc.stream), torch.cuda.CUDAGraph()
    x = torch.from_numpy(logits(rng, 2, 60000, "f32")).cuda()
    h, ids = torch.zeros(2, device="cuda"), torch.zeros(2, 9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        lp.apply(x, entropy=h, top_ids=ids)
    for _ in range(2):
        z = logits(rng, 2, 60000, "f32")
        x.copy_(torch.from_numpy(z))
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        acc.synchronize()
        for i in range(2):
            assert ids[i].tolist() == ref.order(z[i])[:9].tolist()
            p, want, mean = ref.logprobs(z[i], 1.0)
            assert abs(h[i].item() - want) <= 4 * (1 + mean) * ref.logprobs_bound(0.0, mean, 60000)


def test_refusals(L, acc, lp):
    x, t = torch.zeros(2, 50, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    out = torch.zeros(2, device="cuda")
    torch.cuda.synchronize()

    def call(vocab=50, scale=1.0, tokens=t.data_ptr(), lps=out.data_ptr(), k=0, ids=None, dtype=0, rows=2, stride=50):
        L._lib.check(lp.lib.lc_logprobs(acc.handle, x.data_ptr(), stride, dtype, rows, vocab, scale, tokens, lps, None, None, k, ids, None))
    for wrong in (dict(vocab=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")),
                  dict(tokens=None), dict(k=33), dict(k=-1), dict(ids=t.data_ptr()), dict(dtype=2), dict(rows=-1), dict(stride=-1)):
        with pytest.raises(L.IllegalArgumentError):
            call(**wrong)
    with pytest.raises(L.IllegalArgumentError):
        L._lib.check(lp.lib.lc_logprobs(acc.handle, None, 50, 0, 2, 50, 1.0, None, None, None, out.data_ptr(), 0, None, None))
    call()
    acc.synchronize()
