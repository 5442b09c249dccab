"""Log probabilities at the ends of what `scale` and the logits may be."""
import numpy as np
import pytest

from test_logprobs_gpu import LOWEST, check

import w4_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def lp():
    import llamahat
    return llamahat.CudaKernelFactory().createLogProbs(llamahat.Accelerator(0))


def rows(rng, vocab, kind, size):
    """Logits of the given size: ordinary ones, a few values, masked ones, all but one masked, both ends."""
    x = rng.standard_normal((7, vocab)) * size
    x[1] = rng.integers(-2, 3, vocab) * size
    x[2] = np.where(rng.random(vocab) < 0.9, -np.inf, x[2])
    x[3] = np.where(rng.random(vocab) < 0.9, LOWEST[kind], x[3])
    x[4] = -np.inf
    x[4, vocab // 2] = size
    x[5] = LOWEST[kind]
    x[5, vocab // 3:] = -LOWEST[kind]
    x[6] = -np.abs(x[6])
    x[6, 1] = 0.0
    with np.errstate(over="ignore"):
        return x.astype(ref.NP[kind])


# Scales next to sizes of logits at which their products matter, and ordinary ones.
EXTREMES = [(1e38, 1e-38), (1e38, 1e-35), (1e38, 1e-41), (3.4e38, 1e-38), (3.4e38, 1e-45), (3.4e38, 1.0), (1e30, 1e-30), (2e30, 1e-30),
            (1e29, 1e-29), (1e25, 1.0), (1e38, 1e30), (1e-30, 1e30), (1e-31, 1e31), (1e-37, 1e38), (1e-38, 1e38), (1e-38, 1e30),
            (1e-40, 1e38), (1e-45, 1e38), (1e-45, 1.0), (0.5, 1e38), (1.0, 3e37)]


@pytest.mark.parametrize("scale,size", EXTREMES)
@pytest.mark.parametrize("vocab", [50, 3001, 70000])
def test_extreme_scales(lp, vocab, scale, size):
    rng = np.random.default_rng(vocab)
    x = rows(rng, vocab, "f32", size)
    check(lp, x, [0, 1, vocab // 3, 3, vocab // 2, 5, 1], 9, scale=scale, pad=1)
    check(lp, x, rng.integers(0, vocab, 7), 0, scale=scale)
    if 1e-7 < size < 1e5:
        check(lp, rows(rng, vocab, "f16", size), rng.integers(0, vocab, 7), 9, scale=scale)


def test_close_logits_under_a_large_scale(lp):
    """ln p of {0, -1e-35} under 1e38 is {0, -1000}, not {-ln 2, -ln 2 - 1000}."""
    x = np.array([[0.0, -1e-35]], np.float32)
    check(lp, x, [0], 2, scale=1e38)
    check(lp, x, [1], 2, scale=1e38)


def test_far_logits_under_a_small_scale(lp):
    """ln p of {3e38, -3e38} under 1e-38 is what {6, 0} have: their difference is no fp32 number."""
    x = np.array([[3e38, -3e38, 1e38]], np.float32)
    check(lp, x, [1], 3, scale=1e-38)
    check(lp, x, [1], 3, scale=0.5)  # ln p -3e38


def test_one_row_of_logits_for_all_tokens(lp):
    """Logits at stride 0: the same row for every token."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal(5003).astype(np.float32) * 3
    held, tokens = torch.from_numpy(x).cuda(), torch.arange(0, 5000, 50, dtype=torch.int32).cuda()
    out, ranks = torch.zeros(100, device="cuda"), torch.zeros(100, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    lp.apply(held[None].expand(100, 5003), tokens, out, ranks)
    lp.acc.synchronize()
    p, _, mean = ref.logprobs(x, 1.0)
    at = tokens.cpu().numpy()
    assert np.all(np.abs(out.cpu().numpy() - p[at]) <= ref.logprobs_bound(p - p.max(), mean, 5003)[at])
    place = np.empty(5003, np.int64)
    place[ref.order(x)] = np.arange(5003)
    np.testing.assert_array_equal(ranks.cpu().numpy(), place[at])
