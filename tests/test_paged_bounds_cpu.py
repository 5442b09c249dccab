"""The bounds of the long-sum tests notice what they are there for: the same
mistakes, planted in a plain computation."""
import numpy as np
import pytest

from paged_bounds import sums_bound


def weights_and_values(n, rows=64, d=64):
    """Nearly even weights 2^x and values of one sign, as the tests on the GPU have them."""
    rng = np.random.default_rng(n)
    p = np.exp2(0.1 * rng.standard_normal((rows, n)) + 5.0)
    v = rng.integers(1, 128, (n, d)).astype(np.float64) * (0.02 * np.exp(0.4 * rng.standard_normal((n, 1))))
    return p, v


def down(x):
    """fp32 numbers toward zero (of positive ones)."""
    y = x.astype(np.float32)
    return np.where(y.astype(np.float64) > x, np.nextafter(y, np.float32(0)), y).astype(np.float64)


def nearest(x):
    return x.astype(np.float32).astype(np.float64)


def summed(p, v, add, flush=None):
    """Products of 16 tokens at a time, added one by one to a running sum, and
    that after `flush` of them to one in round-to-nearest."""
    total, run = 0.0, 0.0
    for k in range(0, p.shape[1], 16):
        run = add(run + p[:, k:k + 16] @ v[k:k + 16])
        if flush and (k // 16 + 1) % flush == 0:
            total, run = nearest(total + run), 0.0
    return total + run


@pytest.mark.parametrize("n,chain", [(65536, 0), (65536, 32), (65536, 64)])
def test_a_bound_notices_sums_that_lose_toward_zero(n, chain):
    p, v = weights_and_values(n, rows=8)
    norm = p.sum(1)[:, None]
    want = p @ v / norm
    # scores of the size that the tests have: sum |q k| scale below 1
    bound = sums_bound(1.0, want, n, 64, chain)
    assert (np.abs(summed(p, v, down) / norm - want) > bound).any(1).all()
    assert (np.abs(summed(p, v, nearest) / norm - want) <= bound).all()
    if chain:
        assert (np.abs(summed(p, v, down, flush=chain) / norm - want) <= bound).all()


@pytest.mark.parametrize("chain", [0, 32])
def test_a_bound_notices_weights_of_one_half(chain):
    p, v = weights_and_values(200)
    half = p.astype(np.float16).astype(np.float64)
    norm = p.sum(1)[:, None]
    want = p @ v / norm
    assert (np.abs(half @ v / norm - want) > sums_bound(1.0, want, 200, 64, chain)).any()
    lo = (p - half).astype(np.float16).astype(np.float64)
    assert (np.abs((half + lo) @ v / norm - want) <= sums_bound(1.0, want, 200, 64, chain)).all()
