"""Host checks of the 4-bit weights and the log probabilities (no device):
sizes, refusals before anything is called, and the references themselves."""
import ctypes

import numpy as np
import pytest

import w4_ref as ref

torch = pytest.importorskip("torch")


class NoDevice:
    """Stands where an Accelerator stands; every call through it is refused."""
    handle = None
    device = 0


@pytest.fixture(scope="module")
def L():
    import llamahat
    return llamahat


def weights(L, rows=48, cols=300, group=64, zeros=True, **kw):
    n, m = L.Weights4.sizes(rows, cols, group)
    a = {"codes": torch.zeros(n, dtype=torch.uint8), "scales": torch.zeros(m, dtype=torch.float16),
         "zeros": zeros if torch.is_tensor(zeros) else torch.zeros(m, dtype=torch.uint8) if zeros else None} | kw
    return L.Weights4(a["codes"], a["scales"], a["zeros"], rows, cols, group, acc=NoDevice())


def test_sizes(L):
    assert L.Weights4.sizes(16, 128, 128) == (1024, 16)
    assert L.Weights4.sizes(17, 129, 32) == (4 * 1024, 4 * 64)
    assert L.Weights4.sizes(1, 1, 64) == (1024, 32)
    assert L.Weights4.sizes(128256, 2048, 64) == (128256 * 2048 // 2, 128256 * 32)
    for bad in ((0, 5, 32), (5, 0, 32), (-1, 5, 32), (5, 5, 48), (5, 5, 0), (2 ** 31 - 1, 5, 32)):
        with pytest.raises(L.LlamaCudaError):
            L.Weights4.sizes(*bad)


def test_null_context_is_refused(L):
    from llamahat import _lib
    lib, w = _lib.load(), _lib.LcW4()
    assert lib.lc_w4_quantize(None, w, None, 1, 0) == _lib.LC_ERR_INVALID_ARG
    assert lib.lc_w4_pack(None, w, None, None, None) == _lib.LC_ERR_INVALID_ARG
    assert lib.lc_w4_read(None, w, None, 1, 0) == _lib.LC_ERR_INVALID_ARG
    assert lib.lc_w4_product(None, w, None, 1, None, 1, None, 0, 1, 0) == _lib.LC_ERR_INVALID_ARG
    assert lib.lc_logprobs(None, None, 1, 0, 1, 1, 1.0, None, None, None, None, 0, None, None) == _lib.LC_ERR_INVALID_ARG
    assert "context is NULL" in _lib.last_error()


def test_python_refusals(L):
    with pytest.raises(TypeError):
        weights(L, codes=torch.zeros(1 << 20))
    with pytest.raises(ValueError):
        weights(L, codes=torch.zeros(5, dtype=torch.uint8))
    with pytest.raises(ValueError):
        weights(L, zeros=torch.zeros(3, dtype=torch.uint8))
    with pytest.raises(TypeError):
        weights(L, scales=torch.zeros(1 << 16))
    w = weights(L)
    f = lambda *s, **k: torch.zeros(*s, **k)  # noqa: E731
    half = dict(dtype=torch.float16)
    for call in (lambda: w.apply(f(2, 299), f(2, 48)), lambda: w.apply(f(2, 300), f(2, 47)), lambda: w.apply(f(2, 300), f(3, 48)),
                 lambda: w.apply(f(2, 300), f(2, 48, **half)), lambda: w.apply(f(2, 300), f(2, 48), residual=f(2, 47)),
                 lambda: w.apply(f(2, 300), f(2, 48), residual=f(2, 48, **half)), lambda: w.apply(f(300), f(48)),
                 lambda: w.quantize(f(48, 301)), lambda: w.read(f(47, 300)), lambda: w.apply(f(300, 2).t(), f(2, 48)),
                 lambda: w.pack(f(48, 150, dtype=torch.uint8), f(48, 5, **half)),
                 lambda: w.pack(f(48, 149, dtype=torch.uint8), f(48, 5, **half), f(48, 5, dtype=torch.uint8)),
                 lambda: w.apply(f(2, 300), f(1, 48).expand(2, 48))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: w.apply(f(2, 300, dtype=torch.float64), f(2, 48)), lambda: w.quantize(f(48, 300, dtype=torch.bfloat16)),
                 lambda: w.pack(f(48, 150), f(48, 5, **half), f(48, 5, dtype=torch.uint8))):
        with pytest.raises(TypeError):
            call()
    lp = L.CudaLogProbs(NoDevice())
    with pytest.raises(ValueError):
        lp.apply(f(2, 50), top_ids=f(2, 3, dtype=torch.int32), top_logprobs=f(2, 4))
    with pytest.raises(ValueError):
        lp.apply(f(2, 50), f(1, dtype=torch.int32), f(2))
    with pytest.raises(TypeError):
        lp.apply(f(2, 50), f(2, dtype=torch.int64), f(2))
    with pytest.raises(TypeError):
        lp.apply(f(2, 50), entropy=f(2, **half))
    with pytest.raises(ValueError):
        lp.apply(f(2, 50), entropy=f(1))
    with pytest.raises(L.IllegalArgumentError):  # in order, but there is no device
        lp.apply(f(2, 50), entropy=f(2))


def test_quantize_reference():
    x = np.array([[7.0, -7.0, 3.5, 2.5, -2.5, 0.0, 1.4999]], np.float32)
    code, scale, zero = ref.quantize(x, 32, False)
    assert zero is None and scale[0, 0] == 1.0
    assert code[0].tolist() == [15, 1, 12, 10, 6, 8, 9]  # ties to even
    x = np.array([[-2.0, 5.5, 5.5, 0.25]], np.float32)
    code, scale, zero = ref.quantize(x, 32, True)
    assert scale[0, 0] == 0.5 and zero[0, 0] == 4 and code[0].tolist() == [0, 15, 15, 4]
    assert ref.values(code, scale, zero, 32)[0].tolist() == [-2.0, 5.5, 5.5, 0.0]
    code, scale, zero = ref.quantize(np.full((1, 5), np.nan, np.float32), 32, False)
    assert scale[0, 0] == 0 and (code == 8).all()


def test_product_bound_notices():
    """A scale taken from the neighbouring group, a lost column, a zero point of
    7: the bound is far below what any of them does."""
    rng = np.random.default_rng(1)
    code, scale = rng.integers(0, 16, (20, 256), np.uint8), (0.002 * np.exp(rng.standard_normal((20, 4)))).astype(np.float16)
    x = rng.standard_normal((3, 256))
    y, terms, far = ref.product(x, code, scale, None, 64)
    bound = ref.product_bound(y, terms, far, 4, "f32")
    shifted = ref.product(x, code, np.roll(scale, 1, 1), None, 64)[0]
    less = ref.product(np.where(np.arange(256) == 77, 0.0, x), code, scale, None, 64)[0]
    seven = ref.product(x, code, scale, np.full((20, 4), 7, np.uint8), 64)[0]
    for wrong in (shifted, less, seven):
        assert (np.abs(wrong - y) > bound).mean() > 0.9


def test_logprobs_reference():
    p, h, mean = ref.logprobs(np.log(np.array([0.5, 0.25, 0.125, 0.125])), 1.0)
    np.testing.assert_allclose(np.exp(p), [0.5, 0.25, 0.125, 0.125])
    np.testing.assert_allclose(h, 1.75 * np.log(2))
    p, h, _ = ref.logprobs(np.full(4, -np.inf), 1.0)
    assert (p == -np.inf).all() and h == 0.0
    assert ref.order(np.array([1.0, 3.0, np.nan, 3.0, -np.inf])).tolist() == [1, 3, 0, 2, 4]


def test_factory_and_struct(L):
    from llamahat import _lib
    assert ctypes.sizeof(_lib.LcW4) == 48
    assert hasattr(L.CudaKernelFactory(), "createLogProbs")
