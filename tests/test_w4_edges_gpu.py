"""4-bit weights where the first tests do not go: stages of operands that are used
again and again, the kernel of large F16 prompts in all its forms, few rows with
more than one meeting, codes at the zero point, very wide matrices."""
import numpy as np
import pytest

import w4_ref as ref

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def L():
    import llamahat
    return llamahat


@pytest.fixture(scope="module")
def acc(L):
    return L.Accelerator(0)


def dev(x):
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    torch.cuda.synchronize()
    return t


def host(acc, t):
    acc.synchronize()
    return t.cpu().numpy()


def matrix(rng, rows, cols, group, zeros):
    groups = -(-cols // group)
    code = rng.integers(0, 16, (rows, cols), np.uint8)
    scale = (0.002 * np.exp(rng.standard_normal((rows, groups)))).astype(np.float16)
    return code, scale, rng.integers(0, 16, (rows, groups), np.uint8) if zeros else None


def packed(L, acc, code, scale, zero, group):
    w = L.Weights4.empty(*code.shape, group, zeros=zero is not None, acc=acc)
    torch.cuda.synchronize()
    w.pack(ref.two_to_a_byte(code), scale, zero)
    return w


def check(got, x, code, scale, zero, group, kind, residual=None):
    want, terms, far = ref.product(x, code, scale, zero, group, residual)
    off = np.abs(got.astype(np.float64) - want) - ref.product_bound(want, terms, far, scale.shape[1], kind)
    assert np.all(off <= 0), f"{off.max():g} past the bound at {np.unravel_index(off.argmax(), off.shape)}"


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols,batch", [(300, 16384, 64), (6000, 4096, 33), (40, 10000, 20)])
def test_stages_used_again(L, acc, rows, cols, batch, kind):
    """Tens of blocks through two stages of operands in tensor memory: the same bits
    in every one of many calls, and within the bound."""
    rng = np.random.default_rng(rows)
    code, scale, zero = matrix(rng, rows, cols, 64, True)
    x = rng.standard_normal((batch, cols)).astype(ref.NP[kind])
    w, dx = packed(L, acc, code, scale, zero, 64), dev(x)
    ys = [torch.full((batch, rows), float("nan"), dtype=dx.dtype, device="cuda") for _ in range(20)]
    torch.cuda.synchronize()
    for y in ys:
        w.apply(dx, y)
    first = host(acc, ys[0])
    check(first, x, code, scale, zero, 64, kind)
    for y in ys[1:]:
        np.testing.assert_array_equal(y.cpu().numpy(), first)


def test_widest_rows(L, acc):
    """So many columns that the bytes of a CTA's part pass 32 bits before it is cut into
    phases.  Whole numbers at columns here and there: the sums are exact."""
    cols = 958682 * 8 * 128 - 77
    rng = np.random.default_rng(1)
    at = np.unique(np.concatenate([rng.integers(0, cols // 64, 5000) * 64 + rng.integers(1, 50, 5000), [cols - 1]]))
    code, x = rng.integers(-6, 7, (2, len(at))), rng.integers(-8, 9, len(at)) / 4.0
    w = L.Weights4.empty(2, cols, 64, acc=acc)
    v = torch.zeros(2, cols, dtype=torch.float16, device="cuda")
    v[0, ::64], v[1, ::64] = 7.0, -7.0  # a scale of 1 for every group
    v[:, torch.from_numpy(at).cuda()] = torch.from_numpy(code).half().cuda()
    torch.cuda.synchronize()
    w.quantize(v)
    acc.synchronize()
    del v
    held = torch.zeros(1, cols, device="cuda")
    held[0, torch.from_numpy(at).cuda()] = torch.from_numpy(x).float().cuda()
    y = torch.full((8, 2), float("nan"), device="cuda")
    torch.cuda.synchronize()
    w.apply(held.expand(8, cols), y)
    got = host(acc, y)
    del w, held
    torch.cuda.empty_cache()
    np.testing.assert_array_equal(got, np.repeat((code @ x)[None], 8, 0))
