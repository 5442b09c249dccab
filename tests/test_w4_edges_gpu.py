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


def near_zero_points(rng, rows, cols, group, zeros):
    """Codes at the zero point but for one in fifty, a step beside it; a scale of its
    own for every group.  Row 0 and a third of the others: at the zero point throughout."""
    groups = -(-cols // group)
    zero = rng.integers(8, 16, (rows, groups), np.uint8) if zeros else None
    z = np.repeat(zero, group, 1)[:, :cols] if zeros else np.full((rows, cols), 8, np.uint8)
    code = np.where(rng.random((rows, cols)) < 0.02, z - 1, z).astype(np.uint8)
    code[::3] = z[::3]
    return code, (rng.uniform(0.5, 2.0, (rows, groups))).astype(np.float16), zero


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("batch", [1, 4, 8, 12, 40, 300])
def test_codes_at_the_zero_point(L, acc, batch, zeros, kind):
    """A weight of 0 is 0: rows of W that hold nothing else give the residual itself,
    and errors go by the sizes of (c - z) x.  The bound is that of w4_ref with these as
    the terms: 2^-22 of an fp32 element of x and 2^-39 of the row's largest, up to nine
    additions of an instruction for each group, one rounding per group, scale and join."""
    for rows, cols, group in [(64, 512, 32), (50, 2048, 64), (3, 4096, 128), (130, 1000, 128)]:
        rng = np.random.default_rng(rows + batch)
        code, scale, zero = near_zero_points(rng, rows, cols, group, zeros)
        x = (rng.standard_normal((batch, cols)) + 3.0).astype(ref.NP[kind])
        r = rng.standard_normal((batch, rows)).astype(ref.NP[kind])
        w = packed(L, acc, code, scale, zero, group)
        y, dx, dr = dev(np.full((batch, rows), np.nan, ref.NP[kind])), dev(x), dev(r)
        w.apply(dx, y, residual=dr)
        got = host(acc, y)
        np.testing.assert_array_equal(got[:, ::3], r[:, ::3])
        size = np.abs(ref.values(code, scale, zero, group))
        want = x.astype(np.float64) @ ref.values(code, scale, zero, group).T + r
        terms = np.abs(x.astype(np.float64)) @ size.T + np.abs(r)
        far = np.abs(x.astype(np.float64)).max(1, keepdims=True) * size.sum(1)[None]
        bound = ref.product_bound(want, terms, far, scale.shape[1], kind)
        assert np.all(np.abs(got - want) <= bound), f"{rows} x {cols}, groups of {group}"


def product(L, acc, rng, rows, cols, batch, group, zeros, kind, residual=False):
    code, scale, zero = matrix(rng, rows, cols, group, zeros)
    x = (rng.standard_normal((batch, cols)) * np.exp(rng.standard_normal(cols))).astype(ref.NP[kind])
    r = rng.standard_normal((batch, rows)).astype(ref.NP[kind]) if residual else None
    w, y, dx = packed(L, acc, code, scale, zero, group), dev(np.full((batch, rows), np.nan, ref.NP[kind])), dev(x)
    w.apply(dx, y, residual=None if r is None else dev(r))
    check(host(acc, y), x, code, scale, zero, group, kind, r)


@pytest.mark.parametrize("group", [64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,cols,batch", [(300, 1111, 257),    # ragged units and blocks
                                             (257, 4096, 300),    # few units: the columns over a cluster
                                             (31, 8200, 513),
                                             (9001, 320, 700),    # several units of a CTA
                                             (256, 128, 2049),    # one block
                                             (1, 1, 300)])
def test_large_half_prompts(L, acc, rows, cols, batch, zeros, group):
    """More than 256 F16 rows without a residual: units of 128 rows, operands in shared memory."""
    product(L, acc, np.random.default_rng(cols), rows, cols, batch, group, zeros, "f16")


@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, True), (128, True)])
def test_other_prompts(L, acc, group, zeros):
    """The same rows in units of 64: fine groups, a residual, F32."""
    rng = np.random.default_rng(group)
    for rows, cols, batch in [(300, 1111, 257), (257, 4096, 300), (9001, 320, 400)]:
        product(L, acc, rng, rows, cols, batch, group, zeros, "f16", residual=group > 32)
        product(L, acc, rng, rows, cols, batch, group, zeros, "f32")


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("rows,cols,batch", [(40000, 300, 5), (41111, 300, 8), (60000, 130, 7), (40001, 2100, 6)])
def test_few_rows_meet_again(L, acc, rows, cols, batch, group, zeros):
    """5 to 8 F32 rows of many rows of W: two tiles of columns and several meetings of a CTA."""
    product(L, acc, np.random.default_rng(rows), rows, cols, batch, group, zeros, "f32", residual=zeros)


@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_half_rows_of_two_tiles(L, acc, group, zeros):
    """9 to 12 F16 rows in the kernel for few, and up to 16 of matrices too wide for the other."""
    rng = np.random.default_rng(group)
    for rows, cols, batch in [(3000, 700, 9), (4700, 384, 12), (20, 140000, 16), (700, 133000, 13)]:
        product(L, acc, rng, rows, cols, batch, group, zeros, "f16", residual=zeros)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("batch", [3, 30, 300])
def test_one_residual_for_all_rows(L, acc, batch, kind):
    """A bias: a residual at stride 0."""
    rng = np.random.default_rng(batch)
    code, scale, zero = matrix(rng, 270, 500, 64, True)
    x, r = rng.standard_normal((batch, 500)).astype(ref.NP[kind]), rng.standard_normal((1, 270)).astype(ref.NP[kind])
    w, dx, dr, y = packed(L, acc, code, scale, zero, 64), dev(x), dev(r), dev(np.zeros((batch, 270), ref.NP[kind]))
    w.apply(dx, y, residual=dr.expand(batch, 270))
    check(host(acc, y), x, code, scale, zero, 64, kind, np.repeat(r, batch, 0))
