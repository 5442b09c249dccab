"""4-bit weights against 64-bit references: quantising, packing and reading,
products, and the last step of an answer with all of them."""
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


def dev(x, pad=0):
    """A CUDA tensor of x whose rows lie `pad` elements further apart, with NaN between them."""
    t = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    if pad:
        held = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device="cuda")
        held[:, :t.shape[1]] = t
        t = held[:, :x.shape[1]]
    torch.cuda.synchronize()
    return t


def host(acc, t):
    acc.synchronize()
    return t.cpu().numpy()


def weights(rng, rows, cols, kind):
    w = rng.standard_normal((rows, cols)) * 0.02 * np.exp(0.3 * rng.standard_normal(cols))
    return w.astype(ref.NP[kind])


def packed(L, acc, code, scale, zero, group):
    w = L.Weights4.empty(*code.shape, group, zeros=zero is not None, acc=acc)
    torch.cuda.synchronize()
    w.pack(ref.two_to_a_byte(code), scale, zero)
    return w


# ---------------------------------------------------- quantise, pack, read

SHAPES = [(1, 1), (2, 15), (15, 31), (16, 32), (17, 33), (33, 64), (16, 100), (7, 128), (40, 129), (19, 300), (130, 1024),
          (64, 2085)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("kind", ["f32", "f16"])
def test_quantize_and_read(L, acc, kind, zeros, group):
    rng = np.random.default_rng(group + zeros)
    for rows, cols in SHAPES:
        for pad in (0, 3):
            x = weights(rng, rows, cols, kind)
            code, scale, zero = ref.quantize(x, group, zeros)
            w = L.Weights4.empty(rows, cols, group, zeros=zeros, acc=acc)
            v = dev(x, pad)  # kept until the call is done
            w.quantize(v)
            for out, opad in (("f32", pad), ("f16", 0)):
                back = dev(np.full((rows, cols), 7.0, ref.NP[out]), opad)
                w.read(back)
                want = ref.values(code, scale, zero, group).astype(ref.NP[out])
                np.testing.assert_array_equal(host(acc, back), want, err_msg=f"{rows} x {cols}, pad {pad}, as {out}")
                if opad:  # what lies between the rows is left alone
                    assert torch.isnan(back._base[:, cols:]).all()


@pytest.mark.parametrize("zeros", [False, True])
def test_quantize_hard_values(L, acc, zeros):
    """Ties, zeros, the smallest and largest numbers, NaN and infinities."""
    rng = np.random.default_rng(5)
    x = np.zeros((16, 256), np.float32)
    x[1] = np.arange(256) % 15 - 7           # whole steps
    x[2] = (np.arange(256) % 29 - 14) / 2.0  # halves: ties of a scale of 1
    x[3] = rng.standard_normal(256) * 1e-8   # scales that are subnormal or 0
    x[4] = rng.standard_normal(256) * 1e-40
    x[5] = rng.standard_normal(256) * 3e5    # scales at the cap
    x[6] = rng.standard_normal(256) * 1e38
    x[7] = 1.0
    x[8] = -1.0
    x[9, ::3] = np.nan
    x[9, 1::3] = 0.5
    x[10, ::5] = np.inf
    x[10, 1::5] = -np.inf
    x[10, 2::5] = 3.25
    x[11] = np.nan
    x[12, 5] = np.inf
    x[13] = rng.standard_normal(256) * np.exp(4 * rng.standard_normal(256))
    x[14] = np.nextafter(np.float32(3.5), np.float32(0)) * (1 - 2 * (np.arange(256) % 2))
    x[14, ::32] = 7.0
    x[15] = np.nextafter(np.float32(2.5), np.float32(4))
    x[15, ::32] = -7.0
    for kind in ("f32", "f16"):
        with np.errstate(over="ignore"):
            v = x.astype(ref.NP[kind])
        for group in (32, 128):
            code, scale, zero = ref.quantize(v, group, zeros)
            w = L.Weights4.empty(*v.shape, group, zeros=zeros, acc=acc)
            dv = dev(v)
            w.quantize(dv)
            back = dev(np.zeros(v.shape, np.float32))
            w.read(back)
            np.testing.assert_array_equal(host(acc, back), ref.values(code, scale, zero, group).astype(np.float32))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_pack_holds_any_code(L, acc, zeros, group):
    rng = np.random.default_rng(9)
    for rows, cols in SHAPES:
        groups = -(-cols // group)
        code = rng.integers(0, 16, (rows, cols), np.uint8)
        scale = (rng.standard_normal((rows, groups)) * 0.01).astype(np.float16)  # of either sign
        zero = rng.integers(0, 16, (rows, groups), np.uint8) if zeros else None
        w = packed(L, acc, code, scale, zero, group)
        back = np.zeros((rows, cols), np.float32)  # host memory is staged
        w.read(back)
        np.testing.assert_array_equal(back, ref.values(code, scale, zero, group).astype(np.float32))


# ----------------------------------------------------------------- product

def check_product(L, acc, rng, rows, cols, batch, group, zeros, kind, pad=0, residual=False, x=None):
    groups = -(-cols // group)
    code = rng.integers(0, 16, (rows, cols), np.uint8)
    scale = (0.002 * np.exp(rng.standard_normal((rows, groups)))).astype(np.float16)
    zero = rng.integers(0, 16, (rows, groups), np.uint8) if zeros else None
    if x is None:
        x = rng.standard_normal((batch, cols)) * np.exp(rng.standard_normal(cols))
    x = x.astype(ref.NP[kind])
    r = rng.standard_normal((batch, rows)).astype(ref.NP[kind]) if residual else None
    w = packed(L, acc, code, scale, zero, group)
    y = dev(np.full((batch, rows), np.nan, ref.NP[kind]), pad)
    dx, dr = dev(x, pad), None if r is None else dev(r, pad)
    w.apply(dx, y, residual=dr)
    got = host(acc, y).astype(np.float64)
    want, terms, far = ref.product(x, code, scale, zero, group, r)
    off = np.abs(got - want) - ref.product_bound(want, terms, far, groups, kind)
    assert np.all(off <= 0), f"{rows} x {cols}, batch {batch}, group {group}, {kind}: {off.max():g} past the bound at {np.unravel_index(off.argmax(), off.shape)}"
    if pad:
        assert torch.isnan(y._base[:, rows:]).all()
    return got


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("batch", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 64, 65, 130])
def test_product(L, acc, batch, kind, zeros, group):
    rng = np.random.default_rng(batch * 7 + group)
    for rows, cols in [(1, 1), (15, 33), (16, 128), (100, 200), (129, 640), (300, 1111)]:
        check_product(L, acc, rng, rows, cols, batch, group, zeros, kind, pad=3 if rows == 100 else 0, residual=cols % 2 == 0)


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols,batch", [(2048, 2048, 1), (2048, 8192, 1), (16384, 512, 1), (40000, 256, 3), (64, 16384, 2),
                                             (48, 40000, 1), (48, 20000, 9), (2048, 8192, 8), (4096, 2048, 64), (1777, 2085, 5),
                                             (520, 2048, 300), (5000, 128, 1000), (256, 8192, 64), (100, 20000, 40)])
def test_product_sizes(L, acc, rows, cols, batch, kind):
    rng = np.random.default_rng(rows)
    check_product(L, acc, rng, rows, cols, batch, 128, False, kind)
    check_product(L, acc, rng, rows, cols, batch, 32, True, kind, residual=True)


@pytest.mark.parametrize("rows,cols,batch", [(20, 60000, 8),    # a CTA's columns in parts, one after the other
                                             (17, 140000, 11),  # too wide for the workspace: a few rows at a time
                                             (40, 8192, 1100),  # more rows than the workspace takes at once
                                             (300, 256, 1500)])
def test_product_in_parts(L, acc, rows, cols, batch):
    rng = np.random.default_rng(cols)
    check_product(L, acc, rng, rows, cols, batch, 64, True, "f32", residual=True)
    check_product(L, acc, rng, rows, cols, batch, 128, False, "f16")


@pytest.mark.parametrize("batch", [1, 7, 70])
def test_product_rows_of_unlike_size(L, acc, batch):
    """fp32 rows from the smallest numbers to near the largest, one-sided sums,
    zeros, far outliers: each row has a scale of its own."""
    rng = np.random.default_rng(3)
    size = 10.0 ** rng.uniform(-36, 34, (batch, 1))
    x = rng.standard_normal((batch, 700)) * size
    x[:, 5] *= 1000.0
    x[batch // 2] = np.abs(x[batch // 2])
    if batch > 2:
        x[1] = 0.0
    check_product(L, acc, rng, 50, 700, batch, 64, True, "f32", x=x)
    check_product(L, acc, rng, 50, 700, batch, 128, False, "f32", x=np.abs(x))


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("batch", [3, 40])
def test_product_bad_rows_stay_alone(L, acc, batch, kind):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((batch, 300))
    clean = check_product(L, acc, np.random.default_rng(8), 40, 300, batch, 64, True, kind, x=x)
    g = np.random.default_rng(8)
    code = g.integers(0, 16, (40, 300), np.uint8)
    scale = (0.002 * np.exp(g.standard_normal((40, 5)))).astype(np.float16)
    zero = g.integers(0, 16, (40, 5), np.uint8)
    w = packed(L, acc, code, scale, zero, 64)
    x[1, 17], x[2, 200] = np.nan, np.inf
    y = dev(np.zeros((batch, 40), ref.NP[kind]))
    dx = dev(x.astype(ref.NP[kind]))
    w.apply(dx, y)
    got = host(acc, y).astype(np.float64)
    keep = [b for b in range(batch) if b not in (1, 2)]
    np.testing.assert_array_equal(got[keep], clean[keep])
    assert np.isnan(got[1]).all() and not np.isfinite(got[2]).any()


def test_product_in_place_and_host(L, acc):
    rng = np.random.default_rng(6)
    code, scale, zero = ref.quantize(weights(rng, 70, 256, "f32"), 64, False)
    w = packed(L, acc, code, scale, zero, 64)
    for batch in (1, 30):
        x, r = rng.standard_normal((batch, 256), np.float32), rng.standard_normal((batch, 70), np.float32)
        want, terms, far = ref.product(x, code, scale, zero, 64, r)
        bound = ref.product_bound(want, terms, far, 4, "f32")
        y = dev(r)
        dx = dev(x)
        w.apply(dx, y, residual=y)
        assert np.all(np.abs(host(acc, y) - want) <= bound)
        y = r.copy()
        w.apply(x, y, residual=y)  # host memory
        assert np.all(np.abs(y - want) <= bound)
    w.apply(dev(np.zeros((0, 256), np.float32)), dev(np.zeros((0, 70), np.float32)))


def test_product_is_repeatable_and_captured(L, acc):
    """The same bits again, eagerly and from a graph, on weights that were made on the same stream."""
    rng = np.random.default_rng(12)
    st = torch.cuda.ExternalStream(acc.stream)
    v = dev(weights(rng, 500, 2048, "f32"))
    xs = [dev(rng.standard_normal((b, 2048), np.float32)) for b in (1, 6, 48)]
    ys = [torch.empty(len(x), 500, device="cuda") for x in xs]
    w = L.Weights4.empty(500, 2048, 128, acc=acc)
    torch.cuda.synchronize()

    def step():
        w.quantize(v)
        for x, y in zip(xs, ys):
            w.apply(x, y)
    step()
    first = [host(acc, y) for y in ys]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step()
    for _ in range(3):
        for y in ys:
            y.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        for y, f in zip(ys, first):
            np.testing.assert_array_equal(host(acc, y), f)


def test_shared_rows_and_strides(L, acc):
    """One row of x for all of a batch (stride 0), rows of y far apart, odd addresses."""
    rng = np.random.default_rng(14)
    code, scale, zero = ref.quantize(weights(rng, 90, 200, "f32"), 64, True)
    w = packed(L, acc, code, scale, zero, 64)
    for kind in ("f32", "f16"):
        for batch in (1, 6, 21):
            held = torch.zeros(201, dtype=torch.from_numpy(np.zeros(1, ref.NP[kind])).dtype, device="cuda")
            x = rng.standard_normal(200).astype(ref.NP[kind])
            held[1:] = torch.from_numpy(x)
            y = torch.zeros(batch, 1000, dtype=held.dtype, device="cuda")
            torch.cuda.synchronize()
            w.apply(held[1:].expand(batch, 200), y[:, 7:97])
            want, terms, far = ref.product(x[None], code, scale, zero, 64)
            got = host(acc, y)
            assert np.all(np.abs(got[:, 7:97] - want) <= ref.product_bound(want, terms, far, 4, kind))
            assert not got[:, :7].any() and not got[:, 97:].any()


def test_workspace_and_capture(L):
    """The first product of many rows makes the workspace: not within a capture."""
    acc = L.Accelerator(0)
    w = L.Weights4.empty(64, 256, 64, acc=acc)
    rng = np.random.default_rng(15)
    v, x, y = dev(weights(rng, 64, 256, "f32")), dev(rng.standard_normal((40, 256), np.float32)), dev(np.zeros((40, 64), np.float32))
    w.quantize(v)
    st, graph = torch.cuda.ExternalStream(acc.stream), torch.cuda.CUDAGraph()
    acc.synchronize()
    with pytest.raises(L.IllegalStateError):
        with torch.cuda.graph(graph, stream=st):
            w.apply(x, y)
    w.apply(x, y)
    whole = host(acc, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        w.apply(x, y)
    y.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        graph.replay()
    np.testing.assert_array_equal(host(acc, y), whole)
    del graph


def test_threads_share_a_context(L, acc):
    """Two threads, products of many rows through the one workspace: each call is whole."""
    import threading
    rng = np.random.default_rng(16)
    code, scale, zero = ref.quantize(weights(rng, 300, 512, "f32"), 64, False)
    w = packed(L, acc, code, scale, zero, 64)
    xs = [dev(rng.standard_normal((b, 512), np.float32)) for b in (33, 90)]
    ys = [torch.zeros(len(x), 300, device="cuda") for x in xs]
    torch.cuda.synchronize()
    alone = []
    for x, y in zip(xs, ys):
        w.apply(x, y)
        alone.append(host(acc, y))
    wrong = []

    def run(x, y, want):
        for _ in range(100):
            w.apply(x, y)
        acc.synchronize()
        if not np.array_equal(y.cpu().numpy(), want):
            wrong.append(len(x))
    threads = [threading.Thread(target=run, args=a) for a in zip(xs, ys, alone)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


# ----------------------------------------------------- refusals on a device

def test_refusals(L, acc):
    w = L.Weights4.empty(64, 256, 64, acc=acc)
    x, y = dev(np.zeros((2, 256), np.float32)), dev(np.zeros((2, 64), np.float32))
    with pytest.raises(L.IllegalArgumentError):  # rows of y that overlap
        L._lib.check(w.lib.lc_w4_product(acc.handle, w._w, x.data_ptr(), 256, y.data_ptr(), 63, None, 0, 2, 0))
    with pytest.raises(L.IllegalArgumentError):
        L._lib.check(w.lib.lc_w4_product(acc.handle, w._w, x.data_ptr(), 256, y.data_ptr(), 64, y.data_ptr(), 65, 2, 0))
    with pytest.raises(L.IllegalArgumentError):
        L._lib.check(w.lib.lc_w4_product(acc.handle, w._w, x.data_ptr(), 256, None, 64, None, 0, 2, 0))
    with pytest.raises(L.IllegalArgumentError):
        L._lib.check(w.lib.lc_w4_product(acc.handle, w._w, x.data_ptr(), 256, y.data_ptr(), 64, None, 0, 2, 3))
    with pytest.raises(L.IllegalArgumentError):
        L._lib.check(w.lib.lc_w4_product(acc.handle, w._w, x.data_ptr(), 256, y.data_ptr(), 64, None, 0, -1, 0))
    bad = L._lib.LcW4(w.tensors[0].data_ptr() + 4, w.tensors[1].data_ptr(), None, 63, 256, 64)
    with pytest.raises(L.IllegalArgumentError):  # alignment
        L._lib.check(w.lib.lc_w4_quantize(acc.handle, bad, x.data_ptr(), 256, 0))
    h = np.zeros(1 << 16, np.uint8)
    bad = L._lib.LcW4(h.ctypes.data, w.tensors[1].data_ptr(), None, 64, 256, 64)
    with pytest.raises(L.IllegalArgumentError):  # host memory
        L._lib.check(w.lib.lc_w4_quantize(acc.handle, bad, x.data_ptr(), 256, 0))
    with pytest.raises(L.IllegalArgumentError):  # zero points on one side
        L._lib.check(w.lib.lc_w4_pack(acc.handle, w._w, h.ctypes.data, h.ctypes.data, h.ctypes.data))
    with pytest.raises(L.LlamaCudaError):
        L._lib.check(w.lib.lc_w4_product(acc.handle, L._lib.LcW4(w.tensors[0].data_ptr(), w.tensors[1].data_ptr(), None, 64, 256, 48),
                                         x.data_ptr(), 256, y.data_ptr(), 64, None, 0, 2, 0))
    w.apply(x, y)  # the context stays usable
    acc.synchronize()


# ---------------------------------------------- the last step of an answer

def test_answer(L, acc):
    """lm_head in 4 bits, logits, the chosen token's log probability and its
    alternatives: eagerly and from a graph."""
    rng = np.random.default_rng(21)
    vocab, dim, n = 5003, 512, 6
    head, x = weights(rng, vocab, dim, "f32") * 4, rng.standard_normal((n, dim)).astype(np.float32)
    code, scale, zero = ref.quantize(head, 64, True)
    w = L.Weights4.empty(vocab, dim, 64, zeros=True, acc=acc)
    lp = L.CudaKernelFactory().createLogProbs(acc)
    v, dx = dev(head), dev(x)
    chosen = rng.integers(0, vocab, n).astype(np.int32)
    logits = torch.empty(n, vocab, device="cuda")
    out = [torch.empty(n, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda"),
           torch.empty(n, 5, dtype=torch.int32, device="cuda"), torch.empty(n, 5, device="cuda")]
    tokens = dev(chosen[:, None])[:, 0].contiguous()
    torch.cuda.synchronize()
    w.quantize(v)

    def step():
        w.apply(dx, logits)
        lp.apply(logits, tokens, *out, scale=0.8)

    def check():
        z = host(acc, logits).astype(np.float64)
        want, terms, far = ref.product(x, code, scale, zero, 64)
        assert np.all(np.abs(z - want) <= ref.product_bound(want, terms, far, 8, "f32"))
        for i in range(n):
            p, h, mean = ref.logprobs(z[i], np.float32(0.8))
            o = ref.order(z[i])
            b = ref.logprobs_bound(p - p.max(), mean, vocab)
            assert abs(out[0][i].item() - p[chosen[i]]) <= b[chosen[i]]
            assert out[1][i].item() == np.nonzero(o == chosen[i])[0][0]
            assert abs(out[2][i].item() - h) <= 4 * (1 + mean) * b.min()
            assert out[3][i].tolist() == o[:5].tolist()
            assert np.all(np.abs(out[4][i].cpu().numpy() - p[o[:5]]) <= b[o[:5]])
    step()
    check()
    st, graph = torch.cuda.ExternalStream(acc.stream), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        step()
    x[:] = rng.standard_normal((n, dim))
    dx.copy_(torch.from_numpy(x))
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        graph.replay()
    check()
