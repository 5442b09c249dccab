"""Host checks of the paged 8-bit cache operators (no device): refusals of the
Python layer before anything is called, NULL contexts, the configuration of
Llama 3.2 and the references themselves."""
import ctypes

import numpy as np
import pytest

import paged_ref as ref

torch = pytest.importorskip("torch")


class NoDevice:
    """Stands where an Accelerator stands; every call through it is refused."""
    handle = None


@pytest.fixture(scope="module")
def L():
    import llamahat
    return llamahat


def pool(L, n=4, kv=2, page=32, d=64, fmt="i8", **kw):
    c = lambda: torch.zeros(n, kv, page, d, dtype=torch.uint8)  # noqa: E731
    a = {"k": c(), "v": c(), "k_scale": torch.zeros(n, kv), "v_scale": torch.zeros(n, kv)} | kw
    return L.PagedKV8(a["k"], a["v"], a["k_scale"], a["v_scale"], format=fmt, acc=NoDevice())


def test_null_context_is_refused(L):
    from llamahat import _lib
    lib = _lib.load()
    cfg, kv = _lib.LcRopeConfig(), _lib.LcKv8()
    assert lib.lc_rope_apply(None, cfg, None, None, None, 1, 1, 64, 64, 0, 0) == _lib.LC_ERR_INVALID_ARG
    assert lib.lc_pages_step(None, *[None] * 2, 1, 16, None, 1, None, None, 1, 1, *[None] * 7) == _lib.LC_ERR_INVALID_ARG
    assert lib.lc_kv8_append(None, kv, None, None, 128, 0, None, 1) == _lib.LC_ERR_INVALID_ARG
    assert lib.lc_kv8_read(None, kv, None, None, 128, 0, None, 1) == _lib.LC_ERR_INVALID_ARG
    assert lib.lc_kv8_attention(None, kv, None, None, 1, 1, 0, 1, None, None, None, 1, 1, 1, 2, 1.0) == _lib.LC_ERR_INVALID_ARG
    assert "context is NULL" in _lib.last_error()


def test_llama32_configuration(L):
    from llamahat import _lib
    c = _lib.LcRopeConfig()
    _lib.load().lc_rope_config_llama32(ctypes.byref(c))
    mine = L.RopeConfig.llama32().lc
    for name in ("head_dim", "rot_dim", "layout", "scaling", "theta", "factor", "low_freq_factor", "high_freq_factor",
                 "original_max_pos", "attn_factor"):
        assert getattr(c, name) == getattr(mine, name), name


def test_python_refusals(L):
    with pytest.raises(ValueError):
        L.RopeConfig(layout="spiral")
    with pytest.raises(ValueError):
        L.RopeConfig(scaling="guess")
    with pytest.raises(ValueError):
        pool(L, fmt="i4")
    with pytest.raises(ValueError):
        pool(L, v=torch.zeros(4, 2, 16, 64, dtype=torch.uint8))
    with pytest.raises(TypeError):
        pool(L, k=torch.zeros(4, 2, 32, 64))
    with pytest.raises(TypeError):
        pool(L, k_scale=torch.zeros(4, 2, dtype=torch.float16))
    with pytest.raises(ValueError):
        pool(L, k=torch.zeros(4, 32, 2, 64, dtype=torch.uint8).transpose(1, 2))
    cache = pool(L)
    rows, slots = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)
    for k, v, s, err in ((rows, torch.zeros(2, 2, 64), slots, ValueError), (rows, rows.half(), slots, ValueError),
                         (rows.double(), rows.double(), slots, TypeError), (rows, rows, slots.long(), TypeError),
                         (rows, rows, slots[:2], ValueError), (rows[:, :1], rows[:, :1], slots, ValueError),
                         (rows.transpose(1, 2).contiguous().transpose(1, 2), rows, slots, ValueError)):
        with pytest.raises(err):
            cache.append(k, v, s)
    with pytest.raises(ValueError):  # rows that share memory cannot be written
        cache.read(torch.zeros(1, 2, 64).expand(3, 2, 64), torch.zeros(1, 2, 64).expand(3, 2, 64), slots)
    q, lens, table = torch.zeros(3, 4, 64), torch.zeros(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        cache.attention(q, torch.zeros(3, 4, 32), None, lens, table)
    with pytest.raises(ValueError):
        cache.attention(q[:, :, :32].contiguous(), torch.zeros(3, 4, 32)[:, :3], None, lens, table)
    with pytest.raises(ValueError):
        cache.attention(q, q.clone(), lens, lens, table)  # q_start holds n_seqs + 1
    with pytest.raises(TypeError):
        cache.attention(q, q.clone(), None, lens.long(), table)
    rope = L.CudaRoPE(NoDevice())
    with pytest.raises(ValueError):
        rope.apply_scaled(torch.zeros(3, 2, 48), torch.zeros(3, 2, 48), lens, L.RopeConfig())
    with pytest.raises(ValueError):
        rope.apply_scaled(q, torch.zeros(4, 4, 64), lens, L.RopeConfig())
    with pytest.raises(ValueError):
        rope.apply_scaled(torch.zeros(64), torch.zeros(64), lens, L.RopeConfig())
    ro = np.zeros((3, 2, 64), np.float32)
    ro.flags.writeable = False
    with pytest.raises(ValueError):
        rope.apply_scaled(np.zeros((3, 2, 64), np.float32), ro, np.zeros(3, np.int32), L.RopeConfig())


def test_reference_codes():
    """The e4m3 table against torch's own, and encode as the nearest of all codes."""
    want = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.E4M3, want, equal_nan=True)
    rng = np.random.default_rng(0)
    for fmt in ("i8", "e4m3"):
        q = rng.standard_normal(2000) * np.exp(rng.standard_normal(2000) * 3)
        codes = ref.encode(q, fmt)
        values = ref.decode(np.arange(256, dtype=np.uint8), fmt)
        values = values[np.isfinite(values) & (np.abs(values) <= ref.LIMIT[fmt])]
        best = np.abs(np.clip(q, -ref.LIMIT[fmt], ref.LIMIT[fmt])[:, None] - values[None]).min(1)
        got = np.abs(np.clip(q, -ref.LIMIT[fmt], ref.LIMIT[fmt]) - ref.decode(codes, fmt))
        assert np.array_equal(got, best)


def test_quotient_rounded_to_odd_decides_every_tie():
    """Restated in fp32 on the host: a quotient moved to its odd neighbour on the
    true value's side rounds to the code that the exact quotient rounds to."""
    rng = np.random.default_rng(1)
    s = (rng.random(4000) + 0.5).astype(np.float32) / 50
    for c in (0.5, 1.5, 63.5, 126.5):
        x = (np.float64(c) * s.astype(np.float64)).astype(np.float32)
        for x in (x, np.nextafter(x, np.float32(1e9)), np.nextafter(x, np.float32(0))):
            q = x / s  # correctly rounded
            r = x.astype(np.float64) - q.astype(np.float64) * s.astype(np.float64)  # exact: 48 bits
            bits = q.view(np.int32)
            odd = np.where((r == 0) | (bits & 1 == 1), bits, bits + np.where(r > 0, 1, -1)).astype(np.int32).view(np.float32)
            exact = x.astype(np.float64) / s.astype(np.float64)
            assert np.array_equal(np.rint(odd), np.rint(exact).astype(np.float32))
