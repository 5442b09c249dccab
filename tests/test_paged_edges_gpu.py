"""Paged 8-bit cache operators at their edges: half precision against its own
rounding, long sums, batch sizes at the border of a launch's limits, threads
that share a context, the smallest scales and quotients."""
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import attention_case, cache_of, check_attention, dev, exact_on_gpu, lib, make_pool, sync  # noqa: F401

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TESTS = os.path.dirname(os.path.abspath(__file__))


# ------------------------------------------------------- half precision rows

@pytest.mark.parametrize("heads,kv,page,d,lens,counts", [
    (32, 8, 32, 64, [937, 3022, 2500], [253, 278, 461]),
    (8, 2, 64, 128, [1500, 700], [1400, 333]),
    (8, 2, 32, 64, [9000], [64]),
    (32, 8, 32, 64, [4000] * 24, [1] * 24),
])
@pytest.mark.parametrize("positive", [False, True])
def test_attention_of_half_rows_is_off_by_the_rounding_of_the_result(lib, heads, kv, page, d, lens, counts, positive):
    """Half rows are rounded once, at the end: the 2-norm of the error is that of
    rounding the exact result.  Errors of 32-bit sums come to it in quadrature:
    2 % leaves room for a fifth of a half precision rounding, 4e-5 of the
    result, where weights rounded to half precision would add as much as the
    result's own rounding (1.4 times the norm).  The same for the kernel of few
    queries and that of many, so max_q does not choose the accuracy."""
    rng = np.random.default_rng(heads + d)
    pool, table, q_start, q = attention_case(lib, rng, lens, counts, heads, kv, page, d, "i8", "f16", extra_rows=0)
    if positive:
        pool["v"] = np.maximum(pool["v"] & 0x7F, 1)
    want, _, _ = exact_on_gpu(pool, table, q_start, lens, q, "i8", d ** -0.5)
    cache, _ = cache_of(lib, pool, "i8")
    out = torch.full(q.shape, 7.0, dtype=torch.float16, device="cuda")
    cache.attention(dev(q), out, dev(q_start), dev(np.array(lens, np.int32)), dev(table), max_q=max(counts))
    sync()
    rounding = torch.linalg.vector_norm(want.half().double() - want)
    assert float(torch.linalg.vector_norm(out.double() - want) / rounding) <= 1.02


# ------------------------------------------------------------ launch limits

PAGES_OF_N = """
import sys
import numpy as np, torch
import llamahat
pages = llamahat.CudaKernelFactory().createPages(llamahat.Accelerator(0))
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
n = int(sys.argv[1])
z = lambda k: torch.full((k,), -9, dtype=torch.int32, device="cuda")
lens_out, start, slots, pos, ids, count, status = z(n), z(n + 1), z(n), z(n), z(n), z(1), z(2)
table, free = torch.full((n, 1), -1, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
pages.step(i32([0] * n), i32([1] * n), table, free, i32([n]), 16, lens_out, start, slots, pos, ids, count, status)
torch.cuda.synchronize()
assert status.tolist() == [0, 0] and count.tolist() == [0]
assert lens_out.tolist() == [1] * n and start.tolist() == list(range(n + 1)) and ids.tolist() == list(range(n))
assert table[:, 0].tolist() == list(range(n - 1, -1, -1)) and slots.tolist() == [16 * p for p in range(n - 1, -1, -1)]
"""


@pytest.mark.parametrize("n", [2417, 2418, 2440, 2457, 2458])
def test_pages_step_of_batches_whose_sums_need_48_kb(lib, n):
    """In a process of its own: a larger batch before it would have raised the
    kernel's shared-memory limit for good."""
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    r = subprocess.run([sys.executable, "-c", PAGES_OF_N, str(n)],
                       env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-800:]
