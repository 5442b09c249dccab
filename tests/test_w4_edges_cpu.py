"""Calls of the 4-bit weights and of the log probabilities that Python refuses before
the library sees them (no device)."""
import numpy as np
import pytest

from test_w4_cpu import NoDevice, weights

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def L():
    import llamahat
    return llamahat


def test_pack_refuses_scales_of_another_shape(L):
    """Scales the other way round, or with a group too many, have enough elements, but
    every one of them would be another group's."""
    w = weights(L)  # 48 rows, 300 columns, groups of 64
    codes, zeros = torch.zeros(48, 150, dtype=torch.uint8), torch.zeros(48, 5, dtype=torch.uint8)
    for shape in ((5, 48), (48, 6), (1, 240), (48, 5, 1)):
        for scales in (torch.zeros(shape, dtype=torch.float16), np.zeros(shape, np.float16)):
            with pytest.raises(ValueError, match="scales"):  # by Python: the library's error is a ValueError too
                w.pack(codes, scales, zeros)
    for scales in (torch.zeros(48, 5, dtype=torch.float16), np.zeros((48, 5), np.uint16), np.zeros(240, np.float16)):
        with pytest.raises(L.IllegalArgumentError):  # in order, but there is no device
            w.pack(codes, scales, zeros)
    with pytest.raises(ValueError):
        w.pack(codes, np.zeros(239, np.float16), zeros)


def test_logprobs_refuses_alternatives_without_rows(L):
    lp = L.CudaLogProbs(NoDevice())
    for ids, lps in ((torch.zeros(6, dtype=torch.int32), None), (None, torch.zeros(6)), (torch.zeros(2, 3, dtype=torch.int32), torch.zeros(6))):
        with pytest.raises(ValueError):
            lp.apply(torch.zeros(2, 50), top_ids=ids, top_logprobs=lps)
