"""The near ties that the selection is tested with are such, of either sign, and a
selection by 32-bit totals does not pass them."""
import numpy as np
import pytest
import torch

from tests._near_ties import _best, gap_of, near_tie

GAPS = [3e-9, -3e-9, 4e-8, -4e-8]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gaps(dtype):
    rng = np.random.default_rng(6)
    wrong = []
    for gap in GAPS * 3:
        want = gap if dtype is torch.float32 else np.copysign(max(abs(gap), 4e-8), gap)
        x, s = near_tie(rng, 50000, dtype, want)
        assert x[0].argmax() == 77 and x[1].argmax() == 77
        got, ulp = gap_of(x, s)
        # bf16: the small logit's half step of 2^-8 of a value of at most 2, of e^z in S.
        assert abs(got - want) <= (1e-10 if dtype is torch.float32 else 3e-8)
        assert got * gap > 0 and 1e-9 < abs(got) < ulp / 2
        t32 = [np.float32(np.float32(float(s[k])) + np.float32(_best(x[k]))) for k in (0, 1)]
        first = 1 if t32[1] > t32[0] else 0             # the lower beam among equals
        wrong.append(first != (got > 0))
    assert any(wrong)
