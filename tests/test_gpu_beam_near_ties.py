"""beam_select between beams whose best totals 32 bits cannot tell apart, either of
them first."""
import numpy as np
import pytest
import torch

from tests._near_ties import gap_of, near_tie
from tests.test_gpu_beam import check_select
from tests.test_near_ties import GAPS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,R,V", [
    (torch.float32, 4, 1001), (torch.float32, 4, 50000), (torch.float32, 100, 50001),
    (torch.bfloat16, 4, 50000), (torch.bfloat16, 100, 50001)])
def test_near_ties(cuda, dtype, R, V):
    """One request per gap; 200 rows of 50001 take several steps of a wavefront."""
    rng = np.random.default_rng(V)
    rows, scores, firsts = [], [], []
    for r in range(R):
        gap = GAPS[r % len(GAPS)]
        if dtype is torch.bfloat16:                     # as fine as the small logit is
            gap = np.copysign(4e-8, gap)
        x, s = near_tie(rng, V, dtype, gap)
        got, ulp = gap_of(x, s)
        assert got * gap > 0 and 1e-9 < abs(got) < ulp / 2
        rows.append(x)
        scores.append(s)
        firsts.append(1 if got > 0 else 0)
    print(f"near ties {dtype} R={R} V={V}", flush=True)
    out = check_select(torch.cat(rows).to(cuda), torch.stack(scores).to(cuda), 8)
    assert out[1][:, 0].tolist() == firsts and set(firsts) == {0, 1}
