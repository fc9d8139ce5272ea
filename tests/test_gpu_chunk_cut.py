"""Steps with room for fewer tokens than their requests get: the tokens left out have no
row, no position and no slot; those that are kept are as in the whole step."""
import math

import numpy as np
import pytest
import torch

from rngd_pd_amd import kernels as K
from rngd_pd_amd.engines.paged_cache import k_block_index
from tests import _chunk_ref as ref
from tests._util import rand_bf16, to_dev

pytestmark = pytest.mark.gpu
D, SCALE = 128, 1.0 / math.sqrt(128)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


CUT = [
    # Hq, Hkv, [(in the cache before, new)], rows of q, window, sinks
    (32, 8, [(40, 3), (100, 9)], 7, 0, 0),                # few rows of each, the last cut
    (32, 8, [(40, 3), (100, 9), (7, 2)], 3, 0, 0),        # the others have no row at all
    (8, 2, [(300, 4)], 1, 0, 0),
    (32, 8, [(5, 1), (1000, 200)], 150, 0, 0),            # a longer one cut, beside a single token
    (32, 8, [(700, 90), (20, 60), (9, 1)], 101, 0, 0),
    (32, 8, [(3000, 300)], 130, 0, 0),                    # one alone, its context split
    (32, 8, [(0, 500)], 333, 0, 0),
    (32, 8, [(90, 40), (200, 5)], 43, 24, 4),
    (28, 4, [(600, 100), (50, 30)], 117, 64, 0),
]


@pytest.mark.parametrize("Hq,Hkv,lens,N,window,sinks", CUT)
def test_attention(cuda, Hq, Hkv, lens, N, window, sinks):
    """The rows that q has, against those of the whole step in 64 bits; what a request has
    behind its last row, which such a step does not write, is NaN."""
    print(f"cut attention Hq={Hq} Hkv={Hkv} lens={lens} N={N} window={window}", flush=True)
    rng = np.random.default_rng(Hq + N)
    new, ctx = [n for _, n in lens], [p + n for p, n in lens]
    tables, nb = ref.pool(rng, ctx)
    q = to_dev(rand_bf16(rng, (sum(new), Hq, D)))
    ck, cv = (to_dev(rand_bf16(rng, s)) for s in ((nb, Hkv, 16, D), (nb, Hkv, D, 16)))
    want, bound = ref.attention(q, ck, cv, tables, new, ctx, window, sinks, SCALE)
    place, at = k_block_index(D, "cuda"), 0
    for r, (p, n) in enumerate(lens):
        for t in range(p + min(max(N - at, 0), n), p + n):
            b = int(tables[r, t // 16])
            ck[b].view(Hkv, -1)[:, place[t % 16]] = float("nan")
            cv[b, :, :, t % 16] = float("nan")
        at += n
    span = {"window": window, "sinks": sinks} if window else {}
    starts = np.concatenate([[0], np.cumsum(new)]).tolist()
    got = K.chunk_attention(q[:N], ck, cv, torch.from_numpy(tables).to(cuda), _int32(starts), _int32(ctx),
                            max(new), max(ctx), scale=SCALE, **span)
    ref.within(got, want[:N], bound[:N])


@pytest.mark.parametrize("past,new,N", [([20, 0, 9], [5, 30, 6], 17), ([100], [200], 90),
                                        ([33, 70], [1, 140], 128)])
def test_a_step(cuda, past, new, N):
    """Map, write and attention of a step that is cut: the keys, values and results of the
    tokens that are kept equal those of the step with room for all."""
    print(f"cut step past={past} new={new} N={N}", flush=True)
    rng, R, Hq, Hkv = np.random.default_rng(N), len(past), 8, 2
    total, width = sum(new), 32
    held = [-(-p // 16) for p in past]
    ids = rng.permutation(R * width).astype(np.int32)
    tables, at = np.full((R, width), -1, np.int32), 0
    for r, h in enumerate(held):
        tables[r, :h] = ids[at:at + h]
        at += h
    qkv = to_dev(rand_bf16(rng, (total, (Hq + 2 * Hkv) * D)))
    ck, cv = (to_dev(rand_bf16(rng, s)) for s in ((R * width, Hkv, 16, D), (R * width, Hkv, D, 16)))
    inv = torch.tensor([10000.0 ** (-2 * i / D) for i in range(64)], device=cuda)
    results = []
    for rows in (total, N):
        k, v, tab = ck.clone(), cv.clone(), torch.from_numpy(tables).to(cuda)
        m = K.chunk_map(_int32(past), _int32(new), tab, torch.from_numpy(ids[at:]).to(cuda), rows)
        q = K.rope_cache_write(qkv[:rows], inv, m.positions, m.slots, k, v, Hq)
        out = K.chunk_attention(q, k, v, tab, m.starts, m.ctx_lens, max(new), width * 16, scale=SCALE)
        want, bound = ref.attention(q, k, v, tab.cpu().numpy(), new, m.ctx_lens.tolist(), 0, 0, SCALE) \
            if rows == total else results[0][2:]
        ref.within(out, want[:rows], bound[:rows], rows)
        results.append((q, m, want, bound))
    (q, m, *_), (q_cut, m_cut, *_) = results
    assert torch.equal(q_cut, q[:N]) and torch.equal(m_cut.slots, m.slots[:N])
