"""Pairs of beams whose best totals differ by less than 32 bits can tell."""
import numpy as np
import torch


def near_tie(rng, V, dtype, gap):
    """(logits [2, V] of ``dtype``, scores [2] float32): beam 1's best total lies above
    beam 0's by about ``gap`` (64-bit sums of the stored values; see gap_of). The scores
    and best tokens bring the two as near as their types allow, one small logit of
    beam 1 the rest: a change of e^z by d moves the logarithm of the sum S by d / S."""
    x = torch.from_numpy(2.0 * rng.standard_normal((2, V))).to(dtype)
    x[:, 77] = 10.0                                     # mostly the best token of both
    x[1, 3] = 0.5
    s = np.array([-3.0, 0.0])
    s[1] = np.float32(s[0] + _best(x[0]) - _best(x[1]))
    # What is left is at most half an ulp of s1, so e^z changes by a part of S 2^-23.
    off = (s[1] + _best(x[1])) - (s[0] + _best(x[0]))
    S = np.exp(x[1].double().numpy()).sum()
    e = np.exp(float(x[1, 3])) + S * np.expm1(off - gap)
    assert e > 0
    x[1, 3] = float(np.log(e))
    return x, torch.tensor(s, dtype=torch.float32)


def _best(row):
    """The largest logit less the log of the sum of exponentials, in 64 bits."""
    r = row.double().numpy()
    return r.max() - (r.max() + np.log(np.exp(r - r.max()).sum()))


def gap_of(x, s):
    """Beam 1's best total less beam 0's, and 32 bits' ulp of the totals."""
    t = [float(s[k]) + _best(x[k]) for k in (0, 1)]
    return t[1] - t[0], float(np.spacing(np.float32(abs(t[0]))))
