"""Attention over a sliding window and sinks in 64 bits, with how far a correct
bf16 kernel may be off it."""
import math

import numpy as np
import torch

from rngd_pd_amd.engines.paged_cache import k_block_rows


def visible(p, window, sinks):
    """The positions that a query at position p sees, in order."""
    first = max(0, p + 1 - window) if window else 0
    return list(range(min(sinks, first))) + list(range(first, p + 1))


def attend(q, k, v, scale, p_rounded=True):
    """q [H, G, D], k, v [n, H, D] (any dtype) -> (out, bound), 64-bit [H, G, D].

    The kernel's products of bf16 are exact; a score of D terms is off by D 2^-24
    times the sum of their magnitudes (scaled), and so, relatively, is its weight
    e^score; the weights' sum by n 2^-24; a weight that is rounded to bf16 by
    2^-8; the exp2 and its argument by less than 2^-18 together. Each of these
    shifts out by that share of A = sum p |v|; the result is rounded to bf16 once
    (2^-8 of itself, and 2^-134 where it is subnormal)."""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[0] == 0:
        z = torch.zeros_like(q)
        return z, z
    n, D = k.shape[0], q.shape[2]
    kh, vh = k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
    s = torch.matmul(q, kh) * scale
    p = torch.softmax(s, -1)
    out, A = torch.matmul(p, vh), torch.matmul(p, vh.abs())
    mass = float((torch.matmul(q.abs(), kh.abs()) * abs(scale)).max())
    share = 2 * (D * 2.0 ** -24 * mass + n * 2.0 ** -24) + 2.0 ** -18
    share += 2.0 ** -8 if p_rounded else 0.0
    return out, (1 + 2.0 ** -8) * share * A + 2.0 ** -8 * out.abs() + 2.0 ** -134


def paged(rng, ctx, hkv, D=128, extra=3, width=None, held=None):
    """A permuted pool for streams of ctx tokens: (tables [B, width] int32 numpy, nb);
    held(b) gives the block indices that stream b holds (all by default)."""
    mb = width or max(1, max(-(-max(c, 1) // 16) for c in ctx))
    rows = [sorted(held(b)) if held else list(range(-(-c // 16))) for b, c in enumerate(ctx)]
    nb = sum(len(r) for r in rows) + extra
    ids = rng.permutation(nb).astype(np.int32)
    tables, at = np.full((len(ctx), mb), -1, np.int32), 0
    for b, r in enumerate(rows):
        tables[b, r] = ids[at:at + len(r)]
        at += len(r)
    return tables, nb


def decode_reference(q, ck, cv, tables, ctx, window, sinks, scale):
    """decode_attention's result and bound [B, Hq, D], streams one by one."""
    B, Hq, D = q.shape
    nb, H = ck.shape[:2]
    outs, bounds = [], []
    for b, c in enumerate(ctx):
        c_in = min(c, tables.shape[1] * 16)
        pos = [t for t in (visible(c - 1, window, sinks) if c > 0 else []) if t < c_in]
        pos = [t for t in pos if 0 <= tables[b, t // 16] < nb]
        blk = torch.tensor([int(tables[b, t // 16]) for t in pos], dtype=torch.int64, device=q.device)
        slot = torch.tensor([t % 16 for t in pos], dtype=torch.int64, device=q.device)
        if pos:
            k = k_block_rows(ck[blk])[torch.arange(len(pos), device=q.device), :, slot]
            v = cv[blk, :, :, slot]
        else:
            k = v = torch.zeros((0, H, D), device=q.device)
        o, e = attend(q[b].view(H, Hq // H, D), k, v, scale)
        outs.append(o.view(Hq, D))
        bounds.append(e.view(Hq, D))
    return torch.stack(outs), torch.stack(bounds)


def assert_within(got, want, bound, what=""):
    assert torch.isfinite(got).all(), what
    off = (got.double() - want).abs() - bound
    worst = float(off.max())
    at = np.unravel_index(int(off.argmax()), tuple(off.shape))
    assert worst <= 0, (what, worst, at, float(got.double()[at]), float(want[at]), float(bound[at]))


SCALE = 1.0 / math.sqrt(128)
