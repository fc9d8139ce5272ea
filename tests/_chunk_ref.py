"""The operators over several requests' new tokens in 64 bits (and the map in plain
Python), with how far a correct kernel may be off them."""
import numpy as np
import torch

from rngd_pd_amd.engines.paged_cache import k_block_rows


def chunk_map(past, new, tables, free, N):
    """(tables, starts, ctx, positions, slots, taken) token by token; tables [R, W] numpy."""
    tables, W = tables.copy(), tables.shape[1]
    starts, ctx, positions, slots, taken = [0], [], [], [], 0
    for r, (p, n) in enumerate(zip(past, new)):
        p = min(max(p, 0), 16 * W)
        n = min(max(n, 0), 16 * W - p)
        for t in range(p, p + n):
            if t % 16 == 0:
                tables[r, t // 16] = free[taken] if taken < len(free) else -1
                taken += 1
            b = int(tables[r, t // 16])
            positions.append(t)
            slots.append(b * 16 + t % 16 if b >= 0 else -1)
        starts.append(starts[-1] + n)
        ctx.append(p + n)
    pad = [-1] * max(0, N - len(positions))
    return tables, starts, ctx, (positions + pad)[:N], (slots + pad)[:N], taken


def pool(rng, ctx, extra=3, width=None):
    """A permuted pool for requests of ctx tokens: (tables [R, width] int32 numpy, nb)."""
    need = [-(-c // 16) for c in ctx]
    W = width or max(1, max(need))
    nb = sum(need) + extra
    ids = rng.permutation(nb).astype(np.int32)
    tables, at = np.full((len(ctx), W), -1, np.int32), 0
    for r, n in enumerate(need):
        tables[r, :n] = ids[at:at + n]
        at += n
    return tables, nb


def attention(q, ck, cv, tables, new, ctx, window, sinks, scale):
    """(out, bound) [N, Hq, D] in 64 bits, request by request.

    The kernel's products of bf16 are exact; a score of D terms is off by D 2^-24 times
    the sum of their magnitudes (scaled), and so, relatively, is its weight e^score;
    the weights' sum by n 2^-24; a weight is rounded to bf16 once (2^-8); exp2 and its
    argument give less than 2^-18 together, the factors of a join of splits as much
    again. Each of these shifts out by that share of A = sum p |v|; the result is
    rounded to bf16 once (2^-8 of itself, and 2^-134 where it is subnormal)."""
    N, Hq, D = q.shape
    nb, H = ck.shape[:2]
    G, dev = Hq // H, q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    bound, at = torch.zeros_like(out), 0
    for r, (n, c) in enumerate(zip(new, ctx)):
        if n == 0 or c == 0:              # nothing asks, or nothing is there to be seen: zeros
            at += n
            continue
        held = min(-(-c // 16), tables.shape[1])
        ids = [int(i) if 0 <= i < nb else -1 for i in tables[r, :held]]
        t = torch.arange(16 * held, device=dev)
        there = torch.tensor(ids, dtype=torch.int64, device=dev).repeat_interleave(16) >= 0
        idx = torch.tensor([max(i, 0) for i in ids], dtype=torch.int64, device=dev)
        k = k_block_rows(ck[idx]).permute(1, 0, 2, 3).reshape(H, -1, D).double()
        v = cv[idx].permute(1, 0, 3, 2).reshape(H, -1, D).double()
        p = torch.arange(c - n, c, device=dev)[:, None]
        seen = (t <= p) & there
        if window:
            seen = seen & ((t > p - window) | (t < sinks))
        k = torch.where(torch.isfinite(k), k, 0.0)                   # only hidden ones, in these tests
        qr = q[at:at + n].double().view(n, H, G, D).permute(1, 2, 0, 3).reshape(H, G * n, D)
        kt = k.transpose(1, 2).contiguous()
        s = (torch.matmul(qr, kt) * scale).view(H, G, n, -1).masked_fill(~seen, -torch.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
        mass = (torch.matmul(qr.abs(), kt.abs()) * scale).view(H, G, n, -1).masked_fill(~seen, 0.0).amax(-1)
        # A value that is not finite reaches the rows that see it and no other.
        fine = torch.where(torch.isfinite(v), v, 0.0)
        o = torch.matmul(w.view(H, G * n, -1), fine).view(H, G, n, D)
        A = torch.matmul(w.view(H, G * n, -1), fine.abs()).view(H, G, n, D)
        odd = torch.where(torch.isfinite(v), 0.0, v)
        for h, j in {(int(h), int(j)) for h, j in (odd != 0).any(2).nonzero().tolist()}:
            o[h] += torch.where(seen[:, j][None, :, None], odd[h, j], 0.0)
        share = 2 * (D * 2.0 ** -24 * mass + seen.sum(-1) * 2.0 ** -24) + 2.0 ** -17 + 2.0 ** -8
        b = (1 + 2.0 ** -8) * share[..., None] * A + 2.0 ** -8 * o.abs() + 2.0 ** -134
        out[at:at + n] = o.permute(2, 0, 1, 3).reshape(n, Hq, D)
        bound[at:at + n] = b.permute(2, 0, 1, 3).reshape(n, Hq, D)
        at += n
    return out, bound


def rope(x, positions, inv):
    """(y, bound): x [N, heads, 128] turned. The angle's rounding and its cosine and sine
    come to less than 2^-21 of a dim's pair, the two products to 2^-23; y is rounded to
    bf16 once."""
    x = x.double()
    ang = positions.clamp(min=0).double()[:, None] * inv.double()
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b = x[..., :64], x[..., 64:]
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    size = (a.abs() + b.abs()).repeat(1, 1, 2)
    return y, (1 + 2.0 ** -8) * 2.0 ** -20 * size + 2.0 ** -8 * y.abs() + 2.0 ** -134


def e4m3_bound(y, scale, rel):
    """How far an e4m3 value times its scale may be from y, itself known to ``rel``: half
    a step (2^-4 of it, 2^-10 of the scale among the subnormals)."""
    return (2.0 ** -4 * (1 + rel) + rel + 2.0 ** -22) * y.abs() + 2.0 ** -10 * scale


def within(got, want, bound, what=""):
    got, want, bound = got.double(), want.double(), bound.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), what
    off = torch.where(odd, -1.0, (got - want).abs() - bound)
    worst = float(off.max()) if off.numel() else -1.0
    at = np.unravel_index(int(off.argmax()), tuple(off.shape)) if off.numel() else ()
    assert worst <= 0, (what, worst, at, float(got[at]), float(want[at]), float(bound[at]))
