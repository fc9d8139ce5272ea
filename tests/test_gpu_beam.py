"""Beam selection and reordering, and copies of cache blocks, against their
definitions (64 bits on the CPU, and plain indexing)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def select_reference(logits, scores, n, eos=None, last=None):
    """tokens, parents [R, n] and the totals in 64 bits, by sorting everything."""
    R, K = scores.shape
    x = logits.detach().cpu().double().reshape(R, K, -1).numpy()
    s = scores.detach().cpu().double().numpy()
    V = x.shape[2]
    tokens, parents = np.full((R, n), -1, np.int32), np.full((R, n), -1, np.int32)
    totals = np.full((R, n), -np.inf)
    for r in range(R):
        found = []
        for k in range(K):
            if not np.isfinite(s[r, k]):
                continue
            if eos is not None and int(last.reshape(R, K)[r, k]) == eos:
                found.append((-s[r, k], k, 0.0, eos))
                continue
            row = x[r, k]
            if np.isnan(row).any() or not row.max() > -np.inf or row.max() == np.inf:
                continue
            # The maximum apart from the sum's logarithm, which it would swallow
            # where it is the type's lowest value.
            log_sum = math.log(math.fsum(np.exp(row - row.max())))
            order = np.lexsort((np.arange(V), -row))[:n]
            found += [(-(s[r, k] + ((row[t] - row.max()) - log_sum)), k, -row[t], int(t)) for t in order
                      if row[t] > -np.inf]
        found.sort()
        for i, (t, k, _, tok) in enumerate(found[:n]):
            tokens[r, i], parents[r, i], totals[r, i] = tok, k, -t
    return tokens, parents, totals


def check_select(logits, scores, n, eos=None, last=None, **kw):
    from rngd_pd_amd import kernels as K
    got = K.beam_select(logits, scores, n, eos=eos, last_tokens=last, **kw)
    torch.cuda.synchronize()
    want = select_reference(logits, scores, n, eos, None if last is None else last.cpu())
    np.testing.assert_array_equal(got[0].cpu().numpy(), want[0])
    np.testing.assert_array_equal(got[1].cpu().numpy(), want[1])
    have = got[2].cpu().double().numpy()
    none = np.isinf(want[2])
    assert (have[none] == -np.inf).all()
    # A total is rounded to 32 bits once; its 64-bit sums are off by less than 1e-9.
    off = np.abs(have[~none] - want[2][~none])
    assert (off <= 2.0 ** -24 * np.abs(want[2][~none]) + 1e-9).all()
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("R,K,V,n", [
    (1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 17, 6), (1, 4, 1000, 8), (3, 2, 4095, 2), (2, 2, 4096, 4),
    (2, 2, 4097, 4), (1, 16, 8191, 32), (5, 5, 12345, 10), (1, 4, 128256, 8), (2, 16, 32000, 16),
    (1, 3, 262145, 32), (1, 1, 1 << 20, 32)])
def test_select(cuda, dtype, R, K, V, n):
    print(f"select {dtype} R={R} K={K} V={V} n={n}", flush=True)
    g = torch.Generator(device=cuda).manual_seed(V + K)
    x = (torch.randn((R * K, V), generator=g, device=cuda) * 2.5).to(dtype)
    scores = -20 * torch.rand((R, K), generator=g, device=cuda)
    check_select(x, scores, n)
    last = torch.randint(0, 3, (R, K), generator=g, device=cuda, dtype=torch.int32)
    check_select(x, scores, n, eos=1, last=last)


@pytest.mark.parametrize("dtype,R,K,V,n", [
    (torch.bfloat16, 16, 16, 40001, 8), (torch.float32, 16, 16, 40001, 8),
    (torch.float32, 60, 16, 18433, 16), (torch.bfloat16, 75, 16, 20483, 32),
    (torch.bfloat16, 230, 16, 14403, 4)])
def test_select_many_rows(cuda, dtype, R, K, V, n):
    """Rows enough for several steps of a wavefront, with rows of every kind among
    them: ties, sorted ones, values masked, far from zero, infinite or NaN."""
    print(f"select {dtype} R={R} K={K} V={V} n={n}", flush=True)
    inf = float("inf")
    g = torch.Generator(device=cuda).manual_seed(V + K)
    x = torch.randn((R * K, V), generator=g, device=cuda) * 2.5
    i = torch.arange(V, device=cuda).float()
    x[1::29] = 0.25
    x[2::29] = i / 512
    x[3::29] = -i / 512
    x[4::29] = i % 5
    x[5::29, ::2] = -inf
    x[6::29] = -inf
    x[7::29, :-1] = -inf
    x[8::29, V // 2] = float("nan")
    x[9::29, -1] = inf
    x[10::29] += 1e5
    x[11::29] -= 3e4
    x[12::29] = torch.where(i < 40, 0.0, torch.finfo(dtype).min)
    x[13::29] *= 1e36
    x[14::29] = torch.where(i >= V - 3, 5000.0 + i - V, 4990.0)
    x[15::29, : V - 5] = torch.finfo(dtype).min
    scores = -20 * torch.rand((R, K), generator=g, device=cuda)
    x = x.to(dtype)
    check_select(x, scores, n)
    # From odd addresses, and with beams that have ended.
    wide = torch.empty((R * K, V + 1), dtype=dtype, device=cuda)
    wide[:, 1:] = x
    last = torch.randint(0, 3, (R, K), generator=g, device=cuda, dtype=torch.int32)
    check_select(wide[:, 1:], scores, n, eos=1, last=last)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_select_ties_and_order(cuda, dtype):
    """Equal logits everywhere, few distinct values, sorted rows, equal beams."""
    V, K, n = 9001, 4, 24
    scores = torch.tensor([[-1.0, -3.0, -1.0, -2.0]], device=cuda)
    flat = torch.full((K, V), 1.5, device=cuda).to(dtype)
    check_select(flat, scores, n)
    i = torch.arange(V, device=cuda)
    check_select((i % 7).to(dtype).expand(K, V).contiguous(), scores, n)
    check_select((i.float() / 64).to(dtype).expand(K, V).contiguous(), scores, n)
    check_select((-i.float() / 64).to(dtype).expand(K, V).contiguous(), scores, n)
    check_select(flat, torch.zeros((1, K), device=cuda), 32)
    # Beams equal in all but where their rows lie (odd V: every alignment).
    row = torch.randn(V, device=cuda).to(dtype)
    check_select(row.expand(K, V).contiguous(), torch.full((1, K), -5.0, device=cuda), 16)
    # +0 and -0 are one value: the lower token first.
    z = torch.zeros((K, 64), device=cuda).to(dtype)
    z[:, ::2] = -0.0
    check_select(z, scores, n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_select_masks_and_dead_beams(cuda, dtype):
    inf, nan = float("inf"), float("nan")
    V, K, n = 5000, 5, 10
    g = torch.Generator(device=cuda).manual_seed(5)
    x = torch.randn((K, V), generator=g, device=cuda) * 3
    x[0, 3:] = -inf                                   # three tokens allowed
    x[1] = -inf                                       # none
    x[2, 4500] = nan
    x[3, 17] = inf
    x[4, torch.rand(V, generator=g, device=cuda) < 0.999] = -inf
    scores = torch.tensor([[-1.0, 0.0, 0.0, 0.0, -50.0]], device=cuda)
    check_select(x.to(dtype), scores, n)
    low = torch.finfo(dtype).min
    y = torch.full((K, V), low, device=cuda).to(dtype)
    y[:, 7] = 2.0
    y[1] = low                                        # all at the lowest value: all alike
    check_select(y, torch.zeros((1, K), device=cuda), n)
    for bad in (-inf, inf, nan):
        s = torch.tensor([[bad, -1.0, bad, -2.0, bad]], device=cuda)
        z = torch.randn((K, V), generator=g, device=cuda).to(dtype)
        check_select(z, s, n)
        check_select(z, torch.full((1, K), bad, device=cuda), n)
    # Beams that ended: one candidate each, logits unread (NaN there).
    z = torch.randn((K, V), generator=g, device=cuda).to(dtype)
    z[1] = nan
    last = torch.tensor([[5, 9, 5, 9, 9]], dtype=torch.int32, device=cuda)
    check_select(z, torch.tensor([[-4.0, -1.0, -2.0, -inf, -9.0]], device=cuda), n, eos=9, last=last)
    check_select(z, torch.zeros((1, K), device=cuda), n, eos=9, last=torch.full_like(last, 9))
    # Large scores of either sign.
    check_select(x.to(dtype)[4:].expand(K, V).contiguous(),
                 torch.tensor([[-1e4, 1e4, 0.0, -1e30, 3.0]], device=cuda), n)


def test_select_near_ties_across_beams(cuda):
    """Totals of two beams that 32 bits cannot tell apart."""
    V = 50000
    g = torch.Generator(device=cuda).manual_seed(6)
    x = torch.randn((2, V), generator=g, device=cuda) * 2
    lse = torch.logsumexp(x.double(), -1)
    for step in (-3e-9, 3e-9):
        s0 = -3.0
        # Shift one logit of beam 1 so that its total lies `step` from beam 0's best.
        best = x[0].max().double()
        y = x.clone()
        want = best - lse[0] + lse[1]
        y[1, 77] = want.float()
        l1 = torch.logsumexp(y[1].double(), 0)
        s1 = (s0 + best - lse[0] + step) - (y[1, 77].double() - l1)
        scores = torch.tensor([[s0, float(s1)]], device=cuda)
        check_select(y, scores, 8)


def test_select_strides_outputs_streams_and_graphs(cuda):
    from rngd_pd_amd import kernels as K
    g = torch.Generator(device=cuda).manual_seed(8)
    R, B, V, n = 3, 4, 7001, 6
    wide = torch.randn((R * B, V + 13), generator=g, device=cuda).to(torch.bfloat16)
    scores = -torch.rand((R, B), generator=g, device=cuda)
    want = check_select(wide[:, 5:5 + V], scores, n)
    out = tuple(torch.full_like(t, 77) for t in want)
    ws = torch.full((K.beam_select_workspace_bytes(R, B, V, n),), 255, dtype=torch.uint8, device=cuda)
    K.beam_select(wide[:, 5:5 + V], scores, n, out=out, workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = K.beam_select(wide[:, 5:5 + V], scores, n, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(K.beam_select(wide[:, 5:5 + V], scores, n))
        graphs.append(gr)
    for _ in range(3):
        wide.normal_()
        want = K.beam_select(wide[:, 5:5 + V], scores, n)
        for gr, o in zip(graphs, outs):
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(o, want))


def _caches(cuda, L, nb, H, D, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    mk = lambda *s: torch.randint(-2 ** 15, 2 ** 15, s, generator=g, device=cuda,  # noqa: E731
                                  dtype=torch.int16).view(torch.bfloat16)
    return mk(L, nb, H, 16, D), mk(L, nb, H, D, 16)


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))


@pytest.mark.parametrize("L,H,D,n", [(1, 1, 32, 1), (2, 8, 128, 3), (32, 8, 128, 5), (3, 5, 64, 40),
                                     (2, 1, 128, 449), (1, 2, 96, 1000)])
def test_copy_blocks(cuda, L, H, D, n):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(n)
    nb = 2 * n + 9
    ck, cv = _caches(cuda, L, nb, H, D)
    k0, v0 = ck.clone(), cv.clone()
    ids = rng.permutation(nb)
    dst, src = ids[:n], rng.choice(ids[n:], n)                # sources repeat
    print(f"copy L={L} H={H} D={D} n={n}", flush=True)
    K.copy_blocks(ck, cv, src.tolist() if n < 9 else src, torch.from_numpy(dst) if n > 9 else dst)
    k0[:, dst], v0[:, dst] = k0[:, src], v0[:, src]
    assert _same(ck, k0) and _same(cv, v0)
    K.copy_blocks(ck[0], cv[0], [int(dst[0])], [int(ids[-1])])   # one layer
    k0[0, ids[-1]], v0[0, ids[-1]] = k0[0, dst[0]], v0[0, dst[0]]
    assert _same(ck, k0) and _same(cv, v0)
    K.copy_blocks(ck[::2], cv[::2], [], [])
    K.copy_blocks(ck[::2], cv[::2], [int(dst[0])], [int(ids[n])])  # every other layer
    k0[::2, ids[n]], v0[::2, ids[n]] = k0[::2, dst[0]], v0[::2, dst[0]]
    assert _same(ck, k0) and _same(cv, v0)


def test_copy_blocks_captured(cuda):
    from rngd_pd_amd import kernels as K
    ck, cv = _caches(cuda, 2, 9, 2, 64)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.copy_blocks(ck, cv, [1, 1, 5], [2, 3, 0])
    for i in range(3):
        k0, v0 = _caches(cuda, 2, 9, 2, 64, seed=i + 1)
        ck.copy_(k0)
        cv.copy_(v0)
        g.replay()
        torch.cuda.synchronize()
        k0[:, [2, 3, 0]], v0[:, [2, 3, 0]] = k0[:, [1, 1, 5]], v0[:, [1, 1, 5]]
        assert _same(ck, k0) and _same(cv, v0)


@pytest.mark.parametrize("R,B,L,H,D,ctx,width", [
    (1, 1, 1, 1, 32, [5], 1), (1, 4, 2, 8, 128, [603], 39), (3, 2, 2, 2, 64, [1, 16, 17], 2),
    (2, 16, 3, 1, 128, [320, 333], 22), (4, 3, 2, 8, 128, [0, 47, 48, 5000], 4),
    (2, 5, 32, 8, 128, [15, 31], 3)])
def test_reorder(cuda, R, B, L, H, D, ctx, width):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(R * 7 + B)
    nb = R * B * 2 + 6
    for case in range(4):
        ck, cv = _caches(cuda, L, nb, H, D, seed=case)
        tables = rng.integers(-1, nb + 1, (R, B, width)).astype(np.int32)
        mine = rng.permutation(nb)[:R * B].reshape(R, B)
        parents = rng.integers(0, B, (R, B)).astype(np.int32)
        if case == 1:
            parents = np.tile(np.roll(np.arange(B), 1), (R, 1)).astype(np.int32)   # all move round
        if case == 2:
            parents[:] = rng.integers(-2, B + 2, (R, B))           # some without a parent
        want_t, k0, v0 = tables.copy(), ck.clone(), cv.clone()
        for r, c in enumerate(ctx):
            f = c // 16
            if f < width:
                tables[r, :, f] = mine[r]
                if case == 3 and B > 1:
                    tables[r, 0, f] = -1                           # an invalid block: neither way
            want_t[r] = tables[r]
            if c <= 0:
                continue
            for j in range(B):
                p = parents[r, j]
                if not 0 <= p < B or p == j:
                    continue
                want_t[r, j, :f] = tables[r, p, :f]
                if f < width and c % 16 and tables[r, p, f] >= 0 and tables[r, j, f] >= 0:
                    k0[:, tables[r, j, f]] = ck[:, tables[r, p, f]]
                    v0[:, tables[r, j, f]] = cv[:, tables[r, p, f]]
        tab = torch.from_numpy(tables.reshape(R * B, width).copy()).to(cuda)
        print(f"reorder R={R} K={B} L={L} ctx={ctx} case {case}", flush=True)
        K.beam_reorder(torch.from_numpy(parents).to(cuda),
                       torch.tensor([c for c in ctx for _ in range(B)], dtype=torch.int32,
                                    device=cuda), tab, ck, cv)
        np.testing.assert_array_equal(tab.cpu().numpy().reshape(R, B, width), want_t)
        assert _same(ck, k0) and _same(cv, v0)


def test_refusals(cuda):
    from rngd_pd_amd import kernels as K
    from rngd_pd_amd._lib import PdkError
    ck, cv = _caches(cuda, 2, 9, 2, 64)
    k0 = ck.clone()
    for src, dst in (([1, 2], [3, 3]), ([1, 3], [3, 4]), ([1], [1]), ([-1], [2]), ([1], [9])):
        with pytest.raises((PdkError, ValueError)):
            K.copy_blocks(ck, cv, src, dst)
        with pytest.raises(PdkError):
            K.copy_blocks(ck, cv, np.array(src, np.int32), np.array(dst, np.int32))
    with pytest.raises(ValueError):
        K.copy_blocks(ck, cv, [1, 2], [3])
    with pytest.raises(TypeError):
        K.copy_blocks(ck, cv, torch.tensor([1], device=cuda), [3])
    with pytest.raises(TypeError):
        K.copy_blocks(ck, cv, [1.5], [3])
    with pytest.raises(ValueError):
        K.copy_blocks(ck, cv[:, :5], [1], [3])
    with pytest.raises(ValueError):
        K.copy_blocks(ck[:, :5], cv[:, :5].transpose(0, 1), [1], [3])
    assert _same(ck, k0)
    x, s = torch.zeros((4, 100), device=cuda), torch.zeros((1, 4), device=cuda)
    last = torch.zeros((1, 4), dtype=torch.int32, device=cuda)
    for bad in (lambda: K.beam_select(x[:3], s), lambda: K.beam_select(x, s, 33),
                lambda: K.beam_select(x, s, 0), lambda: K.beam_select(x.t(), s[:, :1]),
                lambda: K.beam_select(x, s, eos=3), lambda: K.beam_select(x, s, last_tokens=last),
                lambda: K.beam_select(x, s, eos=1 << 31, last_tokens=last),
                lambda: K.beam_select(torch.zeros((17, 9), device=cuda), torch.zeros((1, 17), device=cuda)),
                lambda: K.beam_select(x, s, 4, out=(last[:, :2], last, s)),
                lambda: K.beam_select(x, torch.zeros((1, 8), device=cuda)[:, ::2]),
                lambda: K.beam_select(x, s, workspace=torch.zeros(8, device=cuda)),
                lambda: K.beam_select(x[:, :0], s)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: K.beam_select(x.half(), s), lambda: K.beam_select(x, s.double()),
                lambda: K.beam_select(x.cpu(), s), lambda: K.beam_select(x, s, eos=1, last_tokens=last.long())):
        with pytest.raises(TypeError):
            bad()
    tab = torch.zeros((4, 3), dtype=torch.int32, device=cuda)
    ctx = torch.zeros(4, dtype=torch.int32, device=cuda)
    for bad in (lambda: K.beam_reorder(last, ctx, tab[:3], ck, cv),
                lambda: K.beam_reorder(last, ctx[:3], tab, ck, cv),
                lambda: K.beam_reorder(last, ctx, tab.t(), ck, cv),
                lambda: K.beam_reorder(last[0], ctx, tab, ck, cv),
                lambda: K.beam_reorder(last, ctx.cpu().to(cuda), tab, ck, cv[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(PdkError):
        z = torch.zeros((1, 17), dtype=torch.int32, device=cuda)
        K.beam_reorder(z, z[0], torch.zeros((17, 2), dtype=torch.int32, device=cuda), ck, cv)
