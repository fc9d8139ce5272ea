"""A step's map, cache write and attention over several requests' new tokens, against
64 bits."""
import math

import numpy as np
import pytest
import torch

from tests import _chunk_ref as ref
from tests._util import rand_bf16, to_dev

pytestmark = pytest.mark.gpu
D, SCALE = 128, 1.0 / math.sqrt(128)


def _int32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# ---- the map --------------------------------------------------------------------
MAPS = [
    # past, new, width, free blocks short of the need, max_tokens beyond the sum
    ([0], [1], 1, 0, 0),
    ([15, 16, 17, 0], [1, 1, 1, 1], 3, 0, 0),
    ([5, 0, 31, 160], [40, 0, 1, 33], 16, 0, 9),
    ([0, 0, 0], [0, 0, 0], 4, 0, 5),                      # nothing new at all
    ([7, 0, 200], [100, 300, 17], 32, 5, 3),              # the list runs out
    ([3, 3], [50, 50], 8, 99, 0),                         # no free block at all
    ([0, 30], [64, 40], 8, 0, -20),                       # fewer places than tokens
    ([-4, 100, 1 << 30], [3, -2, 5], 7, 0, 4),            # lengths out of range
    ([(7 * i) % 90 for i in range(300)], [i % 5 for i in range(300)], 12, 0, 1),
    ([i % 40 for i in range(4096)], [1] * 4096, 4, 3, 0),  # the most requests
]


@pytest.mark.parametrize("past,new,width,short,spare", MAPS)
def test_map(cuda, past, new, width, short, spare):
    from rngd_pd_amd import kernels as K
    print(f"map R={len(past)} width={width} short={short} spare={spare}", flush=True)
    rng, R = np.random.default_rng(len(past) + width), len(past)
    real = [(min(max(p, 0), 16 * width), n) for p, n in zip(past, new)]
    real = [(p, min(max(n, 0), 16 * width - p)) for p, n in real]
    held = [-(-p // 16) for p, _ in real]
    need = sum(-(-(p + n) // 16) for p, n in real) - sum(held)
    N = sum(n for _, n in real) + spare
    ids = rng.permutation(sum(held) + need + 4).astype(np.int32)
    tables, at = np.full((R, width), -1, np.int32), 0
    for r, h in enumerate(held):
        tables[r, :h] = ids[at:at + h]
        at += h
    tables[:, -1] = np.where(tables[:, -1] < 0, -7, tables[:, -1])       # unused entries stay
    free = ids[at:at + max(0, need - short)]
    got_tables = torch.from_numpy(tables).to(cuda)
    m = K.chunk_map(_int32(past, cuda), _int32(new, cuda), got_tables,
                    torch.from_numpy(free).to(cuda), N)
    want = ref.chunk_map(past, new, tables, free, N)
    for name, g, w in zip(("tables", "starts", "ctx", "positions", "slots"),
                          (got_tables, m.starts, m.ctx_lens, m.positions, m.slots), want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w, np.int32).reshape(g.shape)), name
    assert m.taken.tolist() == [want[5]]


# ---- the write ------------------------------------------------------------------
@pytest.mark.parametrize("N,Hq,Hkv,first,kind", [
    (1, 32, 8, 0, "run"), (16, 32, 8, 5, "run"), (37, 28, 4, 100, "run"), (64, 8, 8, 16000, "any"),
    (100, 5, 1, 999_983, "any"), (250, 40, 8, 3, "run"), (33, 6, 3, 12, "some"), (9, 32, 8, -4, "some"),
    (2000, 32, 8, 131_000, "run"), (24, 128, 16, 0, "run"),
    (1100, 6, 3, 7, "any"), (1500, 5, 5, 3, "some"), (300, 8, 2, 40, "pieces"), (1333, 12, 12, 0, "pieces"),
    (5000, 32, 2, 9, "pieces"),           # a q past 32 MB
])
def test_write(cuda, N, Hq, Hkv, first, kind):
    from rngd_pd_amd import kernels as K
    from rngd_pd_amd.engines.paged_cache import k_block_rows
    print(f"write N={N} Hq={Hq} Hkv={Hkv} first={first} {kind}", flush=True)
    rng = np.random.default_rng(N + Hq)
    nb = N // 16 + 4
    if kind == "pieces":                  # of any length, each from somewhere in a block on
        lens = rng.integers(1, 30, N)
        nb = int(sum(-(-(n + 15) // 16) for n in lens)) + 4
        ids, at, slots = rng.permutation(nb), 0, []
        for n in lens:
            piece = (ids[at:at + -(-(n + 15) // 16), None] * 16 + np.arange(16)).reshape(-1)
            slots.append(piece[(off := int(rng.integers(16))):off + n])
            at += -(-(n + 15) // 16)
        slots = np.concatenate(slots)[:N]
    else:
        slots = rng.permutation(nb * 16)[:N]
    if kind == "run":                     # blocks one after another, from the middle of one
        slots = (rng.permutation(nb)[:, None] * 16 + np.arange(16)).reshape(-1)[3:3 + N]
    if kind == "some":                    # some tokens have no place, or one outside the cache
        slots[::3] = -1
        slots[1::5] = nb * 16 + 5
    slots = slots.astype(np.int32)
    wide = to_dev(rand_bf16(rng, (N, (Hq + 2 * Hkv) * D + 24)))
    qkv = wide[:, :(Hq + 2 * Hkv) * D]
    ck, cv = (to_dev(rand_bf16(rng, s)) for s in ((nb, Hkv, 16, D), (nb, Hkv, D, 16)))
    old_k, old_v = k_block_rows(ck).clone(), cv.clone()
    inv = torch.tensor([500000.0 ** (-2 * i / D) for i in range(64)], device=cuda)
    pos = torch.arange(first, first + N, dtype=torch.int32, device=cuda)
    q = K.rope_cache_write(qkv, inv, pos, torch.from_numpy(slots).to(cuda), ck, cv, Hq)
    x = qkv.reshape(N, Hq + 2 * Hkv, D)
    y, bound = ref.rope(x[:, :Hq + Hkv], pos, inv)
    ref.within(q, y[:, :Hq], bound[:, :Hq], "q")
    k = k_block_rows(ck)
    at = np.flatnonzero((slots >= 0) & (slots < nb * 16))
    b, s = (torch.from_numpy(v[at]).long().to(cuda) for v in (slots // 16, slots % 16))
    at = torch.from_numpy(at).to(cuda)
    ref.within(k[b, :, s], y[at, Hq:], bound[at, Hq:], "k")
    assert torch.equal(cv[b, :, :, s], x[at, Hq + Hkv:])
    # Every other place of the cache is as it was.
    k[b, :, s] = old_k[b, :, s]
    cv[b, :, :, s] = old_v[b, :, :, s]
    assert torch.equal(k, old_k) and torch.equal(cv, old_v)


# ---- the attention ----------------------------------------------------------------
ATTENTION = [
    # Hq, Hkv, [(in the cache before, new)], window, sinks
    (32, 8, [(0, 1)], 0, 0),
    (32, 8, [(15, 1), (16, 1), (0, 1), (500, 1)], 0, 0),
    (32, 8, [(31, 2), (0, 8), (100, 7), (9, 0), (4000, 3)], 0, 0),        # drafts
    (32, 8, [(0, 33)], 0, 0),
    (32, 8, [(0, 300)], 0, 0),
    (32, 8, [(1000, 200), (3, 1), (0, 9), (70, 100), (600, 1), (5, 0)], 0, 0),   # all kinds together
    (32, 8, [(3000, 130)], 0, 0),                                           # a split context
    (8, 8, [(17, 40), (200, 32), (33, 33)], 0, 0),                          # no groups
    (28, 4, [(77, 19), (300, 4), (5, 5)], 0, 0),                            # 7 heads to a group
    (40, 8, [(129, 31), (64, 6), (0, 7)], 0, 0),
    (13, 1, [(250, 50), (90, 2)], 0, 0),
    (16, 1, [(600, 40), (31, 2), (32, 3)], 0, 0),
    (4, 2, [(3 * i, 1 + i % 20) for i in range(70)], 0, 0),                 # more than 64 requests
    (32, 8, [(40, 20), (300, 1), (200, 5), (0, 90)], 16, 0),
    (32, 8, [(700, 100), (33, 1), (513, 3), (0, 40)], 64, 4),
    (8, 2, [(0, 200), (1000, 3), (900, 64)], 33, 33),
    (32, 8, [(2000, 100), (2000, 1)], 1000, 17),
    (16, 8, [(90, 30), (50, 1)], 1, 0),
]


def _operands(rng, Hq, Hkv, lens, width=None):
    ctx = [p + n for p, n in lens]
    tables, nb = ref.pool(rng, ctx, width=width)
    N = sum(n for _, n in lens)
    return (to_dev(rand_bf16(rng, (N, Hq, D))), to_dev(rand_bf16(rng, (nb, Hkv, 16, D))),
            to_dev(rand_bf16(rng, (nb, Hkv, D, 16))), tables, ctx)


def _starts(lens):
    return [sum(n for _, n in lens[:r]) for r in range(len(lens) + 1)]


def _attend(q, ck, cv, tables, lens, window=0, sinks=0, out=None, max_new=None, max_ctx=None, **kw):
    from rngd_pd_amd import kernels as K
    span = {"window": window, "sinks": sinks} if window else {}
    return K.chunk_attention(q, ck, cv, torch.from_numpy(tables).to(q.device),
                             _int32(_starts(lens), q.device), _int32([p + n for p, n in lens], q.device),
                             max_new or max(n for _, n in lens), max_ctx or max(p + n for p, n in lens),
                             scale=SCALE, out=out, **span, **kw)


@pytest.mark.parametrize("Hq,Hkv,lens,window,sinks", ATTENTION)
def test_attention(cuda, Hq, Hkv, lens, window, sinks):
    print(f"chunk attention Hq={Hq} Hkv={Hkv} lens={lens[:6]} window={window} sinks={sinks}", flush=True)
    rng = np.random.default_rng(Hq + len(lens) + window)
    q, ck, cv, tables, ctx = _operands(rng, Hq, Hkv, lens)
    want, bound = ref.attention(q, ck, cv, tables, [n for _, n in lens], ctx, window, sinks, SCALE)
    got = _attend(q, ck, cv, tables, lens, window, sinks)
    ref.within(got, want, bound, "plain")
    assert torch.equal(got, _attend(q, ck, cv, tables, lens, window, sinks)), "twice"
    # Bounds larger than the lengths plan other splits; q as columns of a wider tensor.
    wide = np.full((len(lens), tables.shape[1] + 300), -1, np.int32)
    wide[:, :tables.shape[1]] = tables
    cols = torch.zeros((q.shape[0], Hq + 3, D), dtype=q.dtype, device=cuda)
    cols[:, 1:Hq + 1] = q
    got = _attend(cols[:, 1:Hq + 1], ck, cv, wide, lens, window, sinks, max_new=5000,
                  max_ctx=wide.shape[1] * 16)
    ref.within(got, want, bound, "wide")


@pytest.mark.parametrize("Hq,Hkv,lens", [
    (32, 8, [(40, 3), (100, 1), (7, 2)]),
    (32, 8, [(40, 50), (100, 1), (0, 2)]),
    (8, 8, [(700, 64), (20, 40)]),
])
def test_blocks_that_are_missing(cuda, Hq, Hkv, lens):
    """Entries of -1 or outside the cache hide their tokens; a row without any is zero."""
    print(f"missing blocks {lens}", flush=True)
    rng = np.random.default_rng(len(lens))
    q, ck, cv, tables, ctx = _operands(rng, Hq, Hkv, lens)
    tables[0, 1] = -1
    tables[0, 0] = ck.shape[0] + 3
    tables[-1, :] = -1
    want, bound = ref.attention(q, ck, cv, tables, [n for _, n in lens], ctx, 0, 0, SCALE)
    got = _attend(q, ck, cv, tables, lens)
    assert not got[_starts(lens)[-2]:].any()
    ref.within(got, want, bound)


@pytest.mark.parametrize("lens", [[(30, 4), (17, 1)], [(30, 70), (17, 1)], [(2000, 40)], [(2000, 3)]])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
def test_hidden_values_that_are_not_finite(cuda, lens, odd):
    """What stands behind a request's last token, in other blocks and in tokens that a row
    does not see reaches no row; in a token that is seen it does."""
    print(f"not finite {lens} {odd}", flush=True)
    from rngd_pd_amd.engines.paged_cache import k_block_index
    rng = np.random.default_rng(7)
    Hq, Hkv = 8, 2
    q, ck, cv, tables, ctx = _operands(rng, Hq, Hkv, lens)
    place = k_block_index(D, cuda)
    used = torch.zeros(ck.shape[0], dtype=torch.bool, device=cuda)
    used[torch.from_numpy(tables[tables >= 0]).long().to(cuda)] = True
    ck[~used], cv[~used] = float("nan"), odd
    for r, c in enumerate(ctx):
        last = int(tables[r, (c - 1) // 16])
        for s in range((c - 1) % 16 + 1, 16):
            ck[last].view(Hkv, -1)[:, place[s]] = float("nan")
            cv[last, :, :, s] = odd
    clean, bound = ref.attention(q, ck, cv, tables, [n for _, n in lens], ctx, 0, 0, SCALE)
    assert torch.isfinite(clean).all()
    ref.within(_attend(q, ck, cv, tables, lens), clean, bound, "behind")
    # Two of the first request's new tokens (or old ones under a window).
    p, n = lens[0]
    for t, dims in ((p + n // 2, slice(0, D, 3)), (p + n - 1, slice(5, 70))):
        cv[int(tables[0, t // 16]), :, dims, t % 16] = odd
    want, bound = ref.attention(q, ck, cv, tables, [n for _, n in lens], ctx, 0, 0, SCALE)
    assert not torch.isfinite(want).all()
    got = _attend(q, ck, cv, tables, lens)
    ref.within(got, want, bound, "new")
    want, bound = ref.attention(q, ck, cv, tables, [n for _, n in lens], ctx, n // 2 + 1, 0, SCALE)
    ref.within(_attend(q, ck, cv, tables, lens, window=n // 2 + 1), want, bound, "window")


@pytest.mark.parametrize("past,new,window,sinks", [
    (3500, 256, 0, 0), (4000, 1000, 0, 0), (3500, 256, 1500, 100), (3490, 251, 1, 0), (0, 1000, 0, 0),
    (16001, 127, 0, 0)])
def test_one_request_shared_by_teams(cuda, past, new, window, sinks):
    """A request alone, its splits shared by teams of a workgroup: plain, with blocks missing
    and with values that are not finite hidden and seen."""
    print(f"one request {past} + {new} window={window}", flush=True)
    rng = np.random.default_rng(past + new)
    q, ck, cv, tables, ctx = _operands(rng, 32, 8, [(past, new)])
    check = lambda what: ref.within(                                         # noqa: E731
        _attend(q, ck, cv, tables, [(past, new)], window, sinks),
        *ref.attention(q, ck, cv, tables, [new], ctx, window, sinks, SCALE), what)
    check("plain")
    tables[0, 3:40:6] = -1
    tables[0, -1] = ck.shape[0]
    check("missing blocks")
    for t in range(past + 5, past + new, 61):
        if (b := int(tables[0, t // 16])) >= 0 and b < ck.shape[0]:
            cv[b, :, t % 7::9, t % 16] = (float("inf"), -float("inf"), float("nan"))[t % 3]
    check("not finite")


def test_rows_behind_the_last_request_stay(cuda):
    rng = np.random.default_rng(3)
    for lens in ([(100, 3), (20, 1)], [(100, 60), (20, 1)]):
        q, ck, cv, tables, ctx = _operands(rng, 32, 8, lens)
        N = q.shape[0]
        more = torch.cat([q, torch.full((9, 32, D), float("nan"), dtype=q.dtype, device=cuda)])
        out = torch.full_like(more, 7.0)
        assert _attend(more, ck, cv, tables, lens, out=out) is out
        assert (out[N:] == 7).all()
        assert torch.equal(out[:N], _attend(q, ck, cv, tables, lens))


@pytest.mark.parametrize("lens", [[(-60, 100)], [(-60, 100), (5, 1)], [(-3, 4), (9, 2)], [(-9, 9)]])
def test_contexts_shorter_than_the_new_tokens(cuda, lens):
    """Tokens at positions below 0 see nothing."""
    rng = np.random.default_rng(13)
    q, ck, cv, tables, ctx = _operands(rng, 32, 8, lens, width=4)
    want, bound = ref.attention(q, ck, cv, tables, [n for _, n in lens], ctx, 0, 0, SCALE)
    got = _attend(q, ck, cv, tables, lens, max_ctx=64)
    assert not got[:min(-lens[0][0], lens[0][1])].any()
    ref.within(got, want, bound)


def test_scores_far_apart(cuda):
    """Weights that underflow and maxima that grow along the context."""
    rng = np.random.default_rng(5)
    lens = [(900, 60), (333, 2)]
    q, ck, cv, tables, ctx = _operands(rng, 8, 2, lens)
    q, ck = q * 8, ck * 4
    want, bound = ref.attention(q, ck, cv, tables, [n for _, n in lens], ctx, 0, 0, SCALE)
    ref.within(_attend(q, ck, cv, tables, lens), want, bound)


def test_long_cache_offsets(cuda):
    """Blocks whose offsets pass 32 bits."""
    from rngd_pd_amd import kernels as K
    nb = (1 << 32) // (8 * 16 * D * 2) + 40                 # 32 KiB a block: past 4 GiB
    ck = torch.zeros((nb, 8, 16, D), dtype=torch.bfloat16, device=cuda)
    cv = torch.zeros((nb, 8, D, 16), dtype=torch.bfloat16, device=cuda)
    rng = np.random.default_rng(11)
    N, past = 40, 24
    qkv = to_dev(rand_bf16(rng, (N, 48 * D)))
    inv = torch.full((64,), 0.01, device=cuda)
    tables = torch.full((1, 8), -1, dtype=torch.int32, device=cuda)
    tables[0, :2] = _int32([nb - 1, 3], cuda)
    for b in (nb - 1, 3):
        ck[b].normal_()
        cv[b].normal_()
    m = K.chunk_map(_int32([past], cuda), _int32([N], cuda), tables, _int32([nb - 5, nb - 2, 9], cuda), N)
    q = K.rope_cache_write(qkv, inv, m.positions, m.slots, ck, cv, 32)
    for new in (N, 2):                                       # both kinds of request
        starts = _int32([0, new], cuda)
        got = K.chunk_attention(q[N - new:], ck, cv, tables, starts, m.ctx_lens, new, 64, scale=SCALE)
        want, bound = ref.attention(q[N - new:], ck, cv, tables.cpu().numpy(), [new], [64], 0, 0, SCALE)
        ref.within(got, want, bound)


@pytest.mark.parametrize("new", [1, 3, 20])
def test_long_contexts_beside_many_short_ones(cuda, new):
    """So many requests that none is split: a walk longer than the ids that a wavefront
    reads at a time."""
    lens = [(9000 - new, new), (16900, new)] + [(i % 23, 1) for i in range(140)] + [(8190, new)]
    print(f"long beside short, {new} new", flush=True)
    rng = np.random.default_rng(new)
    q, ck, cv, tables, ctx = _operands(rng, 16, 8, lens)
    tables[1, 510:530:3] = -1                                # missing about where ids are read anew
    tables[1, 770] = -1
    want, bound = ref.attention(q, ck, cv, tables, [n for _, n in lens], ctx, 0, 0, SCALE)
    ref.within(_attend(q, ck, cv, tables, lens), want, bound)


@pytest.mark.parametrize("new", [1544, 1400, 20])
def test_rows_left_over_of_a_round(cuda, new):
    """q with rows for just over a round of the card's workgroups, which are split, and a
    request that has them all or fewer; its workspace holds what is left over alone."""
    from rngd_pd_amd import kernels as K
    N, past, Hq, Hkv = 1544, 1000, 64, 4
    print(f"rows left over, {new} of {N} new", flush=True)
    rng = np.random.default_rng(new)
    q, ck, cv, tables, ctx = _operands(rng, Hq, Hkv, [(past, new)])
    want, bound = ref.attention(q, ck, cv, tables, [new], ctx, 0, 0, SCALE)
    more = torch.cat([q, torch.full((N - new, Hq, D), float("nan"), dtype=q.dtype, device=cuda)])
    out = torch.full_like(more, 7.0)
    need = K.chunk_workspace_bytes(N, 1, N, tables.shape[1] * 16, Hq, Hkv)
    assert need < 64 << 20
    ws = torch.full((need + 4096,), 85, dtype=torch.uint8, device=cuda)
    _attend(more, ck, cv, tables, [(past, new)], out=out, max_new=N, max_ctx=tables.shape[1] * 16,
            workspace=ws[:need])
    ref.within(out[:new], want, bound)
    assert (out[new:] == 7).all() and (ws[need:] == 85).all()


@pytest.mark.parametrize("R", [1, 2, 5, 64])
def test_workspaces_stay_small(R):
    """Whatever is left over, the splits' sums take at most some 277 MB."""
    from rngd_pd_amd import kernels as K
    for N in (40, 776, 3104, 6208, 6300, 8192, 70000):
        for Hq, Hkv in ((32, 8), (64, 4), (8, 8)):
            assert K.chunk_workspace_bytes(N, R, N, 1 << 19, Hq, Hkv) <= 300 << 20


def test_side_stream_and_own_workspace(cuda):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(9)
    lens = [(3000, 100), (2000, 1)]
    q, ck, cv, tables, ctx = _operands(rng, 32, 8, lens)
    want = _attend(q, ck, cv, tables, lens)
    need = K.chunk_workspace_bytes(q.shape[0], 2, 100, max(ctx), 32, 8)
    assert need > 0
    side = torch.cuda.Stream()
    ws = torch.empty(need, dtype=torch.uint8, device=cuda)
    torch.cuda.synchronize()
    got = _attend(q, ck, cv, tables, lens, workspace=ws, stream=side)
    handle = _attend(q, ck, cv, tables, lens, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(handle, want)
    with pytest.raises(ValueError, match="workspace"):
        _attend(q, ck, cv, tables, lens, workspace=ws[:need - 16])
    with pytest.raises(ValueError, match="overlap"):
        _attend(q, ck, cv, tables, lens, out=q)


def test_a_step_in_a_graph(cuda):
    """Map, write and attention captured once and replayed as the requests grow, with
    eager work in between."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(21)
    R, Hq, Hkv, W, N = 3, 8, 2, 64, 40
    nb = R * W
    ids = rng.permutation(nb).astype(np.int32)
    ck, cv = (torch.zeros(s, dtype=torch.bfloat16, device=cuda) for s in ((nb, Hkv, 16, D), (nb, Hkv, D, 16)))
    inv = torch.tensor([10000.0 ** (-2 * i / D) for i in range(64)], device=cuda)
    qkv = torch.zeros((N, (Hq + 2 * Hkv) * D), dtype=torch.bfloat16, device=cuda)
    past, new = _int32([0] * R, cuda), _int32([1] * R, cuda)
    tables = torch.full((R, W), -1, dtype=torch.int32, device=cuda)
    free = torch.from_numpy(ids).to(cuda)

    def step():
        m = K.chunk_map(past, new, tables, free, N)
        q = K.rope_cache_write(qkv, inv, m.positions, m.slots, ck, cv, Hq)
        return m, K.chunk_attention(q, ck, cv, tables, m.starts, m.ctx_lens, N, W * 16, scale=SCALE,
                                    out=torch.zeros_like(q))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        m, out = step()
    tables.fill_(-1)
    ck.zero_()
    cv.zero_()
    eager_k, eager_v, eager_tables = ck.clone(), cv.clone(), tables.clone()
    have, taken = [0] * R, 0
    for lens in ([20, 1, 7], [1, 1, 1], [5, 30, 0], [1, 2, 33]):
        qkv.copy_(to_dev(rand_bf16(rng, tuple(qkv.shape))))
        past.copy_(_int32(have, cuda))
        new.copy_(_int32(lens, cuda))
        free.copy_(torch.from_numpy(np.roll(ids, -taken)).to(cuda))
        graph.replay()
        torch.cuda.synchronize()
        em = K.chunk_map(past, new, eager_tables, free, N)
        q = K.rope_cache_write(qkv, inv, em.positions, em.slots, eager_k, eager_v, Hq)
        want = K.chunk_attention(q, eager_k, eager_v, eager_tables, em.starts, em.ctx_lens, N, W * 16,
                                 scale=SCALE, out=torch.zeros_like(q))
        assert torch.equal(out, want) and torch.equal(ck, eager_k) and torch.equal(cv, eager_v)
        assert torch.equal(tables, eager_tables) and torch.equal(m.slots, em.slots)
        have = [h + n for h, n in zip(have, lens)]
        taken += int(em.taken)


def test_refusals_of_the_wrappers(cuda):
    from rngd_pd_amd import kernels as K
    lens = [(20, 3), (5, 1)]
    q, ck, cv, tables, ctx = _operands(np.random.default_rng(0), 8, 2, lens)
    tab = torch.from_numpy(tables).to(cuda)
    past, new, free = (_int32(v, cuda) for v in ([20, 5], [3, 1], [1, 2]))
    starts, ctx_d = _int32(_starts(lens), cuda), _int32(ctx, cuda)
    inv = torch.ones(64, device=cuda)
    qkv = torch.zeros((4, 12 * D), dtype=torch.bfloat16, device=cuda)
    pos = _int32([20, 21, 22, 5], cuda)

    def attend(**kw):
        a = dict(q=q, ck=ck, cv=cv, tab=tab, starts=starts, ctx=ctx_d, new=3, max_ctx=23)
        more = {k: v for k, v in kw.items() if k not in a}
        a.update(kw)
        return K.chunk_attention(a["q"], a["ck"], a["cv"], a["tab"], a["starts"], a["ctx"], a["new"],
                                 a["max_ctx"], **more)

    for at, (exc, call) in enumerate((
            (TypeError, lambda: K.chunk_map(past.long(), new, tab, free, 4)),
            (TypeError, lambda: K.chunk_map(past, new, tab, free.cpu(), 4)),
            (ValueError, lambda: K.chunk_map(past[:1], new, tab, free, 4)),
            (ValueError, lambda: K.chunk_map(past, new, tab.t(), free, 4)),
            (ValueError, lambda: K.chunk_map(past, new, tab[0], free, 4)),
            (ValueError, lambda: K.chunk_map(past, new, tab, free, -1)),
            (ValueError, lambda: K.rope_cache_write(qkv[:, :11 * D], inv, pos, pos, ck, cv, 8)),
            (ValueError, lambda: K.rope_cache_write(qkv, inv[:32], pos, pos, ck, cv, 8)),
            (ValueError, lambda: K.rope_cache_write(qkv, inv, pos[:3], pos, ck, cv, 8)),
            (ValueError, lambda: K.rope_cache_write(qkv, inv, pos, pos, ck, cv, 0)),
            (TypeError, lambda: K.rope_cache_write(qkv, inv, pos.long(), pos, ck, cv, 8)),
            (ValueError, lambda: K.rope_cache_write(qkv, inv, pos, pos, ck, cv, 8, q_out=q[:3])),
            (ValueError, lambda: K.rope_cache_write(qkv, inv, pos, pos, ck, cv, 8,
                                                    q_out=qkv[:, :8 * D].contiguous().view(4, 8, D)[:, :, :64])),
            (ValueError, lambda: attend(q=q[:, :7])),
            (ValueError, lambda: attend(q=q[:, :, :64])),
            (TypeError, lambda: attend(q=q.float())),
            (ValueError, lambda: attend(starts=starts[:2])),
            (ValueError, lambda: attend(ctx=ctx_d[:1])),
            (ValueError, lambda: attend(tab=tab.t())),
            (ValueError, lambda: attend(max_ctx=0)),
            (ValueError, lambda: attend(max_ctx=tab.shape[1] * 16 + 1)),
            (ValueError, lambda: attend(new=-1)),
            (ValueError, lambda: attend(window=0)),
            (ValueError, lambda: attend(sinks=3)),
            (ValueError, lambda: attend(out=q[:3])),
            (TypeError, lambda: attend(stream="x")),
    )):
        print(at, exc, flush=True)
        with pytest.raises(exc):
            call()
    none = q[:0]
    assert tuple(attend(q=none, starts=_int32([0, 0, 0], cuda)).shape) == (0, 8, D)
    assert tuple(K.rope_cache_write(qkv[:0], inv, pos[:0], pos[:0], ck, cv, 8).shape) == (0, 8, D)
    m = K.chunk_map(past, new, tab.clone(), free[:0], 0)
    assert m.positions.numel() == 0 and m.starts.tolist() == [0, 3, 4]


def test_operands_that_are_no_tensors(cuda):
    """TypeError for each, whichever it is."""
    from rngd_pd_amd import kernels as K
    lens = [(3000, 100)]
    q, ck, cv, tables, ctx = _operands(np.random.default_rng(0), 8, 2, lens)
    tab, starts, ctx_d = torch.from_numpy(tables).to(cuda), _int32(_starts(lens), cuda), _int32(ctx, cuda)
    inv, pos = torch.ones(64, device=cuda), _int32([0] * 100, cuda)
    qkv = torch.zeros((100, 12 * D), dtype=torch.bfloat16, device=cuda)
    attention = [q, ck, cv, tab, starts, ctx_d, 100, 3100]
    calls = [lambda i=i: K.chunk_attention(*attention[:i], [1], *attention[i + 1:]) for i in range(6)]
    calls += [lambda: K.chunk_attention(*attention, workspace=1 << 28), lambda: K.chunk_attention(*attention, out=[])]
    write = [qkv, inv, pos, pos, ck, cv, 8]
    calls += [lambda i=i: K.rope_cache_write(*write[:i], [1], *write[i + 1:]) for i in range(6)]
    calls += [lambda: K.rope_cache_write(*write, q_out=[])]
    lengths = [ctx_d, ctx_d, tab, pos, 100]
    calls += [lambda i=i: K.chunk_map(*lengths[:i], [1], *lengths[i + 1:]) for i in range(4)]
    for at, call in enumerate(calls):
        print(at, flush=True)
        with pytest.raises(TypeError):
            call()
