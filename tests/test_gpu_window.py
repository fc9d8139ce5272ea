"""Attention over a sliding window and sinks, decode and prompt, against 64 bits."""
import math

import numpy as np
import pytest
import torch

from tests._span_ref import SCALE, assert_within, attend, decode_reference, paged, visible
from tests._util import rand_bf16, to_dev

pytestmark = pytest.mark.gpu
D = 128


def _inputs(rng, B, Hq, Hkv, nb):
    return (to_dev(rand_bf16(rng, (B, Hq, D))), to_dev(rand_bf16(rng, (nb, Hkv, 16, D))),
            to_dev(rand_bf16(rng, (nb, Hkv, D, 16))))


DECODE = [
    # Hq, Hkv, window, sinks, ctx
    (32, 8, 1, 0, [1, 2, 17, 300]),                       # the token itself alone
    (32, 8, 1, 4, [1, 3, 5, 6, 40]),
    (32, 8, 16, 0, [15, 16, 17, 31, 32, 33, 48, 49]),     # block edges
    (32, 8, 32, 1, [31, 32, 33, 63, 64, 65, 95, 97]),     # span edges
    (32, 8, 33, 33, [34, 66, 67, 98, 99, 130, 1000]),     # window and sinks meet
    (8, 8, 100, 64, [1, 64, 100, 163, 164, 165, 229, 5000]),
    (32, 8, 512, 4, [700]),
    (64, 8, 1000, 16, [4096, 1015, 1016, 1017]),
    (28, 4, 77, 5, [500, 81, 82, 83]),                    # groups that are no power of two
    (24, 8, 200, 0, [999, 12]),
    (40, 8, 129, 7, [321, 2000, 136]),
    (12, 1, 300, 4, [1500]),
    (13, 1, 50, 4, [70, 700]),
    (16, 1, 4096, 4, [9000, 4100]),
    (32, 8, 5000, 4, [40, 600]),                          # wider than the context
    (32, 8, 1 << 40, 0, [40, 600]),
    (4, 2, 255, 31, [256 + 13 * i for i in range(50)]),
    (8, 8, 64, 4, [64 + 31 * i for i in range(33)]),
    (8, 8, 64, 4, [3 + 7 * i for i in range(70)]),        # more than 64 streams
]


@pytest.mark.parametrize("Hq,Hkv,window,sinks,ctx", DECODE)
def test_decode(cuda, Hq, Hkv, window, sinks, ctx):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(Hq + window % 1000 + len(ctx))
    print(f"window Hq={Hq} Hkv={Hkv} window={window} sinks={sinks} ctx={ctx[:6]}", flush=True)
    tables, nb = paged(rng, ctx, Hkv)
    q, ck, cv = _inputs(rng, len(ctx), Hq, Hkv, nb)
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    got = K.decode_attention(q, ck, cv, tab, ctx_d, max(ctx), scale=SCALE, window=window, sinks=sinks)
    want, bound = decode_reference(q, ck, cv, tables, ctx, window, sinks, SCALE)
    assert_within(got, want, bound, "plain")
    # A larger max_ctx plans other splits; it changes no result beyond the bound.
    wide = torch.full((len(ctx), tables.shape[1] + 40), -1, dtype=torch.int32, device=cuda)
    wide[:, :tables.shape[1]] = tab
    got = K.decode_attention(q, ck, cv, wide, ctx_d, wide.shape[1] * 16, scale=SCALE,
                             window=window, sinks=sinks)
    assert_within(got, want, bound, "wide table")


@pytest.mark.parametrize("Hq,Hkv,window,sinks,ctx", [c for c in DECODE if c[2] < 1 << 20])
def test_append_is_the_write_then_the_attention(cuda, Hq, Hkv, window, sinks, ctx):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(3 * Hq + window + len(ctx))
    tables, nb = paged(rng, ctx, Hkv)
    B = len(ctx)
    q, ck, cv = _inputs(rng, B, Hq, Hkv, nb)
    kn, vn = (to_dev(rand_bf16(rng, (B, Hkv, D))) for _ in range(2))
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    ck2, cv2 = ck.clone(), cv.clone()
    K.cache_append(kn, vn, ck, cv, tab, ctx_d)
    want = K.decode_attention(q, ck, cv, tab, ctx_d, max(ctx), scale=SCALE, window=window, sinks=sinks)
    wide = torch.zeros((B, Hkv, 2, D), dtype=torch.bfloat16, device=cuda)
    wide[:, :, 1] = vn
    got = K.decode_attention_append(q, kn, wide[:, :, 1], ck2, cv2, tab, ctx_d, max(ctx),
                                    scale=SCALE, window=window, sinks=sinks)
    assert torch.equal(ck, ck2) and torch.equal(cv, cv2)
    assert torch.equal(got, want)


def test_blocks_behind_the_window_are_not_read(cuda):
    """Freed blocks (table -1), and NaN wherever no visible token lies: in hidden
    tokens of visible blocks, in slots behind the context, in unheld blocks."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(7)
    Hq, Hkv, window, sinks = 32, 8, 90, 5
    ctx = [5000, 40000, 91, 96, 200, 1]

    def held(b):
        c = ctx[b]
        return set(range(-(-min(sinks, c) // 16))) | set(range(max(0, c - window) // 16, -(-c // 16)))
    tables, nb = paged(rng, ctx, Hkv, held=held)
    q, ck, cv = _inputs(rng, len(ctx), Hq, Hkv, nb)
    want, bound = decode_reference(q, ck, cv, tables, ctx, window, sinks, SCALE)
    from rngd_pd_amd.engines.paged_cache import k_block_index
    place = k_block_index(D, cuda)
    seen = torch.zeros((nb, 16), dtype=torch.bool, device=cuda)
    for b, c in enumerate(ctx):
        for t in visible(c - 1, window, sinks):
            seen[int(tables[b, t // 16]), t % 16] = True
    flat = ck.view(nb, Hkv, 16 * D)
    for s in range(16):
        bad = (~seen[:, s]).nonzero()[:, 0]
        for value, half in ((float("nan"), bad[::2]), (float("inf"), bad[1::2])):
            flat[half[:, None, None], torch.arange(Hkv, device=cuda)[:, None], place[s]] = value
            cv[half, :, :, s] = value
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    got = K.decode_attention(q, ck, cv, tab, ctx_d, max(ctx), scale=SCALE, window=window, sinks=sinks)
    assert_within(got, want, bound)


def test_rows_without_tokens_and_contexts_past_the_table(cuda):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(8)
    Hq, Hkv = 32, 8
    for window, sinks in ((20, 4), (64, 0), (4, 100)):
        ctx = [0, 130, 160, 128 + 25, 5000, 100]
        tables, nb = paged(rng, [128] * len(ctx), Hkv)
        tables[5] = -1                                    # nothing valid at all
        tables[1, 7] = nb + 3
        q, ck, cv = _inputs(rng, len(ctx), Hq, Hkv, nb)
        tab = torch.from_numpy(tables).to(cuda)
        ctx_d = torch.tensor(ctx, dtype=torch.int32, device=cuda)
        want, bound = decode_reference(q, ck, cv, tables, ctx, window, sinks, SCALE)
        got = K.decode_attention(q, ck, cv, tab, ctx_d, 128, scale=SCALE, window=window, sinks=sinks)
        assert_within(got, want, bound, (window, sinks))
        assert (got[0] == 0).all() and (got[5] == 0).all()
        kn, vn = (to_dev(rand_bf16(rng, (len(ctx), Hkv, D))) for _ in range(2))
        ck2, cv2 = ck.clone(), cv.clone()
        K.cache_append(kn, vn, ck, cv, tab, ctx_d)
        want = K.decode_attention(q, ck, cv, tab, ctx_d, 128, scale=SCALE, window=window, sinks=sinks)
        got = K.decode_attention_append(q, kn, vn, ck2, cv2, tab, ctx_d, 128, scale=SCALE,
                                        window=window, sinks=sinks)
        assert torch.equal(ck, ck2) and torch.equal(cv, cv2) and torch.equal(got, want)


def test_any_length_on_the_device_stays_in_bounds(cuda):
    """Lengths are device data: whatever they hold, only the table's tokens are
    read, and a window that starts behind them leaves the sinks."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(18)
    ctx = [2 ** 31 - 1, -(2 ** 31), -1, 2 ** 31 - 20, 10 ** 9, 64]
    tables, nb = paged(rng, [64] * 6, 8)
    q, ck, cv = _inputs(rng, 6, 32, 8, nb)
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    for window, sinks in ((10, 5), (1 << 30, 0), (40, 0)):
        want, bound = decode_reference(q, ck, cv, tables, ctx[-1:] * 6, window, sinks, SCALE)
        got = K.decode_attention(q, ck, cv, tab, ctx_d, 64, scale=SCALE, window=window, sinks=sinks)
        assert_within(got[5:], want[5:], bound[5:])
        assert (got[1:3] == 0).all() and torch.isfinite(got).all()
        if sinks:
            few, few_bound = decode_reference(q, ck, cv, tables, [5] * 6, 5, 0, SCALE)
            for b in (0, 3, 4):
                assert_within(got[b], few[b], few_bound[b])
        elif window == 40:
            assert (got[[0, 3, 4]] == 0).all()


def test_streams_that_share_blocks(cuda):
    """Four rows of one request at consecutive positions (a verification step):
    each sees the others' new tokens, inside its own window."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(9)
    Hq, Hkv, window, sinks = 32, 8, 18, 3
    ctx = [45, 46, 47, 48, 49, 2, 3, 4]
    tables, nb = paged(rng, [64, 16], Hkv)
    tables = np.concatenate([np.repeat(tables[:1], 5, 0), np.repeat(tables[1:], 3, 0)])
    q, ck, cv = _inputs(rng, 8, Hq, Hkv, nb)
    kn, vn = (to_dev(rand_bf16(rng, (8, Hkv, D))) for _ in range(2))
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    ck2, cv2 = ck.clone(), cv.clone()
    K.cache_append(kn, vn, ck, cv, tab, ctx_d)
    want, bound = decode_reference(q, ck, cv, tables, ctx, window, sinks, SCALE)
    got = K.decode_attention_append(q, kn, vn, ck2, cv2, tab, ctx_d, 64, scale=SCALE, window=window,
                                    sinks=sinks)
    assert torch.equal(ck, ck2) and torch.equal(cv, cv2)
    assert_within(got, want, bound)


def test_equals_full_attention_inside_the_window(cuda):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(10)
    ctx = [512, 33, 16, 1, 300]
    tables, nb = paged(rng, ctx, 8)
    q, ck, cv = _inputs(rng, len(ctx), 32, 8, nb)
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    want = K.decode_attention(q, ck, cv, tab, ctx_d, 512, scale=SCALE)
    for window, sinks in ((512, 0), (600, 4), (508, 4)):
        got = K.decode_attention(q, ck, cv, tab, ctx_d, 512, scale=SCALE, window=window, sinks=sinks)
        assert torch.equal(got, want)


def test_long_cache_offsets(cuda):
    """A cache whose last block starts beyond 2^31 elements."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(11)
    Hkv, nb = 8, (1 << 31) // (8 * 16 * D) + 40
    q = to_dev(rand_bf16(rng, (2, 32, D)))
    ck = torch.zeros((nb, Hkv, 16, D), dtype=torch.bfloat16, device=cuda)
    cv = torch.zeros((nb, Hkv, D, 16), dtype=torch.bfloat16, device=cuda)
    ck[-40:].normal_()
    cv[-40:].normal_()
    tables = np.full((2, 2000), -1, np.int32)
    tables[0, [0, *range(1990, 2000)]] = np.arange(nb - 11, nb)
    tables[1, [0, 1, *range(500, 510)]] = np.arange(nb - 30, nb - 18)
    ctx = [32000, 8150]
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    want, bound = decode_reference(q, ck, cv, tables, ctx, 150, 4, SCALE)
    got = K.decode_attention(q, ck, cv, tab, ctx_d, 32000, scale=SCALE, window=150, sinks=4)
    assert_within(got, want, bound)


def test_streams_graphs_and_workspaces(cuda):
    """On another stream; captured twice over one set of tensors; replayed between
    eager calls with new inputs."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(12)
    ctx, window, sinks = [3000, 700], 900, 4                 # splits: needs a workspace
    tables, nb = paged(rng, ctx, 8)
    q, ck, cv = _inputs(rng, 2, 32, 8, nb)
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    args = dict(scale=SCALE, window=window, sinks=sinks)
    want = K.decode_attention(q, ck, cv, tab, ctx_d, 3000, **args)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = K.decode_attention(q, ck, cv, tab, ctx_d, 3000, stream=side, **args)
    side.synchronize()
    assert torch.equal(got, want)
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.decode_attention(q, ck, cv, tab, ctx_d, 3000, **args))
        graphs.append(g)
    for i in range(3):
        q.normal_()
        want = K.decode_attention(q, ck, cv, tab, ctx_d, 3000, **args)
        for g, o in zip(graphs, outs):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want), i
    ws = torch.empty(K.workspace_bytes(2, 32, K.window_span(3000, window, sinks)),
                     dtype=torch.uint8, device=cuda)
    assert torch.equal(K.decode_attention(q, ck, cv, tab, ctx_d, 3000, workspace=ws, **args), want)


# ---- the prompt form ----------------------------------------------------------
PROMPT = [
    # T, Hq, Hkv, window, sinks
    (1, 32, 8, 1, 0), (2, 8, 8, 1, 0), (31, 32, 8, 7, 0), (32, 8, 2, 32, 1), (33, 32, 8, 16, 4),
    (64, 12, 4, 33, 33), (65, 32, 8, 31, 40), (129, 7, 1, 50, 3), (200, 32, 8, 1, 4),
    (200, 32, 8, 500, 4), (470, 32, 8, 128, 4), (513, 40, 8, 100, 64), (700, 24, 8, 255, 1),
    (1000, 16, 16, 97, 129), (1111, 64, 8, 512, 0), (300, 20, 1, 64, 16),
    # Two teams: even and odd numbers of tiles, sinks in front, several query tiles in a workgroup.
    (470, 32, 8, 470, 0), (289, 8, 8, 289, 0), (1000, 8, 2, 1000, 0), (777, 7, 1, 400, 40),
    (600, 6, 6, 300, 70), (1024, 16, 2, 260, 0),
]


def _prompt_reference(q, k, v, window, sinks, scale):
    T, Hq, _ = q.shape
    H = k.shape[1]
    G = Hq // H
    t = torch.arange(T, device=q.device)
    hidden = (t > t[:, None]) | ((t <= t[:, None] - window) & (t >= sinks))
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for h in range(Hq):
        qh, kh, vh = q[:, h].double(), k[:, h // G].double(), v[:, h // G].double()
        s = (torch.matmul(qh, kh.t().contiguous()) * scale).masked_fill(hidden, -math.inf)
        p = torch.softmax(s, -1)
        o, A = torch.matmul(p, vh), torch.matmul(p, vh.abs())
        mass = float((torch.matmul(qh.abs(), kh.abs().t().contiguous()) * scale).max())
        share = 2 * (128 * 2.0 ** -24 * mass + T * 2.0 ** -24) + 2.0 ** -18 + 2.0 ** -8
        out[:, h] = o                                    # (attend()'s bound, row by row)
        bound[:, h] = (1 + 2.0 ** -8) * share * A + 2.0 ** -8 * o.abs() + 2.0 ** -134
    return out, bound


@pytest.mark.parametrize("T,Hq,Hkv,window,sinks", PROMPT)
def test_prompt(cuda, T, Hq, Hkv, window, sinks):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(T + Hq)
    print(f"prompt T={T} Hq={Hq} Hkv={Hkv} window={window} sinks={sinks}", flush=True)
    qkv = to_dev(rand_bf16(rng, (T, Hq + 2 * Hkv, D)))
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    got = K.prefill_attention(q, k, v, scale=SCALE, window=window, sinks=sinks)
    want, bound = _prompt_reference(q, k, v, window, sinks, SCALE)
    assert_within(got, want, bound)
    # Other layouts: heads first; rows off 16 bytes.
    kt = k.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(v.numel() + 1, dtype=torch.bfloat16, device=cuda)
    odd[1:] = v.reshape(-1)
    out = torch.full((T, Hq, D), float("nan"), dtype=torch.bfloat16, device=cuda)
    got2 = K.prefill_attention(q.contiguous(), kt, odd[1:].view(T, Hkv, D), scale=SCALE,
                               window=window, sinks=sinks, out=out)
    assert got2 is out and torch.equal(got2, got)


def test_prompt_last_row_is_the_decode_form(cuda):
    """The prompt's last query and the decode form over the same tokens: both
    within their bounds of one value."""
    from rngd_pd_amd import kernels as K
    from rngd_pd_amd.engines.paged_cache import k_block_tiled
    rng = np.random.default_rng(13)
    T, Hq, Hkv, window, sinks = 333, 32, 8, 70, 4
    q = to_dev(rand_bf16(rng, (T, Hq, D)))
    k, v = (to_dev(rand_bf16(rng, (T, Hkv, D))) for _ in range(2))
    got = K.prefill_attention(q, k, v, scale=SCALE, window=window, sinks=sinks)[-1]
    nb = -(-T // 16)
    pad = torch.zeros((nb * 16, Hkv, D), dtype=torch.bfloat16, device=cuda)
    pad[:T] = k
    ck = k_block_tiled(pad.view(nb, 16, Hkv, D).transpose(1, 2).contiguous()).contiguous()
    pad[:T] = v
    cv = pad.view(nb, 16, Hkv, D).permute(0, 2, 3, 1).contiguous()
    tab = torch.arange(nb, dtype=torch.int32, device=cuda)[None]
    one = K.decode_attention(q[-1:], ck, cv, tab, torch.tensor([T], dtype=torch.int32, device=cuda),
                             T, scale=SCALE, window=window, sinks=sinks)[0]
    pos = torch.tensor(visible(T - 1, window, sinks), device=cuda)
    want, bound = attend(q[-1].view(Hkv, -1, D), k[pos], v[pos], SCALE)
    assert_within(got.view(Hkv, -1, D), want, bound, "prompt")
    assert_within(one.view(Hkv, -1, D), want, bound, "decode")


def test_prompt_without_a_window_is_causal(cuda):
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(14)
    T, Hq, Hkv = 150, 32, 8
    q = to_dev(rand_bf16(rng, (T, Hq, D)))
    k, v = (to_dev(rand_bf16(rng, (T, Hkv, D))) for _ in range(2))
    want, bound = _prompt_reference(q, k, v, T, 0, SCALE)
    assert_within(K.prefill_attention(q, k, v, scale=SCALE), want, bound)
    assert K.prefill_attention(q[:0], k[:0], v[:0]).shape == (0, Hq, D)


def test_prompt_large_scores(cuda):
    """Scores far apart: the running maximum moves on every tile."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(15)
    T, Hq, Hkv = 400, 8, 2
    q = to_dev(rand_bf16(rng, (T, Hq, D)))
    k, v = (to_dev(rand_bf16(rng, (T, Hkv, D))) for _ in range(2))
    k *= torch.linspace(0.1, 20, T, device=cuda).to(torch.bfloat16)[:, None, None]
    want, bound = _prompt_reference(q, k, v, 100, 4, SCALE)
    assert_within(K.prefill_attention(q, k, v, scale=SCALE, window=100, sinks=4), want, bound)


@pytest.mark.parametrize("window,sinks", [(40, 4), (300, 0)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_prompt_hidden_values_reach_no_query(cuda, window, sinks, value):
    """NaN or infinity in k and v of token t spoils the queries that see it and no
    other, those of its own tile among them."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(17)
    T, Hq, Hkv, at = 230, 8, 2, [101, 117]
    q = to_dev(rand_bf16(rng, (T, Hq, D)))
    k, v = (to_dev(rand_bf16(rng, (T, Hkv, D))) for _ in range(2))
    want, bound = _prompt_reference(q, k, v, window, sinks, SCALE)
    k[at[0]], v[at[1]] = value, value
    got = K.prefill_attention(q, k, v, scale=SCALE, window=window, sinks=sinks)
    t = torch.arange(T, device=cuda)
    clean = torch.ones(T, dtype=torch.bool, device=cuda)
    for a in at:
        clean &= (t < a) | (t - a >= window)
    assert 0 < int(clean.sum()) < T
    assert_within(got[clean], want[clean], bound[clean])
    assert not torch.isfinite(got[at[1]]).any()


@pytest.mark.parametrize("T,window,sinks", [(230, 40, 4), (1500, 1500, 0), (33, 33, 0)])
def test_prompt_values_that_are_not_finite(cuda, T, window, sinks):
    """A dim that is NaN in every token of one head, an infinity in one token's dim
    and one of each sign in two tokens': as the sums over the seen tokens have them."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(21)
    q = to_dev(rand_bf16(rng, (T, 8, D)))
    k, v = (to_dev(rand_bf16(rng, (T, 2, D))) for _ in range(2))
    want, bound = _prompt_reference(q, k, v, window, sinks, SCALE)
    want, bound = want.clone(), bound.clone()
    inf, t = float("inf"), torch.arange(T, device=cuda)

    def sees(a):
        return ((t >= a) & ((t - a < window) | (a < sinks))).cpu().to(want.device)

    v[:, 0, 5] = float("nan")
    v[20, 1, 7] = inf
    v[9, 0, 90] = inf
    v[25, 0, 90] = -inf
    got = K.prefill_attention(q, k, v, scale=SCALE, window=window, sinks=sinks)
    assert torch.isnan(got[:, :4, 5]).all()
    s20, s9, s25 = sees(20), sees(9), sees(25)
    assert (got[s20.to(cuda), 4:, 7] == inf).all()
    assert (got[(s9 & ~s25).to(cuda), :4, 90] == inf).all()
    assert (got[(s25 & ~s9).to(cuda), :4, 90] == -inf).all()
    assert torch.isnan(got[(s9 & s25).to(cuda), :4, 90]).all()
    # All others.
    plain = torch.ones_like(want, dtype=torch.bool)
    plain[:, :4, 5] = False
    plain[s20, 4:, 7] = False
    plain[s9 | s25, :4, 90] = False
    assert_within(got[plain.to(cuda)], want[plain], bound[plain])


def test_refusals(cuda):
    from rngd_pd_amd import kernels as K
    from rngd_pd_amd._lib import PdkError
    rng = np.random.default_rng(16)
    tables, nb = paged(rng, [64], 8)
    q, ck, cv = _inputs(rng, 1, 32, 8, nb)
    tab, ctx = torch.from_numpy(tables).to(cuda), torch.tensor([64], dtype=torch.int32, device=cuda)
    for kw in (dict(window=0), dict(window=-1), dict(sinks=4), dict(window=4, sinks=-1),
               dict(window=8, sinks=16385)):
        with pytest.raises(ValueError):
            K.decode_attention(q, ck, cv, tab, ctx, 64, **kw)
    with pytest.raises(ValueError):
        K.decode_attention(q, ck, cv, tab, ctx, 65, window=4)
    with pytest.raises(PdkError, match="16384"):
        big = torch.full((1, 5000), -1, dtype=torch.int32, device=cuda)
        K.decode_attention(q, ck, cv, big, ctx, 80000, window=20000)
    with pytest.raises(ValueError):
        K.decode_attention(q, ck, cv, tab, ctx, 64, window=4, out=q[:, :8])
    with pytest.raises(ValueError, match="overlap"):
        K.decode_attention(q, ck, cv, tab, ctx, 64, window=4, out=q)
    with pytest.raises(ValueError):
        K.decode_attention(q, ck, cv, tab.cpu(), ctx, 64, window=4)
    wide = to_dev(rand_bf16(rng, (1, 17 * 8, D)))
    with pytest.raises(PdkError, match="group"):
        K.decode_attention(wide, ck, cv, tab, ctx, 64, window=4)
    with pytest.raises(ValueError):
        K.prefill_attention(q, q[:, :8], q[:, :4])
    with pytest.raises(ValueError):
        K.prefill_attention(q, q[:, :8], q[:, :8], window=0)
    with pytest.raises(PdkError):
        K.prefill_attention(q, q[:, :5], q[:, :5])       # 32 heads over 5
    with pytest.raises(TypeError):
        K.prefill_attention(q, q[:, :8].float(), q[:, :8])
    with pytest.raises(ValueError, match="overlap"):
        K.prefill_attention(q, ck[:1, :, 0], ck[1:2, :, 0], out=q)
