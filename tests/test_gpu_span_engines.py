"""A sliding window through the engines, and beam search: the decoder, the prefill,
the batched attention and the scheduler with a windowed config; BeamSearch against
a search that keeps its hypotheses apart and decodes each of them by itself."""
import math

import numpy as np
import pytest
import torch

from tests._span_ref import SCALE, assert_within, decode_reference, paged
from tests._util import rand_bf16, to_dev

pytestmark = pytest.mark.gpu
D = 128


def _cfg(**kw):
    from rngd_pd_amd.engines.llama_decode import LlamaConfig
    return LlamaConfig(**{**dict(hidden=512, n_heads=8, n_kv_heads=2, head_dim=128, inter=1024,
                                 vocab=1000, n_layers=2), **kw})


@pytest.mark.parametrize("tiled", [False, True])
@pytest.mark.parametrize("splits,Hq,Hkv,window,sinks,ctx", [
    (1, 8, 2, 20, 4, [1, 20, 21, 45, 300]), (2, 32, 8, 100, 5, [700, 99, 3, 131]),
    (2, 24, 8, 33, 0, [65, 500]), (2, 32, 8, 2000, 4, [2500])])
def test_fused_rope_equals_two_calls(cuda, tiled, splits, Hq, Hkv, window, sinks, ctx):
    """RoPE, cache write and windowed attention in one launch, against the cache
    append kernel followed by the windowed attention: bit for bit."""
    from rngd_pd_amd import _lib
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(window)
    B, N = len(ctx), (Hq + 2 * Hkv) * D
    tables, nb = paged(rng, ctx, Hkv)
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    ck, cv = to_dev(rand_bf16(rng, (nb, Hkv, 16, D))), to_dev(rand_bf16(rng, (nb, Hkv, D, 16)))
    part = torch.randn((splits, B, N), device=cuda)
    inv = (1.0 / 1e4 ** (torch.arange(64, device=cuda) / 64)).float()
    ck2, cv2 = ck.clone(), cv.clone()
    q = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=cuda)
    st = K.stream_handle()
    _lib.call("pdk_rope_cache_append_partials", part.data_ptr(), splits, N, q.data_ptr(),
              inv.data_ptr(), ctx_d.data_ptr(), tab.data_ptr(), tab.shape[1], ck.data_ptr(),
              cv.data_ptr(), nb, B, Hq, Hkv, D, st)
    want = K.decode_attention(q, ck, cv, tab, ctx_d, max(ctx), scale=SCALE, window=window, sinks=sinks)
    ref, bound = decode_reference(q, ck, cv, tables, ctx, window, sinks, SCALE)
    assert_within(want, ref, bound)
    need = K.workspace_bytes(B, Hq, K.window_span(max(ctx), window, sinks))
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=cuda)
    rows = 16 * -(-B // 16) if tiled else B
    out = torch.zeros(rows * Hq * D, dtype=torch.bfloat16, device=cuda)
    _lib.call("pdk_decode_attn_rope_window", part.data_ptr(), splits, inv.data_ptr(), ck2.data_ptr(),
              cv2.data_ptr(), nb, tab.data_ptr(), tab.shape[1], ctx_d.data_ptr(), max(ctx), window,
              sinks, B, Hq, Hkv, D, SCALE, ws.data_ptr(), ws.numel(), out.data_ptr(), int(tiled), 0, st)
    got = K.act_untile(out, B, Hq * D).view(B, Hq, D) if tiled else out.view(B, Hq, D)
    assert torch.equal(ck, ck2) and torch.equal(cv, cv2) and torch.equal(got, want)


def _decoder(cfg, cache, seed=3, **kw):
    from rngd_pd_amd.engines.llama_decode import LlamaDecoder, LlamaWeights
    return LlamaDecoder(LlamaWeights.random(cfg, seed=seed, device=cache.device), cache, **kw)


def _feed(dec, cache, req, tokens, start=0):
    """Decode tokens one by one under req; the logits after the last."""
    for i, t in enumerate(tokens, start):
        cache.ensure(req, i + 1)
        tab = cache.table(req)[None].contiguous()
        dec.step(torch.tensor([t], dtype=torch.int32, device=cache.device),
                 torch.tensor([i + 1], dtype=torch.int32, device=cache.device), tab, 16 * tab.shape[1])
    return dec.logits[0].clone()


def test_decoder_and_prefill_agree_under_a_window(cuda):
    """The prompt through the windowed prefill and, token by token, through the
    windowed decoder: the same keys and values (bf16 noise of two layers), and
    others than without the window where it hides something."""
    from rngd_pd_amd.engines.llama_decode import LlamaWeights
    from rngd_pd_amd.engines.llama_prefill import LlamaPrefill
    from rngd_pd_amd.engines.paged_cache import PagedKVCache, k_block_rows
    tokens = np.random.default_rng(5).integers(0, 1000, 150).tolist()
    got = {}
    for window, sinks in ((40, 4), (None, 0)):
        cfg = _cfg(window=window, sinks=sinks)
        pre = LlamaPrefill(LlamaWeights.random(cfg, seed=3, device=cuda))
        _, k, v = pre.forward(tokens)
        cache = PagedKVCache(cfg.n_layers, 12, cfg.n_kv_heads, D, device=cuda, seed=2)
        dec = _decoder(cfg, cache, max_batch=1)
        _feed(dec, cache, "r", tokens)
        b = cache.blocks("r")
        kd = k_block_rows(cache.k[:, b]).permute(0, 1, 3, 2, 4).reshape(2, -1, 2, D)[:, :150]
        vd = cache.v[:, b].permute(0, 1, 4, 2, 3).reshape(2, -1, 2, D)[:, :150]
        torch.cuda.synchronize()
        for a, c in ((k, kd), (v, vd)):
            assert (a.float() - c.float()).norm() <= 2e-2 * c.float().norm()
        got[window] = kd[1].float()
        if window:
            noise = (k[1].float() - kd[1].float()).norm()
    # The window shows beyond the noise between the two ways of computing it.
    assert (got[40] - got[None]).norm() > 2 * noise
    assert torch.equal(got[40][:40], got[None][:40])


def test_prefill_of_other_head_dims_takes_the_window(cuda):
    from rngd_pd_amd.engines.llama_decode import LlamaWeights
    from rngd_pd_amd.engines.llama_prefill import LlamaPrefill
    tokens = list(range(90))
    outs = []
    for window in (None, 200, 17):
        cfg = _cfg(hidden=256, n_heads=4, head_dim=64, inter=256, window=window)
        outs.append(LlamaPrefill(LlamaWeights.random(cfg, seed=4, device=cuda)).forward(tokens)[1])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])
    assert torch.equal(outs[0][1, :17], outs[2][1, :17])
    assert not torch.equal(outs[0][1, 40:], outs[2][1, 40:])


def test_window_wider_than_the_context_changes_nothing(cuda):
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    tokens = np.random.default_rng(6).integers(0, 1000, 60).tolist()
    logits = []
    for window, sinks in ((None, 0), (60, 0), (4000, 7)):
        cache = PagedKVCache(2, 8, 2, D, device=cuda, seed=2)
        logits.append(_feed(_decoder(_cfg(window=window, sinks=sinks), cache, max_batch=1), cache,
                            "r", tokens))
    assert torch.equal(logits[0], logits[1]) and torch.equal(logits[0], logits[2])


def test_batched_attention_trims_blocks(cuda):
    """BatchDecodeAttention with a window: blocks behind it go back to the pool and
    the results stay those of a cache that keeps them."""
    from rngd_pd_amd.engines.decode_batch import BatchDecodeAttention
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    engines = []
    for _ in range(2):
        cache = PagedKVCache(1, 40, 2, D, device=cuda, seed=3)
        eng = BatchDecodeAttention(cache, n_q_heads=8, window=50, sinks=3)
        for r, n in (("a", 100), ("b", 20)):
            cache.allocate(r, n)
            eng.admit_loaded(r, n)
        g = torch.Generator(device=cuda).manual_seed(1)
        cache.k.normal_(generator=g)
        cache.v.normal_(generator=g)
        engines.append(eng)
    g = torch.Generator(device=cuda).manual_seed(2)
    for step in range(60):
        q = torch.randn((2, 8, D), generator=g, device=cuda).to(torch.bfloat16)
        kn, vn = (torch.randn((2, 2, D), generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
        outs = []
        for i, eng in enumerate(engines):
            tab, ctx, mx = eng.prepare(["a", "b"])
            outs.append(eng.layer_attention(0, q, kn, vn, tab, ctx, mx))
            eng.advance(["a", "b"])
            if i == 1:
                eng.trim(["a", "b"])
        if step % 8 == 0:
            assert torch.equal(outs[0], outs[1]), step
    held = [sum(b >= 0 for b in engines[1].cache.blocks(r)) for r in "ab"]
    assert held == [5, 5]                               # the sinks' block and a window over 4
    assert engines[1].cache.alloc.free_blocks() == 30
    assert engines[0].cache.alloc.free_blocks() == 40 - 10 - 5


def test_scheduler_returns_blocks_behind_the_window(cuda):
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    from rngd_pd_amd.serving.scheduler import ContinuousScheduler
    outs = {}
    for blocks in (64, 9):                              # plenty, and less than one stream's 11
        cfg = _cfg(window=48, sinks=4)
        cache = PagedKVCache(cfg.n_layers, blocks, cfg.n_kv_heads, D, device=cuda, seed=2)
        dec = _decoder(cfg, cache, max_batch=1)

        def produce(item):
            cache.allocate(item["req_id"], 1)
            return 7, 0, 0.0
        sched = ContinuousScheduler(1, dec, cache, produce, max_blocks=12, use_graphs=blocks == 64)
        outs[blocks] = sched.submit({"req_id": "r", "max_new": 170})["tokens"]
        sched.close()
        assert cache.alloc.free_blocks() == blocks
    assert outs[64] == outs[9] and len(outs[9]) == 170


def _reference_search(dec, cache, prompt, K, eos, max_new):
    """Hypotheses as token lists, each decoded alone from scratch."""
    n = [0]

    def logits(seq):
        n[0] += 1
        x = _feed(dec, cache, ("ref", n[0]), prompt + seq)
        cache.free(("ref", n[0]))
        return x.double().cpu()
    live = [([], 0.0)]
    for _ in range(max_new):
        cand = []
        for i, (seq, score) in enumerate(live):
            if eos is not None and seq and seq[-1] == eos:
                cand.append((-score, i, 0.0, seq))
                continue
            x = logits(seq)
            lp = x - x.max() - torch.log(torch.exp(x - x.max()).sum())
            order = np.lexsort((np.arange(len(x)), -x.numpy()))[:K]
            cand += [(-(score + float(lp[t])), i, -float(x[t]), seq + [int(t)]) for t in order]
        cand.sort(key=lambda c: c[:3])
        # The engine carries 32-bit scores from step to step.
        live = [(seq, float(np.float32(-s))) for s, _, _, seq in cand[:K]]
    return live


@pytest.mark.parametrize("graphs", [False, True])
@pytest.mark.parametrize("K,prompts,eos,max_new,window", [
    (3, [5], None, 9, None), (4, [16, 33], None, 20, None), (2, [1, 17, 40], 11, 18, None),
    (4, [30], None, 12, 24)])
def test_beam_search(cuda, K, prompts, eos, max_new, window, graphs):
    from rngd_pd_amd.engines.beam_search import BeamSearch
    from rngd_pd_amd.engines.llama_decode import LlamaDecoder
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    rng = np.random.default_rng(K)
    cfg = _cfg(vocab=300, window=window, sinks=2 if window else 0)
    cache = PagedKVCache(cfg.n_layers, 90, cfg.n_kv_heads, D, device=cuda, seed=2)
    dec = _decoder(cfg, cache, max_batch=12)
    if eos is not None:                                 # an end token that is often likely
        dec.w.lm_head[eos] *= 2
        dec = LlamaDecoder(dec.w, cache, max_batch=12)
    seqs = [rng.integers(0, 300, n).tolist() for n in prompts]
    want = []
    for i, p in enumerate(seqs):
        want.append(_reference_search(dec, cache, p, K, eos, max_new))
        if len(p) > 1:
            _feed(dec, cache, i, p[:-1])
        else:
            cache.allocate(i, 0)
    before = cache.alloc.free_blocks()
    search = BeamSearch(dec, K, eos=eos, use_graphs=graphs, check_every=4)
    for _ in range(2):                                  # the requests keep their blocks
        got = search.search([(i, len(p), p[-1]) for i, p in enumerate(seqs)], max_new)
        assert cache.alloc.free_blocks() == before
        for g, w in zip(got, want):
            assert [s for s, _ in g] == [s for s, _ in w]
            for (_, a), (_, b) in zip(g, w):
                assert abs(a - b) <= 2.0 ** -23 * max(1.0, abs(b)) * max_new
    if eos is not None:
        assert any(s[-1] == eos for g in got for s, _ in g)


def test_beam_search_refusals(cuda):
    from rngd_pd_amd.engines.beam_search import BeamSearch
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    cache = PagedKVCache(2, 8, 2, D, device=cuda)
    dec = _decoder(_cfg(), cache, max_batch=4)
    cache.allocate("r", 20)
    for k in (0, 17):
        with pytest.raises(ValueError):
            BeamSearch(dec, k)
    s = BeamSearch(dec, 4)
    for reqs, n in (([], 4), ([("r", 10, 1)] * 2, 4), ([("r", 10, 1)], 0), ([("r", 0, 1)], 3)):
        with pytest.raises(ValueError):
            s.search(reqs, n)
    free = cache.alloc.free_blocks()
    with pytest.raises(MemoryError):
        s.search([("r", 20, 1)], 60)
    assert cache.alloc.free_blocks() == free
    assert math.isfinite(s.search([("r", 10, 1)], 2, length_penalty=1.0)[0][0][1])


def test_a_longer_search_after_a_captured_one(cuda):
    """A search's graph dies with it: the decoder's workspace may grow again."""
    from rngd_pd_amd.engines.beam_search import BeamSearch
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    cache = PagedKVCache(2, 160, 2, D, device=cuda)
    dec = _decoder(_cfg(), cache, max_batch=2)
    cache.allocate("r", 200)
    s = BeamSearch(dec, 2)
    first = s.search([("r", 10, 1)], 5)
    s.search([("r", 150, 1)], 400)                      # its contexts are split
    assert s.search([("r", 10, 1)], 5)[0][0][0] == first[0][0][0]
    assert cache.alloc.free_blocks() == 160 - 13
