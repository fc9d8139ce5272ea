"""ChunkPrefill: prompts in pieces on the paged cache, against LlamaPrefill's whole
prompts, a decoder's steps and the kernels one by one."""
import numpy as np
import pytest
import torch

from rngd_pd_amd import kernels as K
from rngd_pd_amd.engines.chunk_prefill import ChunkPrefill
from rngd_pd_amd.engines.llama_decode import LlamaConfig, LlamaDecoder, LlamaWeights
from rngd_pd_amd.engines.llama_prefill import LlamaPrefill
from rngd_pd_amd.engines.paged_cache import PagedKVCache, k_block_rows

pytestmark = pytest.mark.gpu


def _model(cuda, **kw):
    cfg = LlamaConfig(hidden=512, n_heads=8, n_kv_heads=2, head_dim=128, inter=768, vocab=1000,
                      n_layers=2, **kw)
    return cfg, LlamaWeights.random(cfg, seed=3, device=cuda)


def _cache(cfg, cuda, blocks=200):
    return PagedKVCache(cfg.n_layers, blocks, cfg.n_kv_heads, cfg.head_dim, device=cuda, seed=5)


def _rows(cache, req, n):
    """K and V of a request's first n tokens as [L, n, Hkv, D]."""
    b = torch.tensor(cache.blocks(req)[:-(-n // 16)], device=cache.k.device)
    k = k_block_rows(cache.k[:, b]).permute(0, 1, 3, 2, 4).flatten(1, 2)[:, :n]
    v = cache.v[:, b].permute(0, 1, 4, 2, 3).flatten(1, 2)[:, :n]
    return k, v


def _near(got, want, share):
    """Norms of the difference: the two paths round the same values at other places."""
    off = float((got.double() - want.double()).norm() / want.double().norm())
    assert off <= share, off


# Both paths round to bf16 (at most 2^-8, some 2^-9 / sqrt(3) rms) at the same dozen places
# of a layer, the sums before them in another order; two layers' worth of such differences
# stays below 2^-5 of the values.
SHARE = 2.0 ** -5


@pytest.mark.parametrize("window,sinks", [(None, 0), (24, 4)])
def test_pieces_make_the_whole_prompt(cuda, window, sinks):
    cfg, w = _model(cuda, window=window, sinks=sinks)
    cache, pre = _cache(cfg, cuda), LlamaPrefill(w)
    eng = ChunkPrefill(w, cache)
    rng = np.random.default_rng(0)
    prompts = {r: rng.integers(0, cfg.vocab, n).tolist() for r, n in (("a", 130), ("b", 17), ("c", 61))}
    steps = [[("a", 0, 50), ("b", 0, 17)], [("a", 50, 1), ("c", 0, 33)], [("c", 33, 28), ("a", 51, 79)]]
    for step in steps:
        out = eng.step([(r, p, prompts[r][p:p + n]) for r, p, n in step])
        assert len(out) == len(step) and all(0 <= t < cfg.vocab for t in out)
    for r, tokens in prompts.items():
        first, k, v = pre.forward(tokens)
        got_k, got_v = _rows(cache, r, len(tokens))
        _near(got_k, k, SHARE)
        _near(got_v, v, SHARE)


def test_every_token_and_a_rejected_draft(cuda):
    """The tokens after each new one are those of one step at a time, and a draft's
    blocks are written over."""
    cfg, w = _model(cuda)
    rng = np.random.default_rng(1)
    prompt = rng.integers(0, cfg.vocab, 40).tolist()
    cache = _cache(cfg, cuda)
    eng = ChunkPrefill(w, cache)
    eng.step([("a", 0, prompt)])
    draft = rng.integers(0, cfg.vocab, 9).tolist()
    got = eng.step([("a", 40, draft)], every=True)
    hidden = eng.x.clone()
    assert len(got) == 1 and len(got[0]) == 9
    rows, k0 = [], _rows(cache, "a", 49)[0].clone()
    for i, t in enumerate(draft):                    # the same tokens again, one by one
        eng.step([("a", 40 + i, [t])])
        rows.append(eng.x.clone())
    _near(torch.cat(rows), hidden, SHARE)
    _near(_rows(cache, "a", 49)[0], k0, SHARE)
    assert len(cache.blocks("a")) == 4


def test_a_decoder_goes_on(cuda):
    """A prompt in pieces, then LlamaDecoder's steps on the same cache, beside single
    tokens through ChunkPrefill."""
    cfg, w = _model(cuda)
    rng = np.random.default_rng(2)
    prompt = rng.integers(0, cfg.vocab, 77).tolist()
    cache = _cache(cfg, cuda)
    eng, dec = ChunkPrefill(w, cache), LlamaDecoder(w, cache, max_batch=2)
    for r in ("a", "b"):
        eng.step([(r, 0, prompt[:45])])
        eng.step([(r, 45, prompt[45:])])
    for i, t in enumerate(rng.integers(0, cfg.vocab, 5).tolist()):
        n = 78 + i
        cache.ensure("a", n)
        table = cache.table("a").view(1, -1)
        dec.step(torch.tensor([t], device=cuda), torch.tensor([n], dtype=torch.int32, device=cuda),
                 table, n)
        one = dec.x[:1].clone()
        eng.step([("b", n - 1, [t])])
        _near(eng.x, one, SHARE)
    for got, want in zip(_rows(cache, "b", 82), _rows(cache, "a", 82)):
        _near(got, want, SHARE)


def test_fp8_is_the_kernels_one_by_one(cuda):
    cfg, w = _model(cuda)
    rng = np.random.default_rng(4)
    chunks = [("a", 0, rng.integers(0, cfg.vocab, 70).tolist()), ("b", 0, [5]),
              ("c", 0, rng.integers(0, cfg.vocab, 20).tolist())]
    cache = _cache(cfg, cuda)
    eng = ChunkPrefill(w, cache, fp8=True)
    out = eng.step(chunks)
    own = _cache(cfg, cuda)
    tables, free = own.extend([(r, p, len(t)) for r, p, t in chunks])
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)          # noqa: E731
    tab = torch.from_numpy(tables).to(cuda)
    m = K.chunk_map(i32([0, 0, 0]), i32([70, 1, 20]), tab, torch.from_numpy(free).to(cuda), 91)
    x = w.embed[torch.tensor([t for c in chunks for t in c[2]], device=cuda)]
    down = None
    lin = lambda a, wt: K.linear_fp8(*a, *K.quantize_weight_fp8(wt))         # noqa: E731
    for li in range(cfg.n_layers):
        qkv = lin(K.rmsnorm_fp8(x, w.norm1[li], cfg.eps, add=down), w.wqkv[li])
        q = K.rope_cache_write(qkv, eng.inv, m.positions, m.slots, own.k[li], own.v[li], cfg.n_heads)
        ao = K.chunk_attention(q, own.k[li], own.v[li], tab, m.starts, m.ctx_lens, 70, 70,
                               scale=eng.scale)
        o = lin(K.quantize_fp8(ao.view(91, -1)), w.wo[li])
        gu = lin(K.rmsnorm_fp8(x, w.norm2[li], cfg.eps, add=o), w.wgu[li])
        down = lin(K.swiglu_fp8(gu), w.wd[li])
    x = (x.float() + down.float()).to(torch.bfloat16)
    assert torch.equal(x, eng.x) and torch.equal(cache.k, own.k) and torch.equal(cache.v, own.v)
    last = x[[69, 70, 90]]
    h = K.rmsnorm(last.contiguous(), w.norm_f, cfg.eps)
    assert out == K.greedy_argmax(torch.nn.functional.linear(h, w.lm_head)).tolist()
    # Beside 16-bit projections: an operand's rounding to e4m3 is at most 2^-4 of a value
    # (some 2.5 % rms), a product's two operands' some 3.6 % of its norm, eight products.
    ref_cache = _cache(cfg, cuda)
    ref = ChunkPrefill(w, ref_cache)
    ref.step(chunks)
    _near(eng.x, ref.x, 8 * 0.036)


def test_a_prefix_from_the_handoff_and_a_fork(cuda):
    """Pieces go on after KV that the handoff scattered, and after a fork."""
    cfg, w = _model(cuda)
    rng = np.random.default_rng(6)
    prompt = rng.integers(0, cfg.vocab, 90).tolist()
    cache, S = _cache(cfg, cuda), 64
    first, k, v = LlamaPrefill(w).forward(prompt[:50])
    cache.allocate("a", 50)
    cache.write_frame("a", K.pack_kv(k, v, 50, S), 50, S)
    cache.fork("a", ["b"], 50)
    eng = ChunkPrefill(w, cache)
    eng.step([("a", 50, prompt[50:]), ("b", 50, prompt[50:])])
    whole_k, whole_v = LlamaPrefill(w).forward(prompt)[1:]
    for r in "ab":
        got_k, got_v = _rows(cache, r, 90)
        _near(got_k, whole_k, SHARE)
        _near(got_v, whole_v, SHARE)
    assert cache.blocks("a")[:3] == cache.blocks("b")[:3] and cache.blocks("a")[3] != cache.blocks("b")[3]


def test_refusals(cuda):
    cfg, w = _model(cuda)
    cache = _cache(cfg, cuda, blocks=4)
    eng = ChunkPrefill(w, cache, max_tokens=100)
    for bad in ([], [("a", 0, [])], [("a", 0, [1000])], [("a", 0, [-1])], [("a", 0, [1] * 101)],
                [("a", 5, [1])], [("a", 0, [1]), ("a", 0, [1])]):
        with pytest.raises(ValueError):
            eng.step(bad)
    with pytest.raises(MemoryError):
        eng.step([("a", 0, [1] * 65)])
    assert cache.alloc.free_blocks() == 4
    many = ChunkPrefill(w, cache, max_tokens=5000)
    with pytest.raises(ValueError, match="4096 requests"):
        many.step([(i, 0, [1]) for i in range(4097)])
    assert cache.alloc.free_blocks() == 4
    with pytest.raises(ValueError, match="cache"):
        ChunkPrefill(w, PagedKVCache(1, 4, 2, 128, device=cuda))
    with pytest.raises(ValueError, match="max_tokens"):
        ChunkPrefill(w, cache, max_tokens=0)


def _near_best(tokens, rows, w, eps):
    """Each token's logit among those of its hidden row in 64 bits: h, rounded to bf16
    from 32 bits (norm and weight), is off by at most 2^-8 of itself and 2^-17 before
    that; a logit's sum of H products by H 2^-24 of their magnitudes and its rounding by
    2^-8; the largest and the token's may be off in opposite ways. How many rows have no
    other token as near."""
    x = rows.double()
    h = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.norm_f.double()
    head = w.lm_head.double().t().contiguous()
    logits, size = h @ head, h.abs() @ head.abs()
    off = (2.0 ** -8 + 2.0 ** -16 + x.shape[1] * 2.0 ** -24) * size + 2.0 ** -8 * logits.abs()
    best = (logits - off).amax(1, keepdim=True)
    near = logits + off >= best
    assert near.gather(1, torch.tensor(tokens, device=x.device)[:, None]).all()
    return int((near.sum(1) == 1).sum())


@pytest.mark.parametrize("fp8", [False, True])
def test_tokens_of_every_request(cuda, fp8):
    """The tokens that a step returns, request by request: with ``every`` those after each
    new token, without the last of them, and of its hidden rows the greedy ones."""
    cfg, w = _model(cuda)
    rng = np.random.default_rng(8)
    cache = _cache(cfg, cuda)
    eng = ChunkPrefill(w, cache, fp8=fp8)
    eng.step([(r, 0, rng.integers(0, cfg.vocab, n).tolist()) for r, n in (("a", 40), ("c", 3))])
    chunks = [(r, p, rng.integers(0, cfg.vocab, n).tolist())
              for r, p, n in (("a", 40, 7), ("b", 0, 33), ("c", 3, 1), ("d", 0, 18))]
    ends = np.cumsum([len(t) for *_, t in chunks])
    every, rows = eng.step(chunks, every=True), eng.x.clone()
    last, same = eng.step(chunks), eng.x.clone()
    assert [len(t) for t in every] == [7, 33, 1, 18] and rows.shape == same.shape == (59, cfg.hidden)
    # The same kernels and products on the same rows.
    h = K.rmsnorm(rows, w.norm_f, cfg.eps)
    want = K.greedy_argmax(torch.nn.functional.linear(h, w.lm_head)).tolist()
    assert every == [want[e - len(t):e] for e, (*_, t) in zip(ends, chunks)]
    h = K.rmsnorm(same[torch.tensor(ends - 1, device=cuda)].contiguous(), w.norm_f, cfg.eps)
    assert last == K.greedy_argmax(torch.nn.functional.linear(h, w.lm_head)).tolist()
    # In 64 bits.
    assert _near_best(sum(every, []), rows, w, cfg.eps) > 0
    alone = [_near_best([t], same[e - 1:e], w, cfg.eps) for t, e in zip(last, ends)]
    if torch.equal(rows, same):
        assert all(t[-1] == one for t, one, sure in zip(every, last, alone) if sure)
    _near(same, rows, SHARE)


def test_chunks_may_come_from_an_iterator(cuda):
    """As PagedKVCache.extend takes them, and tokens as an array."""
    cfg, w = _model(cuda)
    tokens = np.random.default_rng(9).integers(0, cfg.vocab, 30)
    one, two = (ChunkPrefill(w, _cache(cfg, cuda)) for _ in range(2))
    want = one.step([("a", 0, tokens.tolist()), ("b", 0, [7])])
    assert two.step((r, 0, t) for r, t in (("a", tokens), ("b", [7]))) == want
    assert torch.equal(one.x, two.x)
