"""Workspaces of calls on streams other than the current one: nothing else is given
their memory while queued work uses it."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


def _busy(dev):
    """Some milliseconds of work on the current stream."""
    a = torch.ones((4096, 4096), device=dev)
    for _ in range(12):
        a = torch.matmul(a, a).clamp_(0, 1)
    return a


def _operands(dev, n, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=g, device=dev).to(torch.bfloat16)  # noqa: E731
    return mk(n, 8, D), mk(n, 2, D), mk(n, 2, D)


def _own(dev, sizes):
    """Tensors of the current stream filled with sevens, many of each size."""
    return [torch.full((n,), 7.0, device=dev) for n in sizes for _ in range(4)]


@pytest.mark.parametrize("window", [None, 1900])
def test_batched_attention_on_another_stream(cuda, window):
    """The workspace grows while the stream of the calls is still busy; memory that the
    current stream takes meanwhile keeps what is written there."""
    from rngd_pd_amd.engines.decode_batch import BatchDecodeAttention
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    cache = PagedKVCache(1, 140, 2, D, device=cuda, seed=1)
    cache.k.normal_()
    cache.v.normal_()
    cache.allocate("r", 2200)
    tab = cache.table("r")[None].contiguous()
    runs = [(700, 1), (2100, 2)]
    ctx = [torch.tensor([n], dtype=torch.int32, device=cuda) for n, _ in runs]
    ops = [_operands(cuda, 1, seed) for _, seed in runs]
    torch.cuda.synchronize()
    want = []
    for (n, _), c, (q, k, v) in zip(runs, ctx, ops):
        eng = BatchDecodeAttention(cache, n_q_heads=8, window=window)
        want.append(eng.layer_attention(0, q, k, v, tab, c, n))
    torch.cuda.synchronize()
    eng = BatchDecodeAttention(cache, n_q_heads=8, window=window)
    outs = [torch.empty_like(q) for q, _, _ in ops]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        busy = _busy(cuda)
    sizes = []
    for (n, _), c, (q, k, v), out in zip(runs, ctx, ops, outs):
        eng.layer_attention(0, q, k, v, tab, c, n, out=out, stream=side)
        sizes.append(eng._ws.buffer.numel())
    assert sizes[0] < sizes[1]
    own = _own(cuda, sizes)
    torch.cuda.synchronize()
    assert all(bool((t == 7).all()) for t in own)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    del busy


def test_workspace_of_a_captured_call_outlives_growth(cuda):
    """A graph of a split call replays right after a longer eager call has replaced
    the engine's workspace and its memory could have been given to others."""
    from rngd_pd_amd.engines.decode_batch import BatchDecodeAttention
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    cache = PagedKVCache(1, 140, 2, D, device=cuda, seed=1)
    cache.k.normal_()
    cache.v.normal_()
    cache.allocate("r", 2200)
    tab = cache.table("r")[None].contiguous()
    short, long = (torch.tensor([n], dtype=torch.int32, device=cuda) for n in (700, 2100))
    q, k, v = _operands(cuda, 1, 5)
    eng = BatchDecodeAttention(cache, n_q_heads=8)
    want = eng.layer_attention(0, q, k, v, tab, short, 700).clone()
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        eng.layer_attention(0, q, k, v, tab, short, 700, out=out)
    size = eng._ws.buffer.numel()
    eng.layer_attention(0, q, k, v, tab, long, 2100)
    own = _own(cuda, [size])
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(bool((t == 7).all()) for t in own)


def test_decoder_on_another_stream(cuda):
    """LlamaDecoder.step(stream=...) with contexts that outgrow its workspace."""
    from rngd_pd_amd.engines.llama_decode import LlamaConfig, LlamaDecoder, LlamaWeights
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    cfg = LlamaConfig(hidden=512, n_heads=8, n_kv_heads=2, head_dim=128, inter=1024, vocab=1000,
                      n_layers=2)
    weights = LlamaWeights.random(cfg, seed=3, device=cuda)
    cache = PagedKVCache(2, 140, 2, D, device=cuda, seed=1)
    cache.k.normal_()
    cache.v.normal_()
    cache.allocate("r", 2200)
    tab = cache.table("r")[None].contiguous()
    tok = torch.tensor([17], dtype=torch.int32, device=cuda)
    ctx = [torch.tensor([n], dtype=torch.int32, device=cuda) for n in (700, 2100)]
    dec = LlamaDecoder(weights, cache, max_batch=1)
    want = []
    for c, n in zip(ctx, (700, 2100)):
        dec.step(tok, c, tab, n)
        want.append(dec.logits.clone())
    dec = LlamaDecoder(weights, cache, max_batch=1)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got, sizes = [], []
    with torch.cuda.stream(side):
        busy = _busy(cuda)
    for c, n in zip(ctx, (700, 2100)):
        dec.step(tok, c, tab, n, stream=side)
        sizes.append(dec._ws.buffer.numel())
        with torch.cuda.stream(side):
            got.append(dec.logits.clone())
    own = _own(cuda, sizes)
    torch.cuda.synchronize()
    assert sizes[0] < sizes[1] and all(bool((t == 7).all()) for t in own)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del busy


def test_searches_keep_no_old_workspaces(cuda):
    """A search's graph goes with it, and so does the workspace it held when a longer
    search needs more."""
    from rngd_pd_amd.engines.beam_search import BeamSearch
    from rngd_pd_amd.engines.llama_decode import LlamaConfig, LlamaDecoder, LlamaWeights
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    cfg = LlamaConfig(hidden=512, n_heads=8, n_kv_heads=2, head_dim=128, inter=1024, vocab=1000,
                      n_layers=2)
    cache = PagedKVCache(2, 160, 2, D, device=cuda)
    dec = LlamaDecoder(LlamaWeights.random(cfg, seed=3, device=cuda), cache, max_batch=2)
    cache.allocate("r", 900)
    search, sizes = BeamSearch(dec, 2), []
    for n in (200, 500, 900):
        search.search([("r", n, 1)], 5)
        sizes.append(dec._ws.buffer.numel())
    assert sizes == sorted(set(sizes)) and dec._ws._kept == []
