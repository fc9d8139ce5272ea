"""BatchDecodeAttention while its cache changes between steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("window", [None, 40])
def test_attention_across_compactions(cuda, window):
    """Steps of two streams, with blocks of retired requests compacted away and given
    to new ones in between: the results of an engine whose blocks stay where they are."""
    from rngd_pd_amd.engines.decode_batch import BatchDecodeAttention
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    engines = []
    for _ in range(2):
        cache = PagedKVCache(1, 40, 2, D, device=cuda, seed=3)
        eng = BatchDecodeAttention(cache, n_q_heads=8, window=window, sinks=3 if window else 0)
        for r, n in (("x", 70), ("a", 60), ("y", 33), ("b", 20)):
            cache.allocate(r, n)
            eng.admit_loaded(r, n)
        g = torch.Generator(device=cuda).manual_seed(1)
        cache.k.normal_(generator=g)
        cache.v.normal_(generator=g)
        engines.append(eng)
    ids = ["a", "b"]
    moved = 0
    for step in range(24):
        if step in (3, 9):
            for eng in engines:
                eng.retire("x" if step == 3 else "y")
            cache = engines[1].cache
            moved += cache.compact()
            # What was moved away from is somebody else's now.
            cache.allocate(("new", step), 64)
            held = cache.table(("new", step)).long()
            cache.k[:, held] = float("nan")
            cache.v[:, held] = float("nan")
        g = torch.Generator(device=cuda).manual_seed(step)
        q = torch.randn((2, 8, D), generator=g, device=cuda).to(torch.bfloat16)
        kn, vn = (torch.randn((2, 2, D), generator=g, device=cuda).to(torch.bfloat16)
                  for _ in range(2))
        outs = []
        for eng in engines:
            tables, ctx, max_ctx = eng.prepare(ids)
            outs.append(eng.layer_attention(0, q, kn, vn, tables, ctx, max_ctx))
            eng.advance(ids)
        assert torch.equal(outs[0], outs[1]), step
    assert moved > 0
