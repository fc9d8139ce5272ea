"""Engines whose sinks cover more than any context: prompts and decode steps see all."""
import numpy as np
import pytest
import torch

from tests.test_gpu_span_engines import D, _cfg, _decoder, _feed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sinks", [16385, (1 << 31) - 1])
def test_decoder_and_prefill(cuda, sinks):
    from rngd_pd_amd.engines.llama_decode import LlamaWeights
    from rngd_pd_amd.engines.llama_prefill import LlamaPrefill
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    tokens = np.random.default_rng(6).integers(0, 1000, 60).tolist()
    logits, keys = [], []
    for window, n in ((None, 0), (5, sinks)):
        cfg = _cfg(window=window, sinks=n)
        cache = PagedKVCache(2, 8, 2, D, device=cuda, seed=2)
        logits.append(_feed(_decoder(cfg, cache, max_batch=1), cache, "r", tokens))
        keys.append(LlamaPrefill(LlamaWeights.random(cfg, seed=3, device=cuda)).forward(tokens)[1])
    assert torch.equal(logits[0], logits[1])
    # (Two ways of rounding a prompt's weights.)
    assert (keys[0].float() - keys[1].float()).norm() <= 2e-2 * keys[0].float().norm()


def test_batched_attention(cuda):
    from rngd_pd_amd.engines.decode_batch import BatchDecodeAttention
    from rngd_pd_amd.engines.paged_cache import PagedKVCache
    outs = []
    for window, sinks in ((600, 0), (5, 20000)):        # all 600 tokens are seen
        cache = PagedKVCache(1, 80, 2, D, device=cuda, seed=3)
        g = torch.Generator(device=cuda).manual_seed(1)
        cache.k.normal_(generator=g)
        cache.v.normal_(generator=g)
        eng = BatchDecodeAttention(cache, n_q_heads=8, window=window, sinks=sinks)
        cache.allocate("r", 599)
        eng.admit_loaded("r", 599)
        q = torch.randn((1, 8, D), generator=g, device=cuda).to(torch.bfloat16)
        kn, vn = (torch.randn((1, 2, D), generator=g, device=cuda).to(torch.bfloat16) for _ in range(2))
        outs.append(eng.layer_attention(0, q, kn, vn, *eng.prepare(["r"])))
        assert eng.trim(["r"]) == 0
    assert torch.equal(outs[0], outs[1])
