"""More sinks than a decode launch takes, in an engine whose contexts are short (host
logic; the launch is a stand-in)."""
import pytest
import torch

from rngd_pd_amd.engines import decode_batch as db
from rngd_pd_amd.engines.paged_cache import PagedKVCache


@pytest.mark.parametrize("sinks", [3, 20000, (1 << 31) - 1])
def test_sinks_beyond_the_context(monkeypatch, sinks):
    seen = {}
    monkeypatch.setattr(db._attn, "decode_attention_append", lambda *a, **kw: seen.update(kw))
    eng = db.BatchDecodeAttention(PagedKVCache(1, 4, 2, 128, device="cpu"), n_q_heads=8, window=5,
                                  sinks=sinks)
    eng.layer_attention(0, torch.zeros((1, 8, 128)), None, None, None, None, 100)
    assert seen["window"] == 5 and seen["sinks"] == min(sinks, 100)
