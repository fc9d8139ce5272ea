"""A prompt under a window that hides nothing of it is the prompt without one, bit for
bit: keys, values and the first token."""
import numpy as np
import pytest
import torch

from tests.test_gpu_span_engines import _cfg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,spans", [
    (1, [(1, 0), (5, 3)]),
    (60, [(60, 0), (59, 1), (1, 59), (4096, 4)]),
    (700, [(700, 0), (500, 200), (1 << 40, 0), (2, (1 << 31) - 1)])])
def test_windows_that_hide_nothing(cuda, T, spans):
    from rngd_pd_amd.engines.llama_decode import LlamaWeights
    from rngd_pd_amd.engines.llama_prefill import LlamaPrefill
    tokens = np.random.default_rng(T).integers(0, 1000, T).tolist()

    def forward(window, sinks):
        cfg = _cfg(window=window, sinks=sinks)
        return LlamaPrefill(LlamaWeights.random(cfg, seed=3, device=cuda)).forward(tokens)
    first, k, v = forward(None, 0)
    for window, sinks in spans:
        got = forward(window, sinks)
        assert got[0] == first and torch.equal(got[1], k) and torch.equal(got[2], v), (window, sinks)
    if T > 1:                                           # one token less seen is another prompt
        assert not torch.equal(forward(T // 2, 0)[1], k)
