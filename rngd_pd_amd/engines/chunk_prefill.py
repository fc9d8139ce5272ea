"""Prefill in pieces, straight into the paged cache: each step takes any number of
next tokens of several requests through the model.

Stands beside LlamaPrefill (engines/prefill_full.py:337-388), which takes one prompt
from its first token and leaves rows for the handoff: here a request goes on from what
the cache holds of it, whoever wrote that (an earlier step, a handed-off prefix, a
decoder, a fork), so that long prompts come in pieces between decode steps, a next turn
costs its own tokens only, and a draft's tokens are verified in one pass. LlamaDecoder
reads the same cache from there on.

One step, with R requests and N tokens in all:

  blocks: PagedKVCache.extend; tables, positions and slots      chunk_map
  per layer
    h = rmsnorm(x + down)                                       rmsnorm or rmsnorm_fp8
    qkv = h . Wqkv^T                                            library or linear_fp8
    RoPE at the positions; K and V into the slots               rope_cache_write
    ao = attention over the cache                               chunk_attention
    o = ao . Wo^T                                               library or quantize_fp8, linear_fp8
    h = rmsnorm(x + o)                                          rmsnorm or rmsnorm_fp8
    gu = h . Wgu^T                                              library or linear_fp8
    act = silu(g) * u                                           swiglu or swiglu_fp8
    down = act . Wd^T                                           library or linear_fp8
  the greedy token of each request's last row                   library, greedy_argmax

With ``fp8`` the projections are 8-bit (e4m3 values; a scale for each 128 columns of a
row and each block of 128 x 128 of a weight), quantised once at the start; the lm_head
and everything between the projections stay 16- and 32-bit.
"""
import math

import numpy as np
import torch

from .. import kernels
from ..kernels.chunk import chunk_map, rope_cache_write, chunk_attention
from ..kernels.fp8 import (GROUP, linear_fp8, quantize_fp8, quantize_weight_fp8, rmsnorm_fp8,
                           swiglu_fp8)

BF16 = torch.bfloat16
MAX_REQUESTS = 4096        # chunk_map's
MAX_CONTEXT = 65535 * 16   # chunk_attention's


class ChunkPrefill:
    def __init__(self, weights, cache, max_tokens=8192, fp8=False):
        """``weights``: LlamaWeights (with ``fp8`` their projections are copied in 8
        bits); ``cache``: the PagedKVCache; ``max_tokens``: of one step, all requests
        together."""
        cfg = self.cfg = weights.cfg
        if (cache.n_layers, cache.n_kv_heads, cache.head_dim) != (cfg.n_layers, cfg.n_kv_heads,
                                                                  cfg.head_dim):
            raise ValueError("cache shape does not match the model")
        if cfg.head_dim != 128:
            raise ValueError("the chunk kernels need head_dim 128")
        if cfg.n_heads % cfg.n_kv_heads or cfg.n_heads // cfg.n_kv_heads > 16:
            raise ValueError(f"{cfg.n_heads} query heads for {cfg.n_kv_heads} KV heads: not 1 to 16 "
                             f"for each")
        widths = (cfg.hidden, cfg.n_heads * cfg.head_dim, cfg.inter)
        if fp8 and (any(w % GROUP for w in widths) or cfg.hidden > 8192):
            raise ValueError(f"8-bit projections need widths that are multiples of {GROUP} and "
                             f"hidden <= 8192, got {widths}")
        if not 1 <= max_tokens <= 1 << 20:
            raise ValueError(f"max_tokens={max_tokens} outside [1, 2^20]")
        self.w, self.cache, self.fp8, self.max_tokens = weights, cache, bool(fp8), max_tokens
        self.device = cache.k.device
        self.inv = cfg.inv_freq().to(self.device)
        self.scale = 1.0 / math.sqrt(cfg.head_dim)
        self._hidden = (None, None)
        self._layers = [(weights.wqkv[i], weights.wo[i], weights.wgu[i], weights.wd[i])
                        for i in range(cfg.n_layers)]
        if fp8:
            self._layers = [tuple(quantize_weight_fp8(w) for w in ws) for ws in self._layers]
            # The copies are written on the current stream; a step may run on another.
            torch.cuda.current_stream(self.device).synchronize()

    @property
    def x(self):
        """The hidden rows [N, hidden] of the last step, request after request, before the
        final norm."""
        x, down = self._hidden
        return x if down is None else x + down

    def _norm(self, x, weight, add):
        """rmsnorm(x + add) as a projection's input; with ``add``, x takes the sum."""
        if self.fp8:
            return rmsnorm_fp8(x, weight, self.cfg.eps, add=add)
        return (kernels.rmsnorm(x, weight, self.cfg.eps, add=add),)

    def _linear(self, x, w):
        return linear_fp8(*x, *w) if self.fp8 else torch.nn.functional.linear(x[0], w)

    def _rows(self, x):
        return quantize_fp8(x) if self.fp8 else (x,)

    def _swiglu(self, gu):
        if self.fp8:
            return swiglu_fp8(gu)
        M = self.cfg.inter
        if M % 8:
            return ((torch.nn.functional.silu(gu[:, :M].float()) * gu[:, M:].float()).to(BF16),)
        return (kernels.swiglu(gu),)

    def _upload(self, arrays):
        """Host int32 arrays on the device, in one copy."""
        flat = torch.from_numpy(np.concatenate([a.reshape(-1) for a in arrays])).to(self.device)
        parts = flat.split([a.size for a in arrays])
        return [p.view(a.shape) for p, a in zip(parts, arrays)]

    @torch.no_grad()
    def step(self, chunks, every=False):
        """One step on the current stream: ``chunks`` holds (req_id, tokens in the cache
        before, the next tokens' ids) of different requests. Returns the greedy next
        token of each (a list), or with ``every`` that after each of its new tokens (a list
        of lists; a draft's tokens are right as far as each equals the one before it).

        The requests' blocks are grown in the cache; what stands behind the tokens given as
        there (a rejected draft's) is written over."""
        cfg, w, cache = self.cfg, self.w, self.cache
        chunks = list(chunks)
        ids = [np.asarray(t, np.int64).reshape(-1) for _, _, t in chunks]
        lens = [(r, int(past), t.size) for (r, past, _), t in zip(chunks, ids)]
        N = sum(n for _, _, n in lens)
        if not lens or min(n for _, _, n in lens) < 1 or N > self.max_tokens:
            raise ValueError(f"a step takes 1 to {self.max_tokens} tokens, at least one per request")
        all_ids = np.concatenate(ids)
        if all_ids.min() < 0 or all_ids.max() >= cfg.vocab:
            raise ValueError(f"a token outside [0, {cfg.vocab})")
        # What the kernels would refuse is refused before the requests' blocks have grown.
        max_ctx = max(p + n for _, p, n in lens)
        if len(lens) > MAX_REQUESTS or max_ctx > MAX_CONTEXT or len(lens) * -(-max_ctx // 16) >= 1 << 27:
            raise ValueError(f"a step takes {MAX_REQUESTS} requests of {MAX_CONTEXT} tokens at most, "
                             f"and tables of fewer than 2^27 entries")
        with torch.cuda.device(self.device):
            tables, free = cache.extend(lens)
            past, new, tables, free, tokens = self._upload(
                [np.asarray([p for _, p, _ in lens], np.int32),
                 np.asarray([n for _, _, n in lens], np.int32), tables, free,
                 all_ids.astype(np.int32)])
            m = chunk_map(past, new, tables, free, N)
            max_new = max(n for _, _, n in lens)
            span = {"window": cfg.window, "sinks": min(cfg.sinks, max_ctx)} if cfg.window else {}
            x = w.embed.index_select(0, tokens)
            down = None
            for li, (wqkv, wo, wgu, wd) in enumerate(self._layers):
                qkv = self._linear(self._norm(x, w.norm1[li], down), wqkv)
                q = rope_cache_write(qkv, self.inv, m.positions, m.slots, cache.k[li], cache.v[li],
                                     cfg.n_heads)
                ao = chunk_attention(q, cache.k[li], cache.v[li], tables, m.starts, m.ctx_lens,
                                     max_new, max_ctx, scale=self.scale, **span)
                o = self._linear(self._rows(ao.view(N, -1)), wo)
                act = self._swiglu(self._linear(self._norm(x, w.norm2[li], o), wgu))
                down = self._linear(act, wd)
            self._hidden = (x, None if every else down)
            if not every:
                last = m.starts[1:].long() - 1
                x, down = x.index_select(0, last), down.index_select(0, last)
            h = kernels.rmsnorm(x, w.norm_f, cfg.eps, add=down)
            out = kernels.greedy_argmax(torch.nn.functional.linear(h, w.lm_head)).tolist()
        if not every:
            return out
        ends = np.cumsum([n for _, _, n in lens]).tolist()
        return [out[e - n:e] for e, (_, _, n) in zip(ends, lens)]
