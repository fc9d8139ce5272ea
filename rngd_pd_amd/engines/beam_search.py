"""Beam search over a decoder and its paged cache.

Each request's K beams are rows of the decoder's batch. They share the prompt's
full blocks (PagedKVCache.fork) and own the blocks of what they generate. A step
is the decoder's step, beam_select over its logits and beam_reorder of the block
tables and partly filled blocks; everything stays on the device, so the steps
after the first replay one captured graph, and the host reads the choices once at
the end (and, with an end token, now and then to see whether every beam has
ended).

A beam that has chosen ``eos`` stays in the race with its score: the search ends
with the K best of ended and running beams. The reference decodes greedily
(greedy_tokens, engines/decode_batch.py:162-171).
"""
import torch

from ..kernels import beam as _beam


class BeamSearch:
    """decoder: engines.llama_decode.LlamaDecoder; ``n_beams`` up to 16, with
    n_beams x requests <= decoder.max_batch."""

    def __init__(self, decoder, n_beams, eos=None, use_graphs=True, check_every=16):
        if not 1 <= n_beams <= _beam.MAX_BEAMS:
            raise ValueError(f"n_beams={n_beams} outside [1, {_beam.MAX_BEAMS}]")
        self.dec, self.cache = decoder, decoder.cache
        self.K, self.eos = n_beams, eos
        self.use_graphs, self.check_every = use_graphs, max(1, check_every)

    def search(self, requests, max_new, length_penalty=0.0):
        """requests: [(req_id, num_tokens, last_token)], each with the prompt's
        first num_tokens - 1 tokens (at least) in the cache under req_id and its
        last token, whose step gives the first logits. Returns, per request, its
        beams as (tokens, score) from the best: up to ``max_new`` tokens, cut after
        the end token; score the summed log probability, over
        len(tokens) ** length_penalty. The requests keep their blocks; the beams'
        own go back to the pool."""
        R, K = len(requests), self.K
        if R < 1 or R * K > self.dec.max_batch:
            raise ValueError(f"{R} requests of {K} beams for a decoder of {self.dec.max_batch} rows")
        if max_new < 1 or any(n < 1 for _, n, _ in requests):
            raise ValueError("max_new and the prompts' lengths must be at least 1")
        with torch.cuda.device(self.dec.device):
            return self._search(requests, max_new, length_penalty)

    def _search(self, requests, max_new, length_penalty):
        R, K = len(requests), self.K
        rows = [[("beam", req, k) for k in range(K)] for req, _, _ in requests]
        ids = [r for row in rows for r in row]
        captured, graphs = self.dec._captured, self.dec._ws.graphs()
        forked = []
        try:
            for (req, n, _), row in zip(requests, rows):
                self.cache.fork(req, row, n - 1)
                forked += row
                for r in row:
                    self.cache.ensure(r, n + max_new - 1)
            hist_tokens, hist_parents, scores = self._run(requests, ids, max_new)
        finally:
            # What was queued may still use the blocks: they go back when it is done.
            torch.cuda.synchronize(self.dec.device)
            self.dec._captured = captured                # this search's graph is gone
            self.dec._ws.graphs_gone(graphs)
            for r in forked:
                self.cache.free(r)
        return [self._beams(hist_tokens[:, r], hist_parents[:, r], scores[r], length_penalty)
                for r in range(R)]

    def _run(self, requests, ids, max_new):
        """The steps; tokens and parents [steps, R, K] and scores [R, K] on the host."""
        dec, R, K, dev = self.dec, len(requests), self.K, self.dec.device
        B = R * K
        i32 = dict(dtype=torch.int32, device=dev)
        tokens = torch.tensor([[t] * K for _, _, t in requests], **i32)
        ctx = torch.tensor([n for _, n, _ in requests for _ in range(K)], **i32)
        tables = self.cache.batch_tables(ids)
        max_ctx = tables.shape[1] * 16
        # All beams are alike before the first step: only the first one counts.
        scores = torch.full((R, K), float("-inf"), device=dev)
        scores[:, 0] = 0.0
        parents = torch.zeros((R, K), **i32)
        hist = torch.empty((2, max_new, R, K), **i32)
        vocab = dec.cfg.vocab
        ws = torch.empty(_beam.beam_select_workspace_bytes(R, K, vocab, K), dtype=torch.uint8,
                         device=dev)
        dec.reserve(max_ctx)

        def step(end):
            dec.step(tokens.view(-1), ctx, tables, max_ctx)
            _beam.beam_select(dec.logits[:B], scores, K, **end, out=(tokens, parents, scores),
                              workspace=ws)
            _beam.beam_reorder(parents, ctx, tables, self.cache.k, self.cache.v)
            ctx.add_(1)

        # The prompt's last token may be the end token: no beam has ended yet.
        step({})
        hist[0, 0].copy_(tokens)
        hist[1, 0].copy_(parents)
        end = {} if self.eos is None else {"eos": self.eos, "last_tokens": tokens}
        graph, done = None, 1
        for t in range(1, max_new):
            if self.use_graphs and graph is None and t > 1:
                graph = torch.cuda.CUDAGraph()
                dec._captured = True                     # its workspace may not move any more
                with torch.cuda.graph(graph, capture_error_mode="thread_local"):
                    step(end)
            if graph is None:
                step(end)
            else:
                graph.replay()
            hist[0, t].copy_(tokens)
            hist[1, t].copy_(parents)
            done = t + 1
            if self.eos is not None and done % self.check_every == 0 \
                    and bool(((tokens == self.eos) | (tokens < 0)).all()):
                break
        out = hist[:, :done].cpu().numpy()
        return out[0], out[1], scores.cpu().numpy()

    def _beams(self, tokens, parents, scores, length_penalty):
        """One request's beams, followed back from the last step."""
        found = []
        for k in range(self.K):
            if scores[k] == float("-inf"):
                continue
            seq, at = [], k
            for t in range(len(tokens) - 1, -1, -1):
                seq.append(int(tokens[t, at]))
                at = int(parents[t, at])
            seq.reverse()
            if self.eos is not None and self.eos in seq:
                seq = seq[:seq.index(self.eos) + 1]
            found.append((seq, float(scores[k]) / len(seq) ** length_penalty))
        return sorted(found, key=lambda b: -b[1])         # stable: the search's order among equals


__all__ = ["BeamSearch"]
