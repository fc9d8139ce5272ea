"""torch-facing wrappers of beam search on the paged cache: the selection over
beams and vocabulary, and the cache's reordering after it.

The reference decodes greedily (greedy_tokens, engines/decode_batch.py:162-171);
these stand beside greedy_argmax.
"""
import functools

import torch

from .. import _lib
from .handoff import _current_device, _need, launch_scope, need_device, stream_handle
from .pages import check_caches

MAX_BEAMS = 16
MAX_OUT = 32


def beam_select(logits, scores, n_out=None, eos=None, last_tokens=None, out=None, workspace=None,
                stream=None):
    """The ``n_out`` best continuations (default: as many as beams) of each of R
    requests' K beams -> (tokens, parents, scores), each [R, n_out] (int32, int32,
    float32) in order.

    logits bf16 or float32 [R*K, V] (unit column stride; row r*K + k is beam k of
    request r), scores float32 [R, K] contiguous: the beams' summed log
    probabilities. A continuation's total is the beam's score + logit - the row's
    log-sum-exp, in 64 bits (exponentials good to 6e-11: totals nearer than about
    1e-10 may change places), rounded once in the returned scores; the lower beam,
    then the lower token, comes first among equals (inside a beam the logits
    decide). With ``eos`` and ``last_tokens`` (int32, R*K of them, contiguous) a
    beam whose last token is eos has ended: it stays in the race as the one
    candidate (eos, its score). Logits of -inf are no candidates, nor is anything
    of a beam whose score is not finite or whose logits hold a NaN or +inf or
    nothing above -inf; places that no candidate fills hold token -1, parent -1
    and score -inf.

    ``out``: the three tensors to write; with n_out = K they may be last_tokens and
    scores themselves (each request's are read before they are written). Other
    overlaps of theirs, or of the workspace, are refused.
    ``workspace``: at least
    beam_select_workspace_bytes of device memory for one call at a time (default:
    allocated by the call on its stream)."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda:
        raise TypeError("logits must be a CUDA tensor")
    dev = logits.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return beam_select(logits, scores, n_out, eos, last_tokens, out, workspace)
    if logits.dtype is not torch.bfloat16 and logits.dtype is not torch.float32:
        raise TypeError(f"logits must be bfloat16 or float32, got {logits.dtype}")
    _need(scores, "scores", torch.float32)
    need_device(dev, scores, "scores")
    if scores.dim() != 2 or not scores.is_contiguous():
        raise ValueError("scores must be contiguous [R, K]")
    R, K = scores.shape
    rows = R * K
    if logits.dim() != 2 or logits.shape[0] != rows or rows == 0 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [R*K = {rows}, V], got {tuple(logits.shape)}")
    V = logits.shape[1]
    ld = logits.stride(0) if rows > 1 else V
    if (V > 1 and logits.stride(1) != 1) or ld < V:
        raise ValueError("logits must have unit column stride and rows that do not overlap")
    n = K if n_out is None else int(n_out)
    if (eos is None) != (last_tokens is None):
        raise ValueError("eos and last_tokens come together")
    last = None
    if eos is not None:
        eos = int(eos)
        if not -(1 << 31) <= eos < 1 << 31:
            raise ValueError(f"eos={eos} is no int32")
        _need(last_tokens, "last_tokens", torch.int32)
        need_device(dev, last_tokens, "last_tokens")
        if last_tokens.numel() != rows or not last_tokens.is_contiguous():
            raise ValueError(f"last_tokens must be contiguous int32, {rows} of them")
        last = last_tokens.data_ptr()
    need = beam_select_workspace_bytes(R, K, V, n)
    if out is None:
        out = (scores.new_empty((R, n), dtype=torch.int32),
               scores.new_empty((R, n), dtype=torch.int32), scores.new_empty((R, n)))
    else:
        for t, name, dt in zip(out, ("tokens", "parents", "scores"),
                               (torch.int32, torch.int32, torch.float32)):
            _need(t, f"out {name}", dt)
            need_device(dev, t, f"out {name}")
            if t.numel() != R * n or not t.is_contiguous():
                raise ValueError(f"out {name} must be contiguous, {R * n} values")
    if workspace is None:
        workspace, ws_bytes = scores.new_empty(need // 4), need   # a multiple of 8
    else:
        need_device(dev, workspace, "workspace")
        ws_bytes = workspace.numel() * workspace.element_size()
        if not workspace.is_contiguous() or ws_bytes < need:
            raise ValueError(f"workspace holds fewer than the {need} bytes needed")
    tokens, parents, totals = out
    _lib.call("pdk_beam_select", logits.data_ptr(), logits.element_size(), ld, R, K, V,
              scores.data_ptr(), last, eos or 0, n, workspace.data_ptr(), ws_bytes,
              tokens.data_ptr(), parents.data_ptr(), totals.data_ptr(), stream_handle())
    return tokens, parents, totals


@functools.lru_cache(maxsize=1024)
def beam_select_workspace_bytes(R, K, V, n):
    """Bytes of beam_select's workspace; raises for sizes it does not take."""
    for name, v in (("R", R), ("K", K), ("V", V), ("n_out", n)):
        if not 1 <= v < 1 << 31:
            raise ValueError(f"{name}={v} outside [1, 2^31)")
    need = int(_lib.lib().pdk_beam_select_workspace_bytes(R, K, V, n))
    if not need:
        raise ValueError(_lib.last_error())
    return need


def beam_reorder(parents, ctx_lens, tables, cache_k, cache_v, stream=None):
    """The paged cache follows a selection, in place: beam k of request r goes on
    as ``parents``[r, k] (int32 [R, K] contiguous; outside [0, K): as itself).

    ``tables`` int32 [R*K, max_blocks] contiguous (row r*K + k is beam k's),
    ``ctx_lens`` int32 [R*K] the tokens the cache holds, the same for a request's
    beams (the first one's is read). Entries of full blocks become the parent's:
    those blocks are shared from then on and never written again. Where ctx is no
    multiple of 16 the block at entry ctx // 16, which must be the beam's own,
    takes the contents of the parent's there, in all layers of cache_k [L, nb,
    Hkv, 16, D] and cache_v [L, nb, Hkv, D, 16] (or one layer's), as if all were
    read before any is written."""
    if not isinstance(cache_k, torch.Tensor) or not cache_k.is_cuda:
        raise TypeError("cache_k must be a CUDA tensor")
    dev = cache_k.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return beam_reorder(parents, ctx_lens, tables, cache_k, cache_v)
    L, nb, H, D, stride = check_caches(cache_k, cache_v)
    for t, name in ((parents, "parents"), (ctx_lens, "ctx_lens"), (tables, "tables")):
        _need(t, name, torch.int32)
        need_device(dev, t, name)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if parents.dim() != 2:
        raise ValueError("parents must be [R, K]")
    R, K = parents.shape
    if tables.dim() != 2 or tables.shape[0] != R * K or ctx_lens.numel() != R * K:
        raise ValueError(f"tables [R*K, max_blocks] and ctx_lens [R*K] need R*K = {R * K} rows")
    _lib.call("pdk_beam_reorder", parents.data_ptr(), ctx_lens.data_ptr(), R, K, tables.data_ptr(),
              tables.shape[1], cache_k.data_ptr(), cache_v.data_ptr(), stride, L, nb, H, D,
              stream_handle())
