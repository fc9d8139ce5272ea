"""torch-facing wrappers of a step over several requests' next tokens on the paged
cache: pieces of prompts, drafts to be verified, single tokens, in one launch each.

The reference's prefill starts every prompt from nothing (engines/prefill_full.py:
337-388) and its decode takes one token per lane (engines/decode_batch.py:305-377);
these take any number of new tokens per request after what the cache holds of it.
"""
import functools
from typing import NamedTuple

import torch

from .. import _lib
from .attention import _check_layer_cache
from .handoff import BF16, _current_device, _need, launch_scope, need_device, stream_handle
from .prefill import check_window, overlap

HEAD_DIM = 128


class ChunkMap(NamedTuple):
    """Where the new tokens of a step's requests are; int32 tensors on the device."""
    starts: torch.Tensor       # [R + 1]: request r's tokens are starts[r] .. starts[r + 1] - 1
    ctx_lens: torch.Tensor     # [R]: what each request has with them
    positions: torch.Tensor    # [N]: of each token in its request; -1 behind the last
    slots: torch.Tensor        # [N]: block * 16 + place in the cache; -1 for none
    taken: torch.Tensor        # [1]: blocks needed of the free list


def _int32(t, name, dev, dims=1):
    if isinstance(t, torch.Tensor) and t.dtype is torch.int32 and t.device == dev \
            and t.dim() == dims and t.is_contiguous():
        return
    _need(t, name, torch.int32)
    need_device(dev, t, name)
    raise ValueError(f"{name} must be contiguous with {dims} dimension{'s' * (dims > 1)}")


def chunk_map(past, new, tables, free, max_tokens, stream=None):
    """Block tables and slots of a step, built on the device from the requests'
    lengths -> ChunkMap.

    past, new int32 [R]: the tokens that request r has in the cache and gets now
    (lengths outside [0, what its table holds] count as the nearest). tables int32
    [R, max_blocks] grows in place: where new tokens need a block beyond the
    ceil(past / 16) that are there, its entry takes the next of ``free`` (int32 [F]
    block ids), request after request. ``taken`` says how many that needs; where it is
    more than F the entries and slots left over are -1 (rope_cache_write skips those
    tokens, chunk_attention hides them), so a caller that cannot know compares.
    ``max_tokens``: the length of positions and slots, at least the sum of ``new``;
    tokens beyond it are left out. ``tables`` overlaps none of the others."""
    if not isinstance(tables, torch.Tensor) or not tables.is_cuda:
        raise TypeError("tables must be a CUDA tensor")
    dev = tables.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return chunk_map(past, new, tables, free, max_tokens)
    # The usual operands pass one test; what does not is told apart.
    if not (isinstance(past, torch.Tensor) and isinstance(new, torch.Tensor)
            and isinstance(free, torch.Tensor)
            and tables.dtype is past.dtype is new.dtype is free.dtype is torch.int32
            and past.device == new.device == free.device == dev
            and tables.dim() == 2 and past.dim() == new.dim() == free.dim() == 1
            and tables.is_contiguous() and past.is_contiguous() and new.is_contiguous()
            and free.is_contiguous()):
        _int32(tables, "tables", dev, 2)
        _int32(past, "past", dev)
        _int32(new, "new", dev)
        _int32(free, "free", dev)
    R, W = tables.shape
    if past.numel() != R or new.numel() != R:
        raise ValueError(f"past and new must hold {R} lengths")
    N = int(max_tokens)
    if not 0 <= N < 1 << 30:
        raise ValueError(f"max_tokens={N} outside [0, 2^30)")
    buf = torch.empty(2 * R + 2 + 2 * N, dtype=torch.int32, device=dev)
    out = ChunkMap(*buf.split_with_sizes([R + 1, R, N, N, 1]))
    at = buf.data_ptr()
    _lib.call("pdk_chunk_map", past.data_ptr(), new.data_ptr(), R, tables.data_ptr(), W,
              free.data_ptr(), free.numel(), N, at, at + 4 * (R + 1), at + 4 * (2 * R + 1),
              at + 4 * (2 * R + 1 + N), at + 4 * (2 * R + 1 + 2 * N), stream_handle())
    return out


def rope_cache_write(qkv, inv_freq, positions, slots, cache_k, cache_v, n_q_heads, q_out=None,
                     stream=None):
    """RoPE at ``positions`` and the keys and values into ``slots`` of one layer's
    cache -> the rotated q [N, n_q, 128] bf16.

    qkv bf16 [N, >= (n_q + 2 n_kv) * 128] (unit column stride) holds q, k, v;
    inv_freq float32 [64]; positions and slots int32 [N] (chunk_map's). A token whose
    slot lies outside the cache is not written; a position below 0 counts as 0. The
    angle is position * inv_freq exactly (rope_cache_append rounds it to 32 bits).
    Slots are different: of two tokens for one slot either may be left, or parts of
    both. Neither q_out nor the caches overlap another tensor of the call."""
    if not isinstance(qkv, torch.Tensor) or not qkv.is_cuda:
        raise TypeError("qkv must be a CUDA tensor")
    dev = qkv.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return rope_cache_write(qkv, inv_freq, positions, slots, cache_k, cache_v, n_q_heads,
                                    q_out)
    n_q_heads = int(n_q_heads)
    # The usual operands pass one test; what does not is told apart, or copied.
    others = (inv_freq, positions, slots, cache_k, cache_v)
    if not all(isinstance(t, torch.Tensor) and t.device == dev and t.is_contiguous() for t in others) \
            or not qkv.dtype is cache_k.dtype is cache_v.dtype is BF16 \
            or not positions.dtype is slots.dtype is torch.int32 \
            or inv_freq.dtype is not torch.float32:
        _refuse_write(qkv, *others)
    nb, H, D, N, width = _write_sizes(qkv, *others, n_q_heads)
    ld = qkv.stride(0) if N > 1 else max(qkv.shape[1], width) + 7 & ~7
    if ld < width or ld % 8 or qkv.data_ptr() % 16:
        qkv = qkv[:, :width].clone(memory_format=torch.contiguous_format)
        ld = width
    if q_out is None:
        q_out = torch.empty((N, n_q_heads, D), dtype=BF16, device=dev)
    else:
        _need(q_out, "q_out")
        need_device(dev, q_out, "q_out")
        if tuple(q_out.shape) != (N, n_q_heads, D) or not q_out.is_contiguous() \
                or q_out.data_ptr() % 16:
            raise ValueError(f"q_out must be contiguous and 16-byte aligned {(N, n_q_heads, D)}")
        if any(overlap(q_out, t) for t in (qkv, inv_freq, positions, slots, cache_k, cache_v)):
            raise ValueError("q_out must not overlap the other tensors")
    if N:
        _lib.call("pdk_rope_cache_write", qkv.data_ptr(), ld, inv_freq.data_ptr(),
                  positions.data_ptr(), slots.data_ptr(), N, n_q_heads, H, D, q_out.data_ptr(),
                  cache_k.data_ptr(), cache_v.data_ptr(), nb, stream_handle())
    return q_out


def _refuse_write(qkv, inv_freq, positions, slots, cache_k, cache_v):
    """Raises for operands that rope_cache_write's own test did not pass."""
    dev = qkv.device
    _need(qkv, "qkv")
    _check_layer_cache(cache_k, cache_v)
    _need(inv_freq, "inv_freq", torch.float32)
    for t, name in ((cache_k, "cache_k"), (cache_v, "cache_v"), (inv_freq, "inv_freq")):
        need_device(dev, t, name)
    if not inv_freq.is_contiguous():
        raise ValueError(f"inv_freq must hold head_dim/2 = {HEAD_DIM // 2} contiguous values")
    _int32(positions, "positions", dev)
    _int32(slots, "slots", dev)


def _write_sizes(qkv, inv_freq, positions, slots, cache_k, cache_v, n_q_heads):
    """(blocks, KV heads, head_dim, tokens, columns) of rope_cache_write's operands."""
    if cache_k.dim() != 4 or cache_k.shape[2] != 16 or cache_v.dim() != 4 \
            or positions.dim() != 1 or slots.dim() != 1:
        _refuse_write(qkv, inv_freq, positions, slots, cache_k, cache_v)
    nb, H, _, D = cache_k.shape
    if cache_v.shape != (nb, H, D, 16):
        raise ValueError(f"cache_v must be [nb, Hkv, D, 16], got {tuple(cache_v.shape)}")
    if D != HEAD_DIM:
        raise ValueError(f"head_dim must be {HEAD_DIM}, got {D}")
    if n_q_heads < 1:
        raise ValueError(f"n_q_heads must be >= 1, got {n_q_heads}")
    if qkv.dim() != 2 or (qkv.shape[1] > 1 and qkv.stride(1) != 1):
        raise ValueError("qkv must be [N, columns] with unit column stride")
    N, columns = qkv.shape
    width = (n_q_heads + 2 * H) * D
    if columns < width:
        raise ValueError(f"qkv rows hold {columns} values, need {width}")
    if inv_freq.numel() != D // 2:
        raise ValueError(f"inv_freq must hold head_dim/2 = {D // 2} contiguous values")
    for t, name in ((positions, "positions"), (slots, "slots")):
        if t.numel() != N:
            raise ValueError(f"{name} must hold {N} entries")
    return nb, H, D, N, width


@functools.lru_cache(maxsize=4096)
def chunk_workspace_bytes(N, R, max_new, max_ctx, n_q_heads, n_kv_heads, window=None, sinks=0):
    """Bytes of chunk_attention's workspace for these sizes (0: it needs none; 284 MB at
    most); raises for sizes it does not take."""
    window, sinks = check_window(window, sinks)
    for v in (N, R, max_new, max_ctx, n_q_heads, n_kv_heads):
        if not 0 <= v < 1 << 31:
            raise ValueError(f"size {v} outside [0, 2^31)")
    need = int(_lib.lib().pdk_chunk_attn_workspace_bytes(N, R, max_new, max_ctx, n_q_heads,
                                                         n_kv_heads, window, sinks))
    if need < 0:
        raise ValueError(_lib.last_error())
    return need


def _refuse_attention(q, cache_k, cache_v, block_tables, starts, ctx_lens):
    """Raises for operands that chunk_attention's own test did not pass."""
    dev = q.device
    _need(q, "q")
    D = _check_layer_cache(cache_k, cache_v)[2]
    need_device(dev, cache_k, "cache_k")
    need_device(dev, cache_v, "cache_v")
    _int32(block_tables, "block_tables", dev, 2)
    _int32(starts, "starts", dev)
    _int32(ctx_lens, "ctx_lens", dev)
    raise ValueError(f"q must be [N, Hq, {D}], got {tuple(q.shape)}")


def chunk_attention(q, cache_k, cache_v, block_tables, starts, ctx_lens, max_new, max_ctx,
                    scale=1.0, window=None, sinks=0, out=None, workspace=None, stream=None):
    """Causal GQA attention of every request's new tokens over all it has in one
    layer's cache, the new tokens' own keys and values among it -> out [N, Hq, 128].

    q bf16 [N, Hq, 128] after RoPE, rows starts[r] .. starts[r + 1] - 1 of request r
    (columns of a wider tensor are taken as they lie); block_tables int32 [R,
    max_blocks], starts int32 [R + 1] non-decreasing from 0, ctx_lens int32 [R] with
    the new tokens (chunk_map's). ``max_new`` and ``max_ctx`` (<= max_blocks * 16) are
    at least any request's new tokens and context. Token i of n stands at position p =
    ctx - n + i and sees the tokens t <= p; with ``window`` those with t > p - window
    or t < ``sinks``. Tokens beyond q's last row are left out, as chunk_map leaves out
    those beyond ``max_tokens``; the others stand where they are. Tokens in blocks that the table does not name (-1, or past it)
    are seen by nobody, and a token that sees nothing gets zeros. Rows behind the last
    request are left as they are. Any Hq/Hkv up to 16. fp32 between the products; a
    weight is rounded to bf16 once, as the product's operand. ``workspace``: device
    memory of chunk_workspace_bytes for one call at a time (default: allocated by the
    call)."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise TypeError("q must be a CUDA tensor")
    dev = q.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return chunk_attention(q, cache_k, cache_v, block_tables, starts, ctx_lens, max_new,
                                   max_ctx, scale, window, sinks, out, workspace)
    # The usual operands pass one test; what does not is told apart.
    if not (isinstance(cache_k, torch.Tensor) and isinstance(cache_v, torch.Tensor)
            and isinstance(block_tables, torch.Tensor) and isinstance(starts, torch.Tensor)
            and isinstance(ctx_lens, torch.Tensor)
            and q.dtype is cache_k.dtype is cache_v.dtype is BF16
            and block_tables.dtype is starts.dtype is ctx_lens.dtype is torch.int32
            and cache_k.device == cache_v.device == block_tables.device == starts.device
            == ctx_lens.device == dev
            and q.dim() == 3 and cache_k.dim() == cache_v.dim() == 4 and block_tables.dim() == 2
            and starts.dim() == ctx_lens.dim() == 1
            and cache_k.is_contiguous() and cache_v.is_contiguous() and block_tables.is_contiguous()
            and starts.is_contiguous() and ctx_lens.is_contiguous()):
        _refuse_attention(q, cache_k, cache_v, block_tables, starts, ctx_lens)
    nb, H, size, D = cache_k.shape
    if size != 16 or cache_v.shape != (nb, H, D, 16):
        _check_layer_cache(cache_k, cache_v)
    if q.shape[2] != D:
        raise ValueError(f"q must be [N, Hq, {D}], got {tuple(q.shape)}")
    if D != HEAD_DIM:
        raise ValueError(f"head_dim must be {HEAD_DIM}, got {D}")
    N, Hq, _ = q.shape
    if H == 0 or Hq % H or not 1 <= Hq // H <= 16:
        raise ValueError(f"{Hq} query heads for {H} KV heads: not 1 to 16 for each")
    ld = q.stride(0) if N > 1 else Hq * D
    if q.stride(2) != 1 or (Hq > 1 and q.stride(1) != D) or ld < Hq * D or ld % 8 \
            or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        ld = Hq * D
    R, W = block_tables.shape
    if starts.numel() != R + 1 or ctx_lens.numel() != R:
        raise ValueError(f"starts and ctx_lens must hold {R + 1} and {R} entries")
    if out is None:
        out = torch.empty((N, Hq, D), dtype=BF16, device=dev)
    else:
        _need(out, "out")
        need_device(dev, out, "out")
        if tuple(out.shape) != (N, Hq, D) or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"out must be contiguous and 16-byte aligned {(N, Hq, D)}")
        if any(overlap(out, t) for t in (q, cache_k, cache_v, block_tables, starts, ctx_lens)):
            raise ValueError("out must not overlap what the call reads")
    max_new, max_ctx = int(max_new), int(max_ctx)
    if max_new < 0 or not 1 <= max_ctx <= W * 16:
        raise ValueError(f"max_new={max_new} below 0 or max_ctx={max_ctx} outside [1, {W * 16}]")
    need = chunk_workspace_bytes(N, R, max_new, max_ctx, Hq, H, window, sinks)
    window, sinks = check_window(window, sinks)
    ws_ptr, ws_bytes = None, 0
    if workspace is not None:
        if not isinstance(workspace, torch.Tensor):
            raise TypeError("workspace must be a CUDA tensor")
        need_device(dev, workspace, "workspace")
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if not workspace.is_contiguous() or ws_bytes < need or ws_ptr % 16:
            raise ValueError(f"workspace must be contiguous, 16-byte aligned and hold {need} bytes")
        if any(overlap(workspace, t) for t in (q, out, cache_k, cache_v, block_tables, starts,
                                               ctx_lens)):
            raise ValueError("workspace must not overlap the other tensors")
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        ws_ptr, ws_bytes = workspace.data_ptr(), need
    if N and max_new:
        _lib.call("pdk_chunk_attn", q.data_ptr(), ld, cache_k.data_ptr(), cache_v.data_ptr(), nb,
                  block_tables.data_ptr(), W, starts.data_ptr(), ctx_lens.data_ptr(), N, R, max_new,
                  max_ctx, Hq, H, D, float(scale), window, sinks, ws_ptr, ws_bytes, out.data_ptr(),
                  stream_handle())
    return out
