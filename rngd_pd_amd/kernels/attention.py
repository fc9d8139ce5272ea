"""torch-facing wrappers of decode attention, cache append and greedy argmax.

Replaces the attention slice of DecodeLayer.forward (kernels/decode_batch.py:81-85),
softmax_dsl (kernels/dsl_batch.py:73-86) and greedy_tokens
(engines/decode_batch.py:162-171) with HIP kernels over the paged cache.
"""
import functools

import torch

from .. import _lib
from .handoff import _current_device, _need, launch_scope, need_device, stream_handle
from .prefill import check_window, overlap

BF16 = torch.bfloat16


@functools.lru_cache(maxsize=4096)
def workspace_bytes(B, n_q_heads, max_ctx, head_dim=128):
    return int(_lib.lib().pdk_decode_attn_workspace_bytes(B, n_q_heads, max_ctx, head_dim))


class Workspace:
    """The attention workspace of a caller that makes many calls: one fp32 buffer,
    replaced when a call needs more.

    It holds the per-split partial maxima, sums and outputs of a split context;
    every entry a call reads is written earlier in that call, so it is neither
    cleared nor filled. It serves one stream at a time: a caller that goes from one
    to another orders them. A buffer is allocated on the stream of the call that
    needs it; one that was replaced is given out again only when what was queued
    on the streams that used it is done, and not at all if a graph being captured
    used it (the graph holds its address)."""

    def __init__(self, device):
        self.device = torch.device(device)
        self.buffer = None
        self._bytes = 0                      # of the buffer
        self._streams = set()                # handles of the streams that used it
        self._in_graph = False
        self._kept = []

    def _new(self, nbytes):
        return torch.empty(nbytes // 4 + 64, dtype=torch.float32, device=self.device)

    def holds(self, nbytes):
        return self._bytes >= nbytes

    def take(self, nbytes, stream=None):
        """The buffer, of at least ``nbytes``, for a call on ``stream`` (default: the
        current one); None where it needs none."""
        if not nbytes:
            return None
        # The usual call: large enough, and nothing new about the stream.
        if self._bytes >= nbytes and stream is None and self.device.index == _current_device() \
                and stream_handle() in self._streams \
                and (self._in_graph or not torch.cuda.is_current_stream_capturing()):
            return self.buffer
        with launch_scope(self.device, stream):
            on = stream_handle()
            if not self.holds(nbytes):
                if self._in_graph:
                    self._kept.append(self.buffer)
                self.buffer = self._new(nbytes)
                self._bytes = self.buffer.numel() * 4
                self._streams, self._in_graph = {on}, False
            elif on not in self._streams:
                self.buffer.record_stream(torch.cuda.current_stream(self.device))
                self._streams.add(on)
            self._in_graph = self._in_graph or torch.cuda.is_current_stream_capturing()
            return self.buffer

    def graphs(self):
        """What graphs hold of it now, for graphs_gone."""
        return self.buffer, self._in_graph

    def graphs_gone(self, before):
        """The graphs that were captured since graphs() returned ``before`` are gone."""
        self._in_graph = before[1] and self.buffer is before[0]


_WORKSPACES = {}


def get_workspace(nbytes, device, stream=None):
    """The Workspace kept per device: at least ``nbytes`` of it for a call on
    ``stream`` (default: the current one). Concurrent calls on different streams
    need their own."""
    key = torch.device(device).index
    if key is None:
        key = _current_device()
    ws = _WORKSPACES.get(key)
    if ws is None:
        ws = _WORKSPACES[key] = Workspace(torch.device("cuda", key))
    return ws.take(max(nbytes, 1 << 20), stream)


def _check_layer_cache(cache_k, cache_v):
    _need(cache_k, "cache_k")
    _need(cache_v, "cache_v")
    if cache_k.dim() != 4 or cache_k.shape[2] != 16:
        raise ValueError(f"cache_k must be one layer [nb, Hkv, 16, D], got {tuple(cache_k.shape)}")
    nb, H, _, D = cache_k.shape
    if tuple(cache_v.shape) != (nb, H, D, 16):
        raise ValueError(f"cache_v must be [nb, Hkv, D, 16], got {tuple(cache_v.shape)}")
    if not (cache_k.is_contiguous() and cache_v.is_contiguous()):
        raise ValueError("paged caches must be contiguous")
    return nb, H, D


def _attention_call(q, cache_k, cache_v, block_tables, ctx_lens, max_ctx, out, workspace,
                    stream=None, span=None):
    """Checked operands of one attention call: (geometry, workspace pointer and
    bytes, out). ``span``: the tokens read at most, under a window; such a call's
    workspace is its own where none is given."""
    _need(q, "q")
    nb, H, D = _check_layer_cache(cache_k, cache_v)
    if q.dim() != 3 or q.shape[2] != D or not q.is_contiguous():
        raise ValueError(f"q must be contiguous [B, Hq, {D}], got {tuple(q.shape)}")
    B, Hq, _ = q.shape
    _need(block_tables, "block_tables", torch.int32)
    _need(ctx_lens, "ctx_lens", torch.int32)
    if block_tables.dim() != 2 or block_tables.shape[0] != B or not block_tables.is_contiguous():
        raise ValueError("block_tables must be contiguous int32 [B, max_blocks]")
    if ctx_lens.numel() != B:
        raise ValueError("ctx_lens must hold B entries")
    if out is None:
        out = torch.empty_like(q)
    need = workspace_bytes(B, Hq, span or max_ctx, D)
    ws = None
    if need:
        if workspace is not None:
            if workspace.numel() * workspace.element_size() < need:
                raise ValueError(f"workspace holds fewer than the {need} bytes needed")
            ws = workspace
        elif span is not None:
            ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        else:
            ws = get_workspace(need, q.device, stream)
    ws_ptr = ws.data_ptr() if ws is not None else None
    ws_bytes = ws.numel() * ws.element_size() if ws is not None else 0
    return (nb, B, Hq, H, D), ws_ptr, ws_bytes, out


def window_span(max_ctx, window=None, sinks=0):
    """The most tokens that a stream of up to ``max_ctx`` reads under a window with
    sinks, in whole 32-token spans: workspace_bytes of it is what such a call
    needs. max_ctx itself without a window."""
    window, sinks = check_window(window, sinks)
    if not window:
        return max_ctx
    n = int(_lib.lib().pdk_decode_attn_window_span(int(max_ctx), window, sinks))
    if not n:
        raise ValueError(f"max_ctx={max_ctx}, window={window}, sinks={sinks} out of range")
    return n


@functools.lru_cache(maxsize=4096)
def _window_plan(B, Hq, D, max_ctx, capacity, window, sinks):
    """(window, sinks) as the C call takes them and the workspace's bytes."""
    if not 1 <= max_ctx <= capacity:
        raise ValueError(f"max_ctx={max_ctx} outside [1, {capacity}]")
    span = window_span(max_ctx, window, sinks)
    return (*check_window(window, sinks), workspace_bytes(B, Hq, span, D))


def _check_window_operands(q, new, cache_k, cache_v, block_tables, ctx_lens, out, workspace):
    """Raises for operands that _window_attention's own test did not pass."""
    for t, name in ((cache_k, "cache_k"), (cache_v, "cache_v"), (block_tables, "block_tables"),
                    (ctx_lens, "ctx_lens")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a CUDA tensor")
        need_device(q.device, t, name)
    if not ctx_lens.is_contiguous():
        raise ValueError("ctx_lens must be contiguous")
    # Shapes and types; the workspace is another matter.
    _attention_call(q, cache_k, cache_v, block_tables, ctx_lens, 1, q, None, span=1)
    B, H, D = q.shape[0], cache_k.shape[1], q.shape[2]
    for t, name in zip(new or (), ("k_new", "v_new")):
        _need(t, name)
        need_device(q.device, t, name)
        if tuple(t.shape) != (B, H, D):
            raise ValueError("k_new/v_new must be [B, Hkv, D]")
    if out is not None:
        _need(out, "out")
        need_device(q.device, out, "out")
        if out.shape != q.shape or not out.is_contiguous():
            raise ValueError(f"out must be contiguous {tuple(q.shape)}")
        if overlap(out, q):
            raise ValueError("out must not overlap q")
    if workspace is not None:
        need_device(q.device, workspace, "workspace")
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")


def _rows16(t):
    """t itself, or a copy where its rows are strided or off 16 bytes."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _window_attention(q, new, cache_k, cache_v, block_tables, ctx_lens, max_ctx, scale, out,
                      workspace, stream, window, sinks):
    """decode_attention (new None) or decode_attention_append (new (k, v)) under a
    window."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise TypeError("q must be a CUDA tensor")
    dev, at = q.device, q.get_device()
    if stream is not None or at != _current_device():
        with launch_scope(dev, stream):
            return _window_attention(q, new, cache_k, cache_v, block_tables, ctx_lens, max_ctx,
                                     scale, out, workspace, None, window, sinks)
    # The usual operands pass one test; what does not is told apart.
    try:
        B, Hq, D = q.shape
        nb, H, block, _ = cache_k.shape
        fine = (q.dtype is BF16 and cache_k.dtype is BF16 and cache_v.dtype is BF16
                and block_tables.dtype is torch.int32 and ctx_lens.dtype is torch.int32
                and cache_k.get_device() == at and cache_v.get_device() == at
                and block_tables.get_device() == at and ctx_lens.get_device() == at
                and cache_k.shape == (nb, H, 16, D) and cache_v.shape == (nb, H, D, 16)
                and block_tables.shape[0] == B and block_tables.dim() == 2
                and ctx_lens.numel() == B and q.is_contiguous() and cache_k.is_contiguous()
                and cache_v.is_contiguous() and block_tables.is_contiguous()
                and ctx_lens.is_contiguous() and out is None and workspace is None)
        if fine and new is not None:
            k_new, v_new = new
            fine = (k_new.dtype is BF16 and v_new.dtype is BF16 and k_new.get_device() == at
                    and v_new.get_device() == at and k_new.shape == (B, H, D)
                    and v_new.shape == (B, H, D))
    except (AttributeError, TypeError, ValueError):
        fine = False
    if not fine:
        _check_window_operands(q, new, cache_k, cache_v, block_tables, ctx_lens, out, workspace)
    width = block_tables.shape[1]
    window, sinks, need = _window_plan(B, Hq, D, int(max_ctx), width * 16,
                                       None if window is None else int(window), int(sinks))
    if out is None:
        out = torch.empty_like(q)
    ws_ptr, ws_bytes = None, 0
    if need:
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if ws_bytes < need:
            raise ValueError(f"workspace holds fewer than the {need} bytes needed")
    kp = vp = None
    if new is not None:
        k_new, v_new = _rows16(new[0]), _rows16(new[1])
        kp, vp = k_new.data_ptr(), v_new.data_ptr()
    _lib.call("pdk_decode_attn_window", q.data_ptr(), kp, vp, cache_k.data_ptr(),
              cache_v.data_ptr(), nb, block_tables.data_ptr(), width, ctx_lens.data_ptr(),
              int(max_ctx), window, sinks, B, Hq, H, D, scale, ws_ptr, ws_bytes, out.data_ptr(),
              stream_handle())
    return out


def decode_attention(q, cache_k, cache_v, block_tables, ctx_lens, max_ctx, scale=1.0,
                     out=None, workspace=None, stream=None, window=None, sinks=0):
    """GQA decode attention for one layer.

    q [B, Hq, D] bf16 (query head h reads KV head h // (Hq/Hkv)); cache_k
    [nb, Hkv, 16, D] (tiled K blocks), cache_v [nb, Hkv, D, 16]; block_tables int32 [B, max_blocks]
    and ctx_lens int32 [B] on the device; ``max_ctx`` >= every ctx_lens[b].

    With ``window`` stream b sees only its last ``window`` tokens and the first
    ``sinks`` (up to 16384): no block between them is read (its table entry may be -1), contexts
    may be as long as the table, and any Hq/Hkv up to 16 is taken. Without
    ``workspace`` such a call allocates its own."""
    if window is not None or sinks:
        return _window_attention(q, None, cache_k, cache_v, block_tables, ctx_lens, max_ctx, scale,
                                 out, workspace, stream, window, sinks)
    (nb, B, Hq, H, D), ws_ptr, ws_bytes, out = _attention_call(
        q, cache_k, cache_v, block_tables, ctx_lens, max_ctx, out, workspace, stream)
    _lib.call("pdk_decode_attn", q.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(), nb,
              block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), int(max_ctx),
              B, Hq, H, D, float(scale), ws_ptr, ws_bytes, out.data_ptr(), stream_handle(stream))
    return out


def decode_attention_append(q, k_new, v_new, cache_k, cache_v, block_tables, ctx_lens, max_ctx,
                            scale=1.0, out=None, workspace=None, stream=None, window=None, sinks=0):
    """cache_append(k_new, v_new) then decode_attention, in one launch where the
    kernel takes it (head_dim 128, 16-byte aligned rows, up to 64 streams), with
    the same results bit for bit, also where streams' tables share the blocks
    that the new tokens go to. k_new, v_new bf16 [B, Hkv, D]. ``window`` and
    ``sinks`` as decode_attention's."""
    if window is not None or sinks:
        return _window_attention(q, (k_new, v_new), cache_k, cache_v, block_tables, ctx_lens,
                                 max_ctx, scale, out, workspace, stream, window, sinks)
    _need(k_new, "k_new")
    _need(v_new, "v_new")
    nb, H, D = _check_layer_cache(cache_k, cache_v)
    B = k_new.shape[0]
    if tuple(k_new.shape) != (B, H, D) or tuple(v_new.shape) != (B, H, D):
        raise ValueError("k_new/v_new must be [B, Hkv, D]")
    k_new, v_new = k_new.contiguous(), v_new.contiguous()
    if D != 128 or B != q.shape[0] or k_new.data_ptr() % 16 or v_new.data_ptr() % 16:
        cache_append(k_new, v_new, cache_k, cache_v, block_tables, ctx_lens, stream=stream)
        return decode_attention(q, cache_k, cache_v, block_tables, ctx_lens, max_ctx, scale=scale,
                                out=out, workspace=workspace, stream=stream)
    (nb, B, Hq, H, D), ws_ptr, ws_bytes, out = _attention_call(
        q, cache_k, cache_v, block_tables, ctx_lens, max_ctx, out, workspace, stream)
    _lib.call("pdk_decode_attn_append", q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(),
              cache_k.data_ptr(), cache_v.data_ptr(), nb, block_tables.data_ptr(),
              block_tables.shape[1], ctx_lens.data_ptr(), int(max_ctx), B, Hq, H, D, float(scale),
              ws_ptr, ws_bytes, out.data_ptr(), stream_handle(stream))
    return out


def decode_attention_rope(qkv_partials, inv_freq, cache_k, cache_v, block_tables, ctx_lens,
                          max_ctx, n_q_heads, scale=1.0, out=None, workspace=None, stream=None,
                          plan_batch=0, ssq=None, eps=None):
    """RoPE, the new token's cache write and attention for one layer in one launch.

    qkv_partials float32 [splits, B, (n_q + 2 n_kv) D] (split-K partial sums of
    the q|k|v projection, splits in {1, 2, 4}); inv_freq float32 [D/2]. Same
    result, bit for bit, as rope_cache_append_partials then decode_attention.
    ``plan_batch`` (>= B; 0 means B) is the batch size the split plan is chosen
    for: equal plan_batch gives each stream the same result whatever B is."""
    _need(qkv_partials, "qkv_partials", torch.float32)
    _need(inv_freq, "inv_freq", torch.float32)
    nb, H, D = _check_layer_cache(cache_k, cache_v)
    if qkv_partials.dim() != 3 or not qkv_partials.is_contiguous():
        raise ValueError("qkv_partials must be contiguous [splits, B, N]")
    splits, B, N = qkv_partials.shape
    if N != (n_q_heads + 2 * H) * D:
        raise ValueError(f"qkv_partials rows hold {N} values, need {(n_q_heads + 2 * H) * D}")
    if inv_freq.numel() != D // 2:
        raise ValueError(f"inv_freq must hold head_dim/2 = {D // 2} values")
    _need(block_tables, "block_tables", torch.int32)
    _need(ctx_lens, "ctx_lens", torch.int32)
    if block_tables.dim() != 2 or block_tables.shape[0] != B or not block_tables.is_contiguous():
        raise ValueError("block_tables must be contiguous int32 [B, max_blocks]")
    if ctx_lens.numel() != B:
        raise ValueError("ctx_lens must hold B entries")
    if out is None:
        out = torch.empty((B, n_q_heads, D), dtype=cache_k.dtype, device=cache_k.device)
    need = workspace_bytes(B, n_q_heads, max_ctx, D)
    ws = None
    if need:
        if workspace is not None:
            if workspace.numel() * workspace.element_size() < need:
                raise ValueError(f"workspace holds fewer than the {need} bytes needed")
            ws = workspace
        else:
            ws = get_workspace(need, cache_k.device, stream)
    if ssq is not None:
        _need(ssq, "ssq", torch.float32)
        if ssq.dim() != 2 or ssq.shape[0] != B or not ssq.is_contiguous():
            raise ValueError(f"ssq must be contiguous float32 [{B}, H/16]")
        _lib.call("pdk_decode_attn_rope_rms", qkv_partials.data_ptr(), splits, ssq.data_ptr(),
                  ssq.shape[1], float(eps), inv_freq.data_ptr(), cache_k.data_ptr(),
                  cache_v.data_ptr(), nb, block_tables.data_ptr(), block_tables.shape[1],
                  ctx_lens.data_ptr(), int(max_ctx), B, n_q_heads, H, D, float(scale),
                  ws.data_ptr() if ws is not None else None,
                  ws.numel() * ws.element_size() if ws is not None else 0, out.data_ptr(),
                  int(plan_batch), stream_handle(stream))
        return out
    _lib.call("pdk_decode_attn_rope", qkv_partials.data_ptr(), splits, inv_freq.data_ptr(),
              cache_k.data_ptr(), cache_v.data_ptr(), nb, block_tables.data_ptr(),
              block_tables.shape[1], ctx_lens.data_ptr(), int(max_ctx), B, n_q_heads, H, D,
              float(scale), ws.data_ptr() if ws is not None else None,
              ws.numel() * ws.element_size() if ws is not None else 0, out.data_ptr(),
              int(plan_batch), stream_handle(stream))
    return out


def attn_read_probe(cache_k, cache_v, block_tables, ctx_lens, max_ctx, n_q_heads, out,
                    stream=None):
    """Decode attention's launch with its K/V loads and none of its arithmetic
    (pdk_attn_read_probe): what attention's access pattern costs by itself.
    ``out`` [B, n_q_heads, D] bf16 receives meaningless values."""
    nb, H, D = _check_layer_cache(cache_k, cache_v)
    B = block_tables.shape[0]
    _need(out, "out")
    if tuple(out.shape) != (B, n_q_heads, D):
        raise ValueError(f"out must be [B, n_q_heads, {D}]")
    _lib.call("pdk_attn_read_probe", cache_k.data_ptr(), cache_v.data_ptr(), nb,
              block_tables.data_ptr(), block_tables.shape[1], ctx_lens.data_ptr(), int(max_ctx),
              B, int(n_q_heads), H, D, out.data_ptr(), stream_handle(stream))
    return out


def cache_append(k_new, v_new, cache_k, cache_v, block_tables, ctx_lens, stream=None):
    """Write each stream's new k/v [B, Hkv, D] at slot ctx_lens[b]-1
    (the one-hot injection of kernels/decode_batch.py:81-82)."""
    _need(k_new, "k_new")
    _need(v_new, "v_new")
    nb, H, D = _check_layer_cache(cache_k, cache_v)
    B = k_new.shape[0]
    if tuple(k_new.shape) != (B, H, D) or tuple(v_new.shape) != (B, H, D):
        raise ValueError("k_new/v_new must be [B, Hkv, D]")
    _lib.call("pdk_cache_append", k_new.contiguous().data_ptr(), v_new.contiguous().data_ptr(),
              cache_k.data_ptr(), cache_v.data_ptr(), nb, block_tables.data_ptr(),
              block_tables.shape[1], ctx_lens.data_ptr(), B, H, D, stream_handle(stream))


def greedy_argmax(logits, out=None, stream=None):
    """First-maximum argmax per row of bf16 logits [B, V] -> int32 [B]."""
    _need(logits, "logits")
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be [B, V] with unit column stride")
    B, V = logits.shape
    if out is None:
        out = torch.empty(B, dtype=torch.int32, device=logits.device)
    _lib.call("pdk_greedy_argmax", logits.data_ptr(), B, V, logits.stride(0), out.data_ptr(),
              stream_handle(stream))
    return out
