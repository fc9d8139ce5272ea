"""torch-facing wrapper of the prompt's attention."""
import torch

from .. import _lib
from .handoff import BF16, _current_device, _need, launch_scope, need_device, stream_handle

HEAD_DIM = 128


def check_window(window, sinks):
    """(window, sinks) as the C entry points take them; window None or a positive
    int (as long as any context beyond 2^30), sinks only with a window."""
    if window is None:
        if sinks:
            raise ValueError("sinks need a window")
        return 0, 0
    window, sinks = int(window), int(sinks)
    if window < 1 or not 0 <= sinks < 1 << 31:
        raise ValueError(f"window must be >= 1 and sinks in [0, 2^31), got {window}, {sinks}")
    return min(window, 1 << 30), sinks


def _rows(t, T):
    """t [T, heads, 128] with contiguous [heads, 128], 16-byte aligned rows, and
    its token stride; a copy where it is laid out otherwise."""
    heads, D = t.shape[1:]
    ld = t.stride(0) if T > 1 else heads * D
    if t.stride(2) != 1 or (heads > 1 and t.stride(1) != D) or ld < heads * D or ld % 8 \
            or ld >= 1 << 24 or t.data_ptr() % 16:
        t, ld = t.clone(memory_format=torch.contiguous_format), heads * D
    return t, ld


def overlap(a, b):
    """Whether the memory that a and b span has bytes in common."""
    def span(t):
        size = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
        return t.data_ptr(), t.data_ptr() + size * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def prefill_attention(q, k, v, scale=1.0, window=None, sinks=0, out=None, stream=None):
    """Causal GQA attention over one prompt of T tokens -> out [T, Hq, 128] bf16.

    q [T, Hq, 128], k and v [T, Hkv, 128] bf16, after RoPE (query head h reads KV
    head h // (Hq/Hkv)); columns of one projection's tensor are taken as they lie,
    other layouts than contiguous [heads, 128] rows are copied first. With
    ``window`` the query at position p sees the tokens t <= p with t > p - window
    or t < ``sinks``. fp32 between the products; a weight is rounded to bf16 once,
    as the product's operand (LlamaPrefill's own prompts without a window keep 32
    bits of it, from K and V laid out for that)."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise TypeError("q must be a CUDA tensor")
    dev = q.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return prefill_attention(q, k, v, scale, window, sinks, out)
    window, sinks = check_window(window, sinks)
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        _need(t, name)
        need_device(dev, t, name)
        if t.dim() != 3 or t.shape[0] != q.shape[0]:
            raise ValueError(f"{name} must be [T, heads, {HEAD_DIM}], got {tuple(t.shape)}")
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    if k.shape != v.shape or k.shape[2] != D:
        raise ValueError("k and v must be [T, Hkv, D] with q's head_dim")
    if out is None:
        out = torch.empty((T, Hq, D), dtype=BF16, device=dev)
    else:
        _need(out, "out")
        need_device(dev, out, "out")
        if out.shape != q.shape or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"out must be contiguous and 16-byte aligned {tuple(q.shape)}")
        if any(overlap(out, t) for t in (q, k, v)):
            raise ValueError("out must not overlap q, k or v")
    if T == 0:
        return out
    (q, q_ld), (k, k_ld), (v, v_ld) = _rows(q, T), _rows(k, T), _rows(v, T)
    _lib.call("pdk_prefill_attn_window", q.data_ptr(), q_ld, k.data_ptr(), k_ld, v.data_ptr(), v_ld,
              T, Hq, Hkv, D, scale, window or T, sinks, out.data_ptr(), stream_handle())
    return out
