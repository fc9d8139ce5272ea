"""torch-facing wrappers of the 8-bit projections: rows and weights in e4m3 with
32-bit scales, and their product.

A row x [K] is kept as e4m3 values and a scale for each 128 columns, a weight [N, K]
as e4m3 values and a scale for each block of 128 x 128 (the last rows' block may be
smaller): the value stands for itself times its scale. Scales of rows come as [T,
K / 128] with a group's lying together (strides 1 and T). The reference's
projections are 16-bit (kernels/decode_batch.py:73-91).
"""
import functools

import torch

from .. import _lib
from .handoff import BF16, _current_device, _need, launch_scope, need_device, stream_handle
from .prefill import overlap

FP8 = torch.float8_e4m3fn
GROUP = 128
TOP = 448.0                # the largest e4m3 value
LEAST = 2.0 ** -100        # a group's largest value counts as at least this


def _rows_of(t, name, dev, width=None):
    """(t, T, columns, row stride) of bf16 rows, copied where they are strided or off
    16 bytes in a way the kernels do not take."""
    _need(t, name)
    need_device(dev, t, name)
    if t.dim() != 2:
        raise ValueError(f"{name} must be [T, columns], got {tuple(t.shape)}")
    T, K = t.shape
    ld = t.stride(0) if T > 1 else K
    if (K > 1 and t.stride(1) != 1) or ld < K or ld % 8 or t.data_ptr() % 16:
        t, ld = t.clone(memory_format=torch.contiguous_format), K
    return t, T, K, ld


def _outputs(out, T, K, dev, others):
    """(values [T, K] e4m3, scales [T, K / 128] float32) of the caller's."""
    values, scales = out
    _need(values, "out values", FP8)
    _need(scales, "out scales", torch.float32)
    for t, name in ((values, "out values"), (scales, "out scales")):
        need_device(dev, t, name)
        if any(overlap(t, o) for o in others) or overlap(values, scales):
            raise ValueError(f"{name} must not overlap the other tensors")
    if tuple(values.shape) != (T, K) or not values.is_contiguous() or values.data_ptr() % 16:
        raise ValueError(f"out values must be contiguous and 16-byte aligned {(T, K)}")
    if tuple(scales.shape) != (T, K // GROUP) or not scales.t().is_contiguous():
        raise ValueError(f"out scales must be {(T, K // GROUP)} with a group's lying together")
    return values, scales


def rmsnorm_fp8(x, weight, eps, add=None, sum_out=None, out=None, stream=None):
    """RMSNorm over the last dim of x [T, H] bf16 in 8 bits -> (values [T, H] e4m3,
    scales [T, H / 128] float32).

    With ``add`` [T, H] the norm is of bf16(x + add), which is written to ``sum_out``
    (default: x itself, as rmsnorm does). y = x * rsqrt(mean(x^2) + eps) * weight is
    32-bit until it is 8: a group's scale is max(|y|, 2^-100) / 448, its values
    y / scale. H a multiple of 128 up to 8192."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError("x must be a CUDA tensor")
    dev = x.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return rmsnorm_fp8(x, weight, eps, add, sum_out, out)
    for t, name in ((weight, "weight"), (add, "add"), (sum_out, "sum_out")):
        if not isinstance(t, torch.Tensor) and (t is not None or name == "weight"):
            raise TypeError(f"{name} must be a CUDA tensor")
    # The usual operands pass one test; what does not is told apart.
    xp, wp, ap, sp = x.data_ptr(), weight.data_ptr(), None, None
    fine = x.dtype is BF16 and weight.dtype is BF16 and x.dim() == 2 and x.is_contiguous() \
        and weight.is_contiguous() and weight.device == dev and not (xp | wp) % 16
    T, H = x.shape if x.dim() == 2 else (0, 0)
    fine = fine and weight.numel() == H and H % GROUP == 0 and GROUP <= H <= 8192
    if add is not None:
        if sum_out is None:
            sum_out = x
        ap, sp, size = add.data_ptr(), sum_out.data_ptr(), 2 * T * H
        fine = fine and add.dtype is BF16 and sum_out.dtype is BF16 and add.shape == x.shape \
            and sum_out.shape == x.shape and add.is_contiguous() and sum_out.is_contiguous() \
            and add.device == dev and sum_out.device == dev and not (ap | sp) % 16 \
            and (sp == xp or sp >= xp + size or xp >= sp + size) \
            and (sp == ap or sp >= ap + size or ap >= sp + size) \
            and (sp >= wp + 2 * H or wp >= sp + size)
    if not fine or (add is None and sum_out is not None):
        _refuse_norm(x, weight, add, sum_out)
    if out is None:
        values = torch.empty((T, H), dtype=FP8, device=dev)
        scales = torch.empty_strided((T, H // GROUP), (1, T), dtype=torch.float32, device=dev)
    else:
        values, scales = _outputs(out, T, H, dev, [t for t in (x, weight, add, sum_out) if t is not None])
    if T:
        _lib.call("pdk_rmsnorm_fp8", xp, ap, wp, T, H, eps, sp, values.data_ptr(), scales.data_ptr(),
                  T, stream_handle())
    return values, scales


def _refuse_norm(x, weight, add, sum_out):
    """Raises for operands that rmsnorm_fp8's own test did not pass."""
    dev = x.device
    for t, name in ((x, "x"), (weight, "weight"), (add, "add"), (sum_out, "sum_out")):
        if t is None:
            continue
        _need(t, name)
        need_device(dev, t, name)
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous and 16-byte aligned")
    if x.dim() != 2:
        raise ValueError(f"x must be [T, H], got {tuple(x.shape)}")
    H = x.shape[1]
    if H % GROUP or not GROUP <= H <= 8192:
        raise ValueError(f"H={H} is no multiple of {GROUP} in [{GROUP}, 8192]")
    if weight.numel() != H:
        raise ValueError(f"weight must hold H={H} values")
    if add is None:
        raise ValueError("sum_out needs add")
    if add.shape != x.shape or sum_out.shape != x.shape:
        raise ValueError("add and sum_out must be shaped like x")
    raise ValueError("sum_out must be x or add itself, or overlap none of x, add and weight")


def _quantized(entry, x, gated, out, stream):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError("x must be a CUDA tensor")
    dev = x.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return _quantized(entry, x, gated, out, None)
    if x.dtype is BF16 and x.dim() == 2 and x.is_contiguous() and x.data_ptr() % 16 == 0 \
            and x.shape[1] % 8 == 0:
        (T, K), ld = x.shape, x.shape[1]
    else:
        x, T, K, ld = _rows_of(x, "x", dev)
    K, rest = divmod(K, 2) if gated else (K, 0)
    if rest or K % GROUP or K < GROUP:
        raise ValueError(f"the columns must be a multiple of {GROUP}{' for each half' * gated}")
    if out is None:
        values = torch.empty((T, K), dtype=FP8, device=dev)
        scales = torch.empty_strided((T, K // GROUP), (1, T), dtype=torch.float32, device=dev)
    else:
        values, scales = _outputs(out, T, K, dev, [x])
    if T:
        _lib.call(entry, x.data_ptr(), ld, T, K, values.data_ptr(), scales.data_ptr(), T,
                  stream_handle())
    return values, scales


def quantize_fp8(x, out=None, stream=None):
    """x [T, K] bf16 in 8 bits -> (values, scales) as rmsnorm_fp8's."""
    return _quantized("pdk_quantize_fp8", x, False, out, stream)


def swiglu_fp8(gate_up, out=None, stream=None):
    """silu(g) * u of gate_up = [g | u] [T, 2M] bf16, 32-bit until it is 8 -> (values
    [T, M], scales) as rmsnorm_fp8's."""
    return _quantized("pdk_swiglu_fp8", gate_up, True, out, stream)


@torch.no_grad()
def quantize_weight_fp8(w):
    """w [N, K] (K a multiple of 128) in 8 bits, a scale for each block of 128 x 128 ->
    (values [N, K] e4m3, scales [ceil(N / 128), K / 128] float32). For the loading of a
    model: torch operations, some rows at a time."""
    if not isinstance(w, torch.Tensor):
        raise TypeError("w must be a tensor")
    if w.dim() != 2 or w.shape[1] % GROUP or 0 in w.shape:
        raise ValueError(f"w must be [N, K] with K a multiple of {GROUP}, got {tuple(w.shape)}")
    N, K = w.shape
    values = torch.empty((N, K), dtype=FP8, device=w.device)
    scales = torch.empty((-(-N // GROUP), K // GROUP), dtype=torch.float32, device=w.device)
    step = GROUP * 32
    for at in range(0, N, step):
        part = w[at:at + step].float()
        n = part.shape[0]
        part = torch.nn.functional.pad(part, (0, 0, 0, -n % GROUP)).view(-1, GROUP, K // GROUP, GROUP)
        s = part.abs().amax((1, 3)).clamp(min=LEAST) / TOP
        scales[at // GROUP:at // GROUP + s.shape[0]] = s
        values[at:at + n] = (part / s[:, None, :, None]).view(-1, K)[:n].to(FP8)
    return values, scales


@functools.lru_cache(maxsize=4096)
def linear_fp8_workspace_bytes(T, K, N):
    """Bytes of linear_fp8's workspace (0: it needs none; 512 MiB at most); raises for sizes
    it does not take."""
    for v in (T, K, N):
        if not 0 <= v < 1 << 31:
            raise ValueError(f"size {v} outside [0, 2^31)")
    need = int(_lib.lib().pdk_linear_fp8_workspace_bytes(T, K, N))
    if need < 0:
        raise ValueError(_lib.last_error())
    return need


def linear_fp8(x, x_scales, w, w_scales, out=None, workspace=None, stream=None):
    """x . w^T of 8-bit rows and weights -> [T, N] bf16.

    x [T, K] e4m3 (unit column stride) with x_scales float32 [T, K / 128] (any positive
    strides), w [N, K] e4m3 contiguous with w_scales float32 [ceil(N / 128), K / 128]
    contiguous, as rmsnorm_fp8, quantize_fp8, swiglu_fp8 and quantize_weight_fp8 give
    them. A group's sums are 32-bit but for the matrix instruction's own cut: of 8
    columns' products what lies 2^-13 below the largest is lost (some 2e-4 of a result).
    They are scaled and added in 32 bits and rounded to bf16 once. K a multiple of 128,
    N of 8. ``workspace``: device memory of linear_fp8_workspace_bytes for one call at a
    time (default: allocated by the call)."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise TypeError("x must be a CUDA tensor")
    dev = x.device
    if stream is not None or dev.index != _current_device():
        with launch_scope(dev, stream):
            return linear_fp8(x, x_scales, w, w_scales, out, workspace)
    if not (isinstance(w, torch.Tensor) and isinstance(x_scales, torch.Tensor)
            and isinstance(w_scales, torch.Tensor) and x.dtype is FP8 and w.dtype is FP8
            and x_scales.dtype is torch.float32 and w_scales.dtype is torch.float32
            and w.device == dev and x_scales.device == dev and w_scales.device == dev):
        for t, name, dt in ((x, "x", FP8), (w, "w", FP8), (x_scales, "x_scales", torch.float32),
                            (w_scales, "w_scales", torch.float32)):
            _need(t, name, dt)
            need_device(dev, t, name)
    if x.dim() != 2 or w.dim() != 2 or x.shape[1] != w.shape[1]:
        raise ValueError(f"x [T, K] and w [N, K] expected, got {tuple(x.shape)}, {tuple(w.shape)}")
    (T, K), N = x.shape, w.shape[0]
    if K % GROUP or K < GROUP or N % 8 or N < 8:
        raise ValueError(f"K={K} must be a multiple of {GROUP}, N={N} of 8")
    if not w.is_contiguous() or w.data_ptr() % 16:
        raise ValueError("w must be contiguous and 16-byte aligned")
    groups = K // GROUP
    if x_scales.shape != (T, groups):
        raise ValueError(f"x_scales must be {(T, groups)}, got {tuple(x_scales.shape)}")
    if w_scales.shape != (-(-N // GROUP), groups) or not w_scales.is_contiguous():
        raise ValueError(f"w_scales must be contiguous {(-(-N // GROUP), groups)}")
    xs_t = x_scales.stride(0) if T > 1 else 1
    xs_g = x_scales.stride(1) if groups > 1 else 1
    if xs_t < 1 or xs_g < 1 or xs_t >= 1 << 21:
        x_scales, xs_t, xs_g = x_scales.contiguous(), groups, 1
    ld = x.stride(0) if T > 1 else K
    if x.stride(1) != 1 or ld < K or ld % 16 or ld >= 1 << 24 or x.data_ptr() % 16:
        x, ld = x.clone(memory_format=torch.contiguous_format), K
    if out is None:
        out = torch.empty((T, N), dtype=BF16, device=dev)
    else:
        _need(out, "out")
        need_device(dev, out, "out")
        if tuple(out.shape) != (T, N) or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"out must be contiguous and 16-byte aligned {(T, N)}")
        if any(overlap(out, t) for t in (x, x_scales, w, w_scales)):
            raise ValueError("out must not overlap the operands")
    need = linear_fp8_workspace_bytes(T, K, N)
    ws_ptr, ws_bytes = None, 0
    if workspace is not None:
        if not isinstance(workspace, torch.Tensor):
            raise TypeError("workspace must be a CUDA tensor")
        need_device(dev, workspace, "workspace")
        ws_ptr, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if not workspace.is_contiguous() or ws_bytes < need or ws_ptr % 16:
            raise ValueError(f"workspace must be contiguous, 16-byte aligned and hold {need} bytes")
        if any(overlap(workspace, t) for t in (x, x_scales, w, w_scales, out)):
            raise ValueError("workspace must not overlap the other tensors")
    elif need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
        ws_ptr, ws_bytes = workspace.data_ptr(), need
    if T:
        _lib.call("pdk_linear_fp8", x.data_ptr(), ld, x_scales.data_ptr(), xs_t, xs_g, w.data_ptr(),
                  w_scales.data_ptr(), T, K, N, ws_ptr, ws_bytes, out.data_ptr(), stream_handle())
    return out
