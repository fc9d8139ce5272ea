"""torch-facing wrapper of the copies of whole blocks inside the paged cache."""
import array

import numpy as np
import torch

from .. import _lib
from .handoff import BF16, _current_device, _need, launch_scope, need_device, stream_handle


def check_caches(cache_k, cache_v):
    """(layers, num_blocks, Hkv, D, layer stride) of cache_k [L, nb, Hkv, 16, D]
    and cache_v [L, nb, Hkv, D, 16], or of one layer's."""
    if cache_k.dtype is BF16 and cache_k.dim() == 5 and isinstance(cache_v, torch.Tensor):
        L, nb, H, block, D = cache_k.shape                # the usual whole cache, in one test
        if (block == 16 and cache_v.shape == (L, nb, H, D, 16) and cache_v.dtype is BF16
                and cache_v.device == cache_k.device and cache_k.is_contiguous()
                and cache_v.is_contiguous()):
            return L, nb, H, D, nb * H * 16 * D
    _need(cache_k, "cache_k")
    _need(cache_v, "cache_v")
    need_device(cache_k.device, cache_v, "cache_v")
    shape = tuple(cache_k.shape)
    if len(shape) not in (4, 5) or shape[-2] != 16:
        raise ValueError(f"cache_k must be [L, nb, Hkv, 16, D] or one layer's, got {shape}")
    L, (nb, H, _, D) = (shape[0] if len(shape) == 5 else 1), shape[-4:]
    if tuple(cache_v.shape) != shape[:-2] + (D, 16):
        raise ValueError(f"cache_v must be {shape[:-2] + (D, 16)}, got {tuple(cache_v.shape)}")
    layer = nb * H * 16 * D
    if len(shape) == 4 or L == 1:
        ok, stride = cache_k.is_contiguous() and cache_v.is_contiguous(), layer
    else:
        stride = cache_k.stride(0)
        ok = cache_k[0].is_contiguous() and cache_v[0].is_contiguous() \
            and cache_v.stride(0) == stride and stride >= layer
    if not ok:
        raise ValueError("each layer of the caches must be contiguous, K and V at one layer stride")
    return L, nb, H, D, stride


def _address(a):
    return a.__array_interface__["data"][0]


def _ids(ids, name, num_blocks):
    """Host block ids as int32."""
    if isinstance(ids, torch.Tensor) and ids.is_cuda:
        raise TypeError(f"{name} must be on the host (a list, a numpy array or a CPU tensor)")
    if type(ids) is np.ndarray and ids.dtype == np.int32 and ids.ndim == 1:
        return ids if ids.flags.c_contiguous else np.ascontiguousarray(ids)
    if type(ids) is list and ids:
        try:
            return np.frombuffer(array.array("i", ids), np.int32)
        except OverflowError:
            raise ValueError(f"{name} holds ids outside [0, {num_blocks})") from None
        except TypeError:
            raise TypeError(f"{name} must be a list of block ids") from None
    a = np.asarray(ids)
    if a.ndim != 1 or (a.size and a.dtype.kind not in "iu"):
        raise TypeError(f"{name} must be a list of block ids")
    if a.dtype != np.int32:
        if a.size and (a.min() < 0 or a.max() >= num_blocks):
            raise ValueError(f"{name} holds ids outside [0, {num_blocks})")
        a = a.astype(np.int32)
    return np.ascontiguousarray(a)


def copy_blocks(cache_k, cache_v, src, dst, stream=None):
    """Copy block src[i] to block dst[i] for every i, K and V of all layers, in
    one launch per 448 pairs.

    cache_k [L, nb, Hkv, 16, D] and cache_v [L, nb, Hkv, D, 16] bf16 (or one
    layer's). src, dst: equally long lists (numpy arrays, CPU tensors) of block
    ids, read during the call. One block may be copied to many; a destination
    that is another pair's destination or any pair's source is refused, so the
    result does not hang on an order."""
    if not isinstance(cache_k, torch.Tensor) or not cache_k.is_cuda:
        raise TypeError("cache_k must be a CUDA tensor")
    if stream is not None or cache_k.device.index != _current_device():
        with launch_scope(cache_k.device, stream):
            return copy_blocks(cache_k, cache_v, src, dst)
    L, nb, H, D, stride = check_caches(cache_k, cache_v)
    s, d = _ids(src, "src", nb), _ids(dst, "dst", nb)
    if s.size != d.size:
        raise ValueError(f"{s.size} sources for {d.size} destinations")
    if s.size:
        _lib.call("pdk_copy_blocks", cache_k.data_ptr(), cache_v.data_ptr(), stride, L, nb, H, D,
                  _address(s), _address(d), s.size, stream_handle())
