"""Argument checks of the windowed attention, block copy and beam search entry
points of the C ABI: a bad call returns its code and a message before anything is
launched (the pointers are placeholders that nothing dereferences)."""
import ctypes

import numpy as np
import pytest

from rngd_pd_amd import _lib

P = 1 << 20                                       # 16-byte aligned placeholder address


def _window(**kw):
    a = dict(q=P, k_new=None, v_new=None, nb=64, mb=8, max_ctx=128, window=32, sinks=4, B=2, hq=32,
             hkv=8, d=128, scale=1.0, ws=P, ws_bytes=1 << 30)
    a.update(kw)
    return _lib.lib().pdk_decode_attn_window(
        a["q"], a["k_new"], a["v_new"], P, P, a["nb"], P, a["mb"], P, a["max_ctx"], a["window"],
        a["sinks"], a["B"], a["hq"], a["hkv"], a["d"], a["scale"], a["ws"], a["ws_bytes"], P, 0)


@pytest.mark.parametrize("kw,code,text", [
    (dict(window=0), _lib.PDK_EINVAL, "window"),
    (dict(sinks=-1), _lib.PDK_EINVAL, "sinks"),
    (dict(sinks=1 << 20), _lib.PDK_EINVAL, "sinks"),
    (dict(q=None), _lib.PDK_EINVAL, "null"),
    (dict(k_new=P), _lib.PDK_EINVAL, "together"),
    (dict(k_new=P + 2, v_new=P), _lib.PDK_EINVAL, "aligned"),
    (dict(d=64), _lib.PDK_ENOTSUP, "head_dim"),
    (dict(hq=17 * 8), _lib.PDK_ENOTSUP, "group"),
    (dict(hq=33), _lib.PDK_EINVAL, "multiple"),
    (dict(B=0), _lib.PDK_EINVAL, "B"),
    (dict(max_ctx=129), _lib.PDK_EINVAL, "max_ctx"),
    (dict(mb=5000, max_ctx=80000, window=16385, sinks=0), _lib.PDK_ENOTSUP, "16384"),
    (dict(mb=70000, max_ctx=128), _lib.PDK_EINVAL, "max_blocks"),
    (dict(scale=0.0), _lib.PDK_EINVAL, "scale"),
    (dict(mb=512, max_ctx=8192, window=2000, B=1, ws=None, ws_bytes=0), _lib.PDK_EINVAL, "workspace"),
])
def test_window_refusals(kw, code, text):
    assert _window(**kw) == code
    assert text in _lib.last_error()


def test_rope_window_refusals():
    lib = _lib.lib()

    def call(splits=2, window=8, sinks=0, d=128):
        return lib.pdk_decode_attn_rope_window(P, splits, P, P, P, 64, P, 8, P, 128, window, sinks, 2,
                                               32, 8, d, 1.0, P, 1 << 30, P, 0, 0, 0)
    assert call(splits=4) == _lib.PDK_EINVAL and "splits" in _lib.last_error()
    assert call(splits=0) == _lib.PDK_EINVAL
    assert call(window=0) == _lib.PDK_EINVAL
    assert call(sinks=-2) == _lib.PDK_EINVAL
    assert call(d=96) == _lib.PDK_ENOTSUP


def test_window_span():
    span = _lib.lib().pdk_decode_attn_window_span
    assert span(100, 5000, 4) == 100                  # never more than the context
    assert span(100000, 512, 0) == 512 + 31           # the first span may hold one token
    assert span(100000, 512, 1) == 512 + 31 + 32
    assert span(100000, 512, 33) == 512 + 31 + 64
    assert span(0, 1, 0) == 0 and span(9, 0, 0) == 0 and span(9, 1, -1) == 0
    assert span((1 << 31) - 1, (1 << 31) - 1, 0) == (1 << 31) - 1


def test_prefill_window_refusals():
    lib = _lib.lib()

    def call(T=64, hq=32, hkv=8, d=128, window=8, sinks=0, scale=1.0, ld=4096, q=P, k_ld=1024):
        return lib.pdk_prefill_attn_window(q, ld, P, k_ld, P, 1024, T, hq, hkv, d, scale, window, sinks,
                                           P, 0)
    assert call(window=0) == _lib.PDK_EINVAL and "window" in _lib.last_error()
    assert call(sinks=-1) == _lib.PDK_EINVAL
    assert call(T=0) == _lib.PDK_EINVAL
    assert call(d=64) == _lib.PDK_ENOTSUP
    assert call(hq=30) == _lib.PDK_EINVAL
    assert call(ld=4097) == _lib.PDK_EINVAL and call(ld=4088) == _lib.PDK_EINVAL
    assert call(scale=-1.0) == _lib.PDK_EINVAL
    assert call(q=P + 8) == _lib.PDK_EINVAL
    assert call(k_ld=1020) == _lib.PDK_EINVAL and call(k_ld=1016) == _lib.PDK_EINVAL
    assert call(hkv=0) == _lib.PDK_EINVAL and call(q=None) == _lib.PDK_EINVAL


def test_copy_blocks_refusals():
    lib = _lib.lib()

    def call(src, dst, k=P, stride=9 * 8 * 16 * 128, L=2, nb=9, h=8, d=128, n=None):
        s, t = np.asarray(src, np.int32), np.asarray(dst, np.int32)
        ptr = lambda a: a.ctypes.data_as(ctypes.c_void_p)   # noqa: E731
        return lib.pdk_copy_blocks(k, P, stride, L, nb, h, d, ptr(s), ptr(t),
                                   len(s) if n is None else n, 0)
    assert call([], []) == _lib.PDK_OK                        # nothing to do: nothing launched
    assert call([1, 2], [3, 3]) == _lib.PDK_EINVAL and "two pairs" in _lib.last_error()
    assert call([1, 3], [3, 4]) == _lib.PDK_EINVAL and "both" in _lib.last_error()
    assert call([4], [4]) == _lib.PDK_EINVAL
    assert call([0], [9]) == _lib.PDK_EINVAL and "outside" in _lib.last_error()
    assert call([-1], [2]) == _lib.PDK_EINVAL
    assert call([1], [2], n=-1) == _lib.PDK_EINVAL
    assert call([1], [2], k=None) == _lib.PDK_EINVAL
    assert call([1], [2], k=P + 8) == _lib.PDK_EINVAL
    assert call([1], [2], stride=9 * 8 * 16 * 128 - 8) == _lib.PDK_EINVAL
    assert call([1], [2], stride=9 * 8 * 16 * 128 + 4) == _lib.PDK_EINVAL
    assert call([1], [2], L=0) == _lib.PDK_EINVAL and call([1], [2], d=0) == _lib.PDK_EINVAL


def test_beam_refusals():
    lib = _lib.lib()

    def call(R=2, K=4, V=1000, n=4, elem=2, ld=None, logits=P, ws=P, ws_bytes=1 << 30, scores=P):
        return lib.pdk_beam_select(logits, elem, V if ld is None else ld, R, K, V, scores, None, 0, n,
                                   ws, ws_bytes, P, P, P, 0)
    assert call(K=17) == _lib.PDK_ENOTSUP and call(K=0) == _lib.PDK_ENOTSUP
    assert call(n=33) == _lib.PDK_ENOTSUP and call(n=0) == _lib.PDK_ENOTSUP
    assert call(R=0) == _lib.PDK_EINVAL and call(R=5000) == _lib.PDK_EINVAL
    assert call(V=0) == _lib.PDK_EINVAL and call(V=(1 << 20) + 1) == _lib.PDK_ENOTSUP
    assert call(elem=8) == _lib.PDK_EINVAL and call(ld=999) == _lib.PDK_EINVAL
    assert call(logits=P + 1) == _lib.PDK_EINVAL and call(logits=None) == _lib.PDK_EINVAL
    assert call(scores=None) == _lib.PDK_EINVAL
    need = lib.pdk_beam_select_workspace_bytes(2, 4, 1000, 4)
    assert need > 0
    assert call(ws_bytes=need - 1) == _lib.PDK_EINVAL and "workspace" in _lib.last_error()
    assert call(ws=P + 8) == _lib.PDK_EINVAL
    assert lib.pdk_beam_select_workspace_bytes(2, 17, 1000, 4) == 0

    def reorder(R=2, K=4, mb=8, L=2, nb=9, stride=9 * 8 * 16 * 128, h=8, d=128, k=P, parents=P):
        return lib.pdk_beam_reorder(parents, P, R, K, P, mb, k, P, stride, L, nb, h, d, 0)
    assert reorder(K=17) == _lib.PDK_ENOTSUP and reorder(K=0) == _lib.PDK_ENOTSUP
    assert reorder(R=0) == _lib.PDK_EINVAL and reorder(mb=0) == _lib.PDK_EINVAL
    assert reorder(stride=8) == _lib.PDK_EINVAL and reorder(k=P + 2) == _lib.PDK_EINVAL
    assert reorder(parents=None) == _lib.PDK_EINVAL and reorder(L=0) == _lib.PDK_EINVAL
