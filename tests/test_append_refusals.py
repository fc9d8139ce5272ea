"""A call of the fused append and attention that is refused writes nothing, also where
it would take two launches: the attention's arguments are checked before the append
(the pointers are placeholders; without a GPU a launch fails with PDK_EHIP)."""
import pytest
import torch

from rngd_pd_amd import _lib

P = 1 << 20
BAD = [
    (dict(d=64), _lib.PDK_ENOTSUP, "head_dim"),
    (dict(hq=17 * 8), _lib.PDK_ENOTSUP, "group"),
    (dict(max_ctx=129), _lib.PDK_EINVAL, "max_ctx"),
    (dict(scale=0.0), _lib.PDK_EINVAL, "scale"),
    (dict(scale=float("nan")), _lib.PDK_EINVAL, "scale"),
    (dict(mb=1024, max_ctx=16384, ws=None, ws_bytes=0), _lib.PDK_EINVAL, "workspace"),
    (dict(mb=2048, max_ctx=16385 + 4000), _lib.PDK_ENOTSUP, "16384"),
]


def _call(window, B, out=P, q=P + (1 << 30), **kw):
    a = dict(mb=8, max_ctx=128, hq=32, hkv=8, d=128, scale=1.0, ws=P, ws_bytes=1 << 30)
    a.update(kw)
    tail = (B, a["hq"], a["hkv"], a["d"], a["scale"], a["ws"], a["ws_bytes"], out, 0)
    head = (q, P, P, P, P, 64, P, a["mb"], P, a["max_ctx"])
    if window:
        return _lib.lib().pdk_decode_attn_window(*head, window, 0, *tail)
    return _lib.lib().pdk_decode_attn_append(*head, *tail)


@pytest.mark.skipif(torch.cuda.is_available(), reason="placeholder pointers")
@pytest.mark.parametrize("window", [0, 1 << 20])
@pytest.mark.parametrize("B", [2, 65, 100])
@pytest.mark.parametrize("kw,code,text", BAD)
def test_refused_before_anything_is_written(window, B, kw, code, text):
    if "workspace" in text and B > 2:
        kw = dict(kw, hq=1, hkv=1)                      # few enough heads to split the context
    assert _call(window, B, **kw) == code
    assert text in _lib.last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="placeholder pointers")
@pytest.mark.parametrize("B", [2, 100])
def test_window_output_over_the_queries(B):
    assert _call(16, B, q=P) == _lib.PDK_EINVAL
    assert "overlap" in _lib.last_error()
