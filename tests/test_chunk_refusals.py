"""Argument checks of the chunk and 8-bit entry points of the C ABI: a bad call returns its
code and a message before anything is launched (the pointers are placeholders that nothing
dereferences), and the Python wrappers refuse what is not on a GPU."""
import ctypes

import pytest
import torch

from rngd_pd_amd import _lib, kernels as K

P = 1 << 20                                       # 16-byte aligned placeholder address
INVAL, NOTSUP, NOMEM = _lib.PDK_EINVAL, _lib.PDK_ENOTSUP, _lib.PDK_ENOMEM


def _call(name, base, kw):
    a = {**base, **kw}
    assert set(a) == set(base), "an argument that the call does not have"
    return getattr(_lib.lib(), name)(*a.values())


MAP = dict(past=P, added=P, R=4, tables=P, W=8, free=P, n_free=9, N=64, starts=P, ctx=P, pos=P,
           slots=P, taken=P, stream=0)
WRITE = dict(qkv=P, ld=48 * 128, inv=P, pos=P, slots=P, N=5, hq=32, hkv=8, d=128, q=P, ck=P, cv=P,
             nb=9, stream=0)
ATTN = dict(q=P, ld=4096, ck=P, cv=P, nb=64, tables=P, W=512, starts=P, ctx=P, N=40, R=2, max_new=30,
            max_ctx=8000, hq=32, hkv=8, d=128, scale=1.0, window=0, sinks=0, ws=P, ws_bytes=1 << 40,
            out=P, stream=0)
NORM = dict(x=P, add=P, w=P, T=4, H=256, eps=1e-5, sum=P, out=P, scales=P, ld=4, stream=0)
QUANT = dict(x=P, ld=512, T=4, K=256, out=P, scales=P, sld=4, stream=0)
LINEAR = dict(x=P, ld=256, xs=P, st=1, sg=4, w=P, ws=P, T=4, K=256, N=64, work=P, work_bytes=1 << 40,
              y=P, stream=0)


@pytest.mark.parametrize("name,base,kw,code,text", [
    ("pdk_chunk_map", MAP, dict(R=0), INVAL, "R must"),
    ("pdk_chunk_map", MAP, dict(R=4097), INVAL, "R must"),
    ("pdk_chunk_map", MAP, dict(W=0), INVAL, "tables"),
    ("pdk_chunk_map", MAP, dict(R=4096, W=1 << 15), INVAL, "tables"),
    ("pdk_chunk_map", MAP, dict(n_free=-1), INVAL, "n_free"),
    ("pdk_chunk_map", MAP, dict(N=-1), INVAL, "max_tokens"),
    ("pdk_chunk_map", MAP, dict(free=None), INVAL, "null"),
    ("pdk_chunk_map", MAP, dict(slots=None), INVAL, "null"),
    ("pdk_chunk_map", MAP, dict(taken=None), INVAL, "null"),
    ("pdk_rope_cache_write", WRITE, dict(d=64), NOTSUP, "head_dim"),
    ("pdk_rope_cache_write", WRITE, dict(N=-1), INVAL, "N must"),
    ("pdk_rope_cache_write", WRITE, dict(hq=0), INVAL, "head"),
    ("pdk_rope_cache_write", WRITE, dict(ld=48 * 128 - 8), INVAL, "ld"),
    ("pdk_rope_cache_write", WRITE, dict(ld=48 * 128 + 4), INVAL, "ld"),
    ("pdk_rope_cache_write", WRITE, dict(nb=0), INVAL, "num_blocks"),
    ("pdk_rope_cache_write", WRITE, dict(slots=None), INVAL, "null"),
    ("pdk_rope_cache_write", WRITE, dict(qkv=P + 2), INVAL, "aligned"),
    ("pdk_chunk_attn", ATTN, dict(d=96), NOTSUP, "head_dim"),
    ("pdk_chunk_attn", ATTN, dict(N=-1), INVAL, "N must"),
    ("pdk_chunk_attn", ATTN, dict(N=(1 << 20) + 1), INVAL, "N must"),
    ("pdk_chunk_attn", ATTN, dict(R=0), INVAL, "R must"),
    ("pdk_chunk_attn", ATTN, dict(hq=33), INVAL, "n_q_heads"),
    ("pdk_chunk_attn", ATTN, dict(hq=17 * 8, ld=17 * 8 * 128), INVAL, "n_q_heads"),
    ("pdk_chunk_attn", ATTN, dict(W=65536), INVAL, "max_blocks"),
    ("pdk_chunk_attn", ATTN, dict(max_ctx=0), INVAL, "max_ctx"),
    ("pdk_chunk_attn", ATTN, dict(max_ctx=512 * 16 + 1), INVAL, "max_ctx"),
    ("pdk_chunk_attn", ATTN, dict(max_new=-1), INVAL, "max_new"),
    ("pdk_chunk_attn", ATTN, dict(window=-1), INVAL, "window"),
    ("pdk_chunk_attn", ATTN, dict(sinks=4), INVAL, "sinks"),
    ("pdk_chunk_attn", ATTN, dict(window=9, sinks=-4), INVAL, "sinks"),
    ("pdk_chunk_attn", ATTN, dict(nb=0), INVAL, "num_blocks"),
    ("pdk_chunk_attn", ATTN, dict(scale=0.0), INVAL, "scale"),
    ("pdk_chunk_attn", ATTN, dict(scale=float("inf")), INVAL, "scale"),
    ("pdk_chunk_attn", ATTN, dict(ld=4088), INVAL, "stride"),
    ("pdk_chunk_attn", ATTN, dict(q=None), INVAL, "null"),
    ("pdk_chunk_attn", ATTN, dict(out=P + 8), INVAL, "aligned"),
    ("pdk_chunk_attn", ATTN, dict(ws=None), INVAL, "workspace"),
    ("pdk_chunk_attn", ATTN, dict(ws_bytes=64), NOMEM, "workspace"),
    ("pdk_rmsnorm_fp8", NORM, dict(T=-1), INVAL, "T must"),
    ("pdk_rmsnorm_fp8", NORM, dict(H=200), INVAL, "H must"),
    ("pdk_rmsnorm_fp8", NORM, dict(H=8320), INVAL, "H must"),
    ("pdk_rmsnorm_fp8", NORM, dict(eps=-1.0), INVAL, "eps"),
    ("pdk_rmsnorm_fp8", NORM, dict(ld=3), INVAL, "scale_ld"),
    ("pdk_rmsnorm_fp8", NORM, dict(sum=None), INVAL, "null"),
    ("pdk_rmsnorm_fp8", NORM, dict(add=P + 8), INVAL, "aligned"),
    ("pdk_quantize_fp8", QUANT, dict(K=100), INVAL, "columns"),
    ("pdk_quantize_fp8", QUANT, dict(ld=248), INVAL, "ld"),
    ("pdk_quantize_fp8", QUANT, dict(sld=2), INVAL, "scale_ld"),
    ("pdk_quantize_fp8", QUANT, dict(scales=None), INVAL, "null"),
    ("pdk_swiglu_fp8", QUANT, dict(ld=504), INVAL, "ld"),
    ("pdk_swiglu_fp8", QUANT, dict(x=P + 4), INVAL, "aligned"),
    ("pdk_linear_fp8", LINEAR, dict(T=-1), INVAL, "T must"),
    ("pdk_linear_fp8", LINEAR, dict(K=192), INVAL, "K must"),
    ("pdk_linear_fp8", LINEAR, dict(N=12), INVAL, "N must"),
    ("pdk_linear_fp8", LINEAR, dict(N=0), INVAL, "N must"),
    ("pdk_linear_fp8", LINEAR, dict(ld=264), INVAL, "x_ld"),
    ("pdk_linear_fp8", LINEAR, dict(ld=1 << 24), INVAL, "x_ld"),
    ("pdk_linear_fp8", LINEAR, dict(st=0), INVAL, "strides"),
    ("pdk_linear_fp8", LINEAR, dict(st=1 << 21), INVAL, "strides"),
    ("pdk_linear_fp8", LINEAR, dict(T=64, K=14336, ld=14336, work=None), INVAL, "workspace"),
    ("pdk_linear_fp8", LINEAR, dict(T=64, K=14336, ld=14336, work=P + 8), INVAL, "workspace"),
    ("pdk_linear_fp8", LINEAR, dict(T=64, K=14336, ld=14336, work_bytes=640), NOMEM, "workspace"),
    ("pdk_linear_fp8", LINEAR, dict(ws=None), INVAL, "null"),
    ("pdk_linear_fp8", LINEAR, dict(w=P + 4), INVAL, "aligned"),
])
def test_refusals(name, base, kw, code, text):
    assert _call(name, base, kw) == code
    assert text in _lib.last_error()


def test_nothing_to_do_is_fine():
    assert _call("pdk_rope_cache_write", WRITE, dict(N=0, qkv=None)) == 0
    assert _call("pdk_chunk_attn", ATTN, dict(N=0, q=None, out=None)) == 0
    assert _call("pdk_chunk_attn", ATTN, dict(max_new=0)) == 0
    assert _call("pdk_rmsnorm_fp8", NORM, dict(T=0, x=None)) == 0
    assert _call("pdk_swiglu_fp8", QUANT, dict(T=0)) == 0
    assert _call("pdk_linear_fp8", LINEAR, dict(T=0)) == 0


def test_workspace_bytes():
    size = K.chunk_workspace_bytes
    assert size(1, 1, 1, 64, 32, 8) == 0                    # nothing to split
    assert size(16, 16, 1, 16000, 32, 8) > 0
    # A window bounds what is walked, and so the splits.
    assert size(16, 16, 1, 65535 * 16, 32, 8, 128, 4) == 0
    for bad in ((1, 0, 1, 64, 32, 8), (1, 1, 1, 0, 32, 8), (16, 16, 1, 1 << 20, 32, 8),
                (1, 1, 1, 64, 33, 8), (-1, 1, 1, 64, 32, 8),
                (1, 1, 1, 64, 32, 8, 0, 0)):
        with pytest.raises(ValueError):
            size(*bad)


def test_linear_workspace_bytes():
    size = K.linear_fp8_workspace_bytes
    assert size(16, 14336, 4096) == 0 and size(8192, 4096, 28672) == 0
    assert size(64, 14336, 4096) > 0
    for T in (17, 64, 65, 128, 300, 470, 1000, 2000, 8192, 1 << 20):       # no plan takes much
        for k, n in ((128, 8), (4096, 4096), (14336, 4096), (4096, 28672), (1 << 20, 8)):
            assert size(T, k, n) <= 1 << 29
    for bad in ((-1, 128, 8), (4, 100, 8), (4, 128, 12), (4, 128, 0), (1 << 21, 128, 8)):
        with pytest.raises(ValueError):
            size(*bad)


def test_wrappers_need_a_gpu_tensor():
    t, i = torch.zeros((4, 256), dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    f8, s = torch.zeros((4, 256), dtype=torch.float8_e4m3fn), torch.ones((4, 2))
    cache = torch.zeros((2, 1, 16, 128), dtype=torch.bfloat16)
    for call in (lambda: K.chunk_map(i, i, i.view(2, 2), i, 4),
                 lambda: K.rope_cache_write(t, s, i, i, cache, cache.transpose(2, 3), 1),
                 lambda: K.chunk_attention(t.view(4, 2, 128), cache, cache, i.view(2, 2), i, i, 1, 16),
                 lambda: K.rmsnorm_fp8(t, t[0], 1e-5), lambda: K.quantize_fp8(t),
                 lambda: K.swiglu_fp8(t), lambda: K.linear_fp8(f8, s, f8, s)):
        with pytest.raises(TypeError, match="CUDA"):
            call()


def test_weights_in_8_bits():
    """The loader's own form, on the CPU: blocks of 128 x 128, the last rows' smaller."""
    gen = torch.Generator().manual_seed(0)
    w = torch.randn((200, 256), generator=gen).to(torch.bfloat16)
    w[130:140, 128:] *= 100
    q, s = K.quantize_weight_fp8(w)
    assert q.dtype is torch.float8_e4m3fn and tuple(s.shape) == (2, 2)
    for i, rows in enumerate((slice(0, 128), slice(128, 200))):
        for j in range(2):
            part = w[rows, 128 * j:128 * j + 128].float()
            assert s[i, j] == part.abs().max() / 448
            back = q[rows, 128 * j:128 * j + 128].float() * s[i, j]
            assert ((back - part).abs() <= 2.0 ** -4 * 1.0001 * part.abs() + 2.0 ** -10 * s[i, j]).all()
    for bad in (w[:, :100], w[0], w[:0]):
        with pytest.raises(ValueError):
            K.quantize_weight_fp8(bad)


def test_linear_workspaces_up_to_their_bound():
    """512 MiB at most, as the header states, and sizes that come near it."""
    size, most = K.linear_fp8_workspace_bytes, 0
    for T in (17, 100, 300, 470, 700, 1000, 1500, 2000, 3000, 4096, 5000, 16384):
        for N in (8, 4096, 6144, 8192, 14336, 28672, 57344):
            for k in (4096, 14336, 28672, 57344, 1 << 17, 1 << 20):
                most = max(most, size(T, k, N))
    assert 500 << 20 <= most <= 512 << 20
    assert size(5000, 28672, 8192) <= 320 << 20


def test_attention_workspaces_up_to_their_bound():
    """The records of longer requests (4096 of four units of 64 x 66 floats) and of those
    of few rows beside them (768 of 2176 floats), 284 MB, and sizes that come near it."""
    most = 0
    for R in (1, 2, 16, 32, 64, 768, 4000):
        for N in (40, 776, 3104, 6208, 8192, 1 << 20):
            for hq, hkv in ((32, 8), (64, 4), (8, 8), (16, 1), (8, 1), (128, 8)):
                for ctx in (4096, 1 << 17, 65535 * 16):
                    most = max(most, K.chunk_workspace_bytes(N, R, N, ctx, hq, hkv))
    bound = 4096 * 4 * 64 * 66 * 4 + 768 * 2176 * 4
    assert 0.99 * bound <= most <= bound <= 284e6
