"""Which operands of a step's entry points may share memory (the pointers are placeholders;
without a GPU a call that is taken fails at its launch, with PDK_EHIP)."""
import pytest
import torch

from rngd_pd_amd import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="placeholder pointers")
AT = {name: (i + 1) << 32 for i, name in enumerate(
    ("qkv", "inv", "pos", "slots", "q", "ck", "cv", "past", "added", "tables", "free", "starts", "ctx", "taken"))}
N, HQ, HKV, NB, D = 5, 4, 2, 9, 128
LD = (HQ + 2 * HKV) * D + 64
CACHE, Q, QKV = NB * HKV * 16 * D * 2, N * HQ * D * 2, ((N - 1) * LD + (HQ + 2 * HKV) * D) * 2


def _write(**kw):
    a = {**AT, **kw}
    return _lib.lib().pdk_rope_cache_write(a["qkv"], LD, a["inv"], a["pos"], a["slots"], N, HQ, HKV, D,
                                           a["q"], a["ck"], a["cv"], NB, 0)


@pytest.mark.parametrize("kw", [
    {}, dict(cv=AT["ck"] + CACHE), dict(ck=AT["cv"] + CACHE), dict(q=AT["qkv"] - Q), dict(q=AT["qkv"] + QKV),
    dict(slots=AT["pos"]), dict(ck=AT["qkv"] + QKV), dict(pos=AT["q"] + Q)])
def test_write_takes(kw):
    assert _write(**kw) == _lib.PDK_EHIP


@pytest.mark.parametrize("kw", [
    dict(cv=AT["ck"]), dict(cv=AT["ck"] + CACHE - 16), dict(q=AT["ck"] + 64), dict(q=AT["cv"] - Q + 16),
    dict(ck=AT["qkv"]), dict(cv=AT["qkv"] + QKV - 16), dict(q=AT["qkv"]), dict(q=AT["qkv"] + QKV - 16),
    dict(pos=AT["ck"]), dict(slots=AT["cv"] + CACHE - 4), dict(inv=AT["q"] + 64)])
def test_write_refuses(kw):
    assert _write(**kw) == _lib.PDK_EINVAL
    assert "overlap" in _lib.last_error()


R, W, FREE = 3, 8, 20
TABLES = R * W * 4


def _map(n_free=FREE, **kw):
    a = {**AT, **kw}
    return _lib.lib().pdk_chunk_map(a["past"], a["added"], R, a["tables"], W, a["free"], n_free, N, a["starts"],
                                    a["ctx"], a["pos"], a["slots"], a["taken"], 0)


@pytest.mark.parametrize("kw", [
    {}, dict(added=AT["past"]), dict(past=AT["tables"] + TABLES), dict(free=AT["tables"] - FREE * 4),
    dict(n_free=0, free=AT["tables"] + 4), dict(ctx=AT["starts"] + 4 * (R + 1)), dict(free=AT["past"])])
def test_map_takes(kw):
    assert _map(**kw) == _lib.PDK_EHIP


@pytest.mark.parametrize("kw", [
    dict(past=AT["tables"]), dict(added=AT["tables"] + TABLES - 4), dict(free=AT["tables"] - FREE * 4 + 4),
    dict(starts=AT["past"]), dict(ctx=AT["starts"] + 4 * R), dict(slots=AT["pos"]), dict(taken=AT["tables"]),
    dict(pos=AT["free"])])
def test_map_refuses(kw):
    assert _map(**kw) == _lib.PDK_EINVAL
    assert "overlap" in _lib.last_error()
