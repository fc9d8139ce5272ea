"""Which of beam_select's operands may share memory: the outputs with the scores and
last tokens of as many beams, place for place; all else is refused (the pointers are
placeholders; without a GPU a call that is taken fails at its launch, with PDK_EHIP)."""
import pytest
import torch

from rngd_pd_amd import _lib

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="placeholder pointers")
R, K, V = 3, 4, 1000
LOGITS, SCORES, LAST, WS = 1 << 30, 2 << 30, 3 << 30, 4 << 30
TOK, PAR, OUT = 5 << 30, 6 << 30, 7 << 30


def _call(n=K, logits=LOGITS, scores=SCORES, last=LAST, ws=WS, tok=TOK, par=PAR, out=OUT, ld=V):
    need = _lib.lib().pdk_beam_select_workspace_bytes(R, K, V, n)
    rc = _lib.lib().pdk_beam_select(logits, 2, ld, R, K, V, scores, last, 7, n, ws, need, tok, par,
                                    out, 0)
    return rc, need


@pytest.mark.parametrize("kw", [
    dict(), dict(n=K + 1), dict(last=None), dict(tok=LAST), dict(out=SCORES),
    dict(tok=LAST, out=SCORES), dict(n=K - 1, last=None), dict(tok=LOGITS),
    dict(par=TOK + 4 * R * K, out=TOK - 4 * R * K),     # side by side
    dict(last=SCORES + 4 * R * K)])
def test_taken(kw):
    assert _call(**kw)[0] == _lib.PDK_EHIP


@pytest.mark.parametrize("kw", [
    dict(n=K + 1, out=SCORES), dict(n=K - 1, out=SCORES), dict(n=K + 1, tok=LAST),
    dict(n=1, tok=LAST), dict(out=SCORES + 4), dict(out=SCORES - 4 * (R * K - 1)),
    dict(tok=LAST + 4 * K), dict(par=TOK), dict(out=PAR), dict(tok=OUT + 4 * (R * K - 1)),
    dict(tok=WS), dict(par=WS + 64), dict(ws=OUT), dict(ws=SCORES), dict(ws=LAST),
    dict(ws=LOGITS), dict(ws=LOGITS + 2 * ((R * K - 1) * 2 * V), ld=2 * V)])
def test_refused(kw):
    assert _call(**kw)[0] == _lib.PDK_EINVAL
    assert "overlap" in _lib.last_error()


def test_workspace_between_rows_is_taken():
    """Rows of a wider tensor: the workspace must lie clear of the last one's end."""
    assert _call(ld=2 * V, ws=LOGITS + 2 * ((R * K - 1) * 2 * V + V))[0] == _lib.PDK_EHIP
