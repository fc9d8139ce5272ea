"""Which stream the attention workspaces belong to, and when a replaced one goes
(host logic; the streams and the allocator are stand-ins)."""
import contextlib

import pytest
import torch

from rngd_pd_amd.engines import decode_batch as db
from rngd_pd_amd.engines.paged_cache import PagedKVCache
from rngd_pd_amd.kernels import attention as at


class Buffer:
    def __init__(self, nbytes, stream):
        self.n, self.allocated_on, self.recorded = nbytes // 4 + 64, stream, []

    def numel(self):
        return self.n

    def record_stream(self, stream):
        self.recorded.append(stream)


@pytest.fixture
def gpu(monkeypatch):
    """The current stream (1 unless a scope says otherwise) and whether it is captured."""
    state = {"stream": 1, "capturing": False, "alive": []}

    @contextlib.contextmanager
    def scope(device, stream=None):
        before = state["stream"]
        state["stream"] = before if stream is None else stream
        yield
        state["stream"] = before
    monkeypatch.setattr(at, "launch_scope", scope)
    monkeypatch.setattr(at, "_current_device", lambda: 0)
    monkeypatch.setattr(at, "stream_handle", lambda s=None: state["stream"] if s is None else s)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: state["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(at.Workspace, "_new", lambda self, n: Buffer(n, state["stream"]))
    return state


def test_workspace_belongs_to_the_calls_stream(gpu):
    ws = at.Workspace("cuda:0")
    assert ws.take(0, 5) is None and ws.buffer is None and ws.holds(0) and not ws.holds(4)
    a = ws.take(1000, 5)
    assert a.allocated_on == 5 and a.recorded == [] and a.numel() * 4 >= 1000
    assert ws.take(500) is a and ws.take(1000, 5) is a and ws.take(8) is a
    assert a.recorded == [1]                            # once for the current stream
    b = ws.take(5000)
    assert b is not a and b.allocated_on == 1 and b.recorded == [] and not ws._kept
    assert gpu["stream"] == 1


def test_workspace_of_a_captured_graph_stays(gpu):
    ws = at.Workspace("cuda:0")
    a = ws.take(1000)
    gpu["capturing"] = True
    assert ws.take(1000, 9) is a
    gpu["capturing"] = False
    b = ws.take(4000)
    assert ws._kept == [a] and b is not a
    ws.take(9000)
    assert ws._kept == [a]                              # no graph has seen b


def test_batched_attention_takes_its_workspace_on_the_calls_stream(gpu, monkeypatch):
    calls = []
    monkeypatch.setattr(db._attn, "decode_attention_append",
                        lambda *a, workspace=None, stream=None, **kw: calls.append((workspace, stream)))
    eng = db.BatchDecodeAttention(PagedKVCache(1, 4, 2, 128, device="cpu"), n_q_heads=8)
    q = torch.zeros((1, 8, 128))
    for ctx, stream in ((64, None), (600, 7), (600, None), (2000, 7)):
        eng.layer_attention(0, q, None, None, None, None, ctx, stream=stream)
    ws = [w for w, _ in calls]
    assert [s for _, s in calls] == [None, 7, None, 7]
    assert ws[0] is None                                # one split: none needed
    assert ws[1].allocated_on == 7 and ws[2] is ws[1] and ws[1].recorded == [1]
    assert ws[3] is not ws[1] and ws[3].allocated_on == 7


def test_get_workspace_per_device_and_stream(gpu, monkeypatch):
    monkeypatch.setattr(at, "_WORKSPACES", {})
    monkeypatch.setattr(at, "_current_device", lambda: 1)
    a = at.get_workspace(100, "cuda:0", 3)
    assert a.allocated_on == 3 and at.get_workspace(1 << 20, torch.device("cuda", 0), 3) is a
    assert at.get_workspace(100, "cuda") is not a       # the current device's
    assert set(at._WORKSPACES) == {0, 1}


def test_workspace_of_a_graph_that_is_gone_goes(gpu):
    ws = at.Workspace("cuda:0")
    ws.take(1000)
    before = ws.graphs()
    gpu["capturing"] = True
    ws.take(1000)
    gpu["capturing"] = False
    ws.graphs_gone(before)
    ws.take(4000)
    assert ws._kept == []
    # A graph from before still holds what it used then.
    gpu["capturing"] = True
    held = ws.take(4000)
    gpu["capturing"] = False
    ws.graphs_gone(ws.graphs())
    ws.take(9000)
    assert ws._kept == [held]
