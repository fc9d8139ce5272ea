"""The device and stream that a call's launches and allocations belong to (host logic;
the streams are stand-ins)."""
import pytest
import torch

from rngd_pd_amd.kernels import handoff as h


class Stream:
    def __init__(self, index):
        self.device, self.cuda_stream = torch.device("cuda", index), 77


def test_stream_of_another_device_is_refused():
    with pytest.raises(ValueError, match="cuda:0"):
        h.launch_scope(torch.device("cuda", 1), Stream(0))
    h.launch_scope(torch.device("cuda", 1), Stream(1))
    h.launch_scope(torch.device("cuda"), Stream(1))     # whatever is current: the stream's


@pytest.mark.parametrize("bad", ["side", 1.5, object()])
def test_what_is_no_stream_is_refused(bad):
    with pytest.raises(TypeError):
        h.launch_scope(torch.device("cuda", 0), bad)


def test_handle_zero_is_the_default_stream(monkeypatch):
    """torch.cuda.ExternalStream takes a handle of 0 for none and makes a new stream."""
    import contextlib
    entered = []

    @contextlib.contextmanager
    def stream(s):
        entered.append(s)
        yield
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda d=None: ("default", d))
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda h, **kw: ("external", h))
    dev = torch.device("cuda", 1)
    for handle in (0, 77):
        with h.launch_scope(dev, handle):
            pass
    assert entered == [("default", None), ("external", 77)]   # the default of the device made current
