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
