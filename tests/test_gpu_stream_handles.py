"""Calls on a stream given by its handle, 0 (the default stream's) among them: in
order with what that stream has queued, whatever stream is current."""
import numpy as np
import pytest
import torch

from tests._span_ref import SCALE, paged
from tests._util import rand_bf16, to_dev

pytestmark = pytest.mark.gpu
D = 128


def _busy(dev):
    a = torch.ones((4096, 4096), device=dev)
    for _ in range(6):
        a = torch.matmul(a, a).clamp_(0, 1)
    return a


@pytest.mark.parametrize("kind", ["default", "side"])
def test_scope_of_a_handle(cuda, kind):
    from rngd_pd_amd.kernels.handoff import launch_scope, stream_handle
    st = torch.cuda.default_stream() if kind == "default" else torch.cuda.Stream()
    with torch.cuda.stream(torch.cuda.Stream()):
        outside = stream_handle()
        with launch_scope(cuda, st.cuda_stream):
            assert stream_handle() == st.cuda_stream
            assert torch.cuda.current_stream().cuda_stream == st.cuda_stream
        assert stream_handle() == outside


@pytest.mark.parametrize("kind", ["default", "side"])
def test_calls_are_in_order_with_the_handles_stream(cuda, kind):
    """Inputs that the stream only gets to write after some milliseconds of work."""
    from rngd_pd_amd import kernels as K
    rng = np.random.default_rng(3)
    ctx = [300, 40]
    tables, nb = paged(rng, ctx, 2)
    ck, cv = to_dev(rand_bf16(rng, (nb, 2, 16, D))), to_dev(rand_bf16(rng, (nb, 2, D, 16)))
    q = to_dev(rand_bf16(rng, (2, 8, D)))
    tab, ctx_d = torch.from_numpy(tables).to(cuda), torch.tensor(ctx, dtype=torch.int32, device=cuda)
    p = to_dev(rand_bf16(rng, (70, 12, D)))
    x, scores = torch.randn((4, 5000), device=cuda), torch.zeros((1, 4), device=cuda)
    held = sorted(set(range(nb)) - set(tables.ravel().tolist()))

    def run(q, p, x, ck, cv, stream):
        kw = {} if stream is None else {"stream": stream}
        a = K.decode_attention(q, ck, cv, tab, ctx_d, 300, scale=SCALE, window=90, sinks=4, **kw)
        b = K.prefill_attention(p[:, :8], p[:, 8:10], p[:, 10:], scale=SCALE, window=20, **kw)
        c = K.beam_select(x, scores, 6, **kw)
        K.copy_blocks(ck, cv, [int(tables[0, 0])], [held[0]], **kw)
        return a, b, *c

    k1, v1 = ck.clone(), cv.clone()
    want = run(q, p, x, k1, v1, None)
    torch.cuda.synchronize()
    late = [torch.zeros_like(t) for t in (q, p, x, ck, cv)]
    st = torch.cuda.default_stream() if kind == "default" else torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        busy = _busy(cuda)
        for t, source in zip(late, (q, p, x, ck, cv)):
            t.copy_(source)
    with torch.cuda.stream(torch.cuda.Stream()):
        got = run(*late, st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(late[3], k1) and torch.equal(late[4], v1)
    del busy
