"""GPU: the framework's own streams are not in torch's pool, and work on them is ordered and recorded like on any other."""
import pytest
import torch

pytestmark = pytest.mark.gpu
D = 'cuda:0'


def test_own_streams_are_nobody_elses():
    from diffalign_amd import streams
    pool = {torch.cuda.Stream(device=D).cuda_stream for _ in range(80)}
    own = [streams.own(D, r) for r in streams.ROLES]
    handles = {s.cuda_stream for s in own}
    assert len(handles) == len(own) and not handles & pool and 0 not in handles
    assert all(s.device == torch.device(D) for s in own) and streams.own('cuda', 'y').cuda_stream == own[0].cuda_stream


def test_work_on_an_own_stream():
    from diffalign_amd import streams
    s, main = streams.own(D, 'node'), torch.cuda.current_stream()
    x = torch.arange(1 << 20, device=D, dtype=torch.float32)
    for k in range(3):
        ready = main.record_event()
        with torch.cuda.stream(s):
            s.wait_event(ready)
            y = x * (k + 1)
            done = s.record_event()
        y.record_stream(main)
        main.wait_event(done)
        assert torch.equal(y, x * (k + 1))


def test_capture_on_the_own_stream():
    from diffalign_amd import graphs, streams
    x, y, u = (torch.zeros(4096, device=D) for _ in range(3))
    graphs._prepare_capture(x.device)
    g, side = torch.cuda.CUDAGraph(), streams.own(D, 'node')
    with graphs._capture(g, x.device):
        main = torch.cuda.current_stream()
        assert main.cuda_stream == streams.own(D, 'capture').cuda_stream
        x += 1
        ev = main.record_event()
        with torch.cuda.stream(side):
            side.wait_event(ev)
            y += x
            done = side.record_event()
        u += 1
        main.wait_event(done)
        x += y
    want_x = want_y = 0.0
    for k in range(4):
        g.replay()
        torch.cuda.synchronize()
        want_y += want_x + 1
        want_x += 1 + want_y
        assert float(y[0]) == want_y and float(x[-1]) == want_x and float(u[7]) == k + 1, k
