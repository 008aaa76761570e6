"""CPU: the scratch of the two-stage kernels and a graph's recording: what a graph keeps the address of belongs to it alone."""
from types import SimpleNamespace as ns

import pytest
import torch

from diffalign_amd import autograd_ops as A


@pytest.fixture
def on(monkeypatch):
    state = ns(stream=1, recording=False)
    monkeypatch.setattr(A, '_WS', {})
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: ns(cuda_stream=state.stream))
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: state.recording)
    return state


def test_eager_calls_of_a_stream_share_their_scratch(on):
    a = A._workspace('cpu', 100)
    assert A._workspace('cpu', 60) is a
    on.stream = 2
    assert A._workspace('cpu', 60) is not a
    on.stream = 1
    b = A._workspace('cpu', 200)
    assert b.numel() == 200 and A._workspace('cpu', 100) is b


def test_a_recorded_call_takes_no_scratch_that_others_have(on):
    """Neither the stream's own, which the next larger eager call hands back to the allocator while the graph still writes to it, nor the one of
    another recording; and leaves none behind."""
    eager = A._workspace('cpu', 100)
    on.recording = True
    first, second = A._workspace('cpu', 100), A._workspace('cpu', 50)
    assert len({t.data_ptr() for t in (eager, first, second)}) == 3 and first.numel() >= 100 and second.numel() >= 50
    on.recording = False
    assert A._workspace('cpu', 100) is eager and list(A._WS.values()) == [eager]
    on.stream, on.recording = 3, True
    A._workspace('cpu', 10)
    assert len(A._WS) == 1
