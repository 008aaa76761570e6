"""CPU: a training step is not recorded while an eager autograd graph of its parameters lives."""
from types import SimpleNamespace as ns

import pytest
import torch

from diffalign_amd import graphs


def test_leaves_of_a_live_graph_are_found():
    lin, other = torch.nn.Linear(3, 2), torch.nn.Linear(3, 2)
    params = [*lin.parameters(), *other.parameters()]
    assert graphs._in_a_live_graph(params) == []
    loss = lin(torch.ones(4, 3)).sum()
    for _ in range(2):                                                     # looking leaves no trace
        assert [id(p) for p in graphs._in_a_live_graph(params)] == [id(p) for p in lin.parameters()]
    loss.backward()                                                        # its buffers are gone, the graph is not
    assert len(graphs._in_a_live_graph(params)) == 2
    kept = loss.detach()
    del loss
    assert graphs._in_a_live_graph(params) == [] and kept.grad_fn is None
    with torch.no_grad():
        out = lin(torch.ones(4, 3))
        assert graphs._in_a_live_graph(params) == []
    out = lin(torch.ones(4, 3))
    with torch.no_grad():                                                  # also found where gradients are off
        assert len(graphs._in_a_live_graph(params)) == 2
    del out


def test_a_step_is_not_recorded_beside_one(monkeypatch):
    """The refusal comes before anything runs; a graph that only a reference cycle holds is collected instead."""
    class Ready(Exception):
        pass

    def reached(dev):
        raise Ready
    monkeypatch.setattr(graphs, '_prepare_capture', reached)
    lin = torch.nn.Linear(3, 2)
    build = lambda: graphs.GraphedTrainStep(ns(model=ns(training=True)), ns(step_dev=torch.zeros(1), params=list(lin.parameters())), ns(X=torch.zeros(1)))
    with pytest.raises(Ready):
        build()
    loss = lin(torch.ones(4, 3)).sum()
    with pytest.raises(RuntimeError, match='alive'):
        build()
    cycle = [loss]
    cycle.append(cycle)
    del loss, cycle
    with pytest.raises(Ready):
        build()
