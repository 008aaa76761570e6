"""CPU: when captured graphs die.  A graph must not be destroyed by Python's cycle collector in the middle of another graph's capture; torch's graph
objects are replaced by recorders here, the class under test is graphs.GraphedChain itself."""
import contextlib
import gc
import os
import re
import weakref
from types import SimpleNamespace as ns

import pytest
import torch

from diffalign_amd import graphs, streams
from diffalign_amd.placeholder import PlaceHolder

T_EVAL, B, N, KX, KE = 4, 2, 3, 5, 3


class Model:
    """What GraphedChain reads of a model at construction."""
    T = T_EVAL

    def __init__(self):
        q = lambda k: torch.zeros(T_EVAL + 1, k, k)
        self.cfg = ns(diffusion=ns(diffusion_steps_eval=T_EVAL, diffuse_edges=True, diffuse_nodes=True))
        self.transition_model_eval = ns(Qts_x=q(KX), Qts_e=q(KE), Qt_bars_x=q(KX), Qt_bars_e=q(KE))
        self.packed = object()

    def _net(self):
        return ns(_pack=lambda dev: self.packed)


@pytest.fixture
def chain(monkeypatch):
    log = ns(collector=[], replays=0, ran=[], captured=[], on=[None])

    class Stream:
        def __init__(self, role):
            self.role = role

        def wait_stream(self, other):
            pass

    made = {}

    @contextlib.contextmanager
    def on(stream):
        log.on.append(stream.role)
        yield
        log.on.pop()

    def body(self, t):
        log.collector.append(gc.isenabled())
        log.ran.append(log.on[-1])

    class Graph:
        def replay(self):
            log.replays += 1

    @contextlib.contextmanager
    def capture(graph, stream=None, **kw):
        log.captured.append(stream.role)
        with on(stream):
            yield
    monkeypatch.setattr(streams, 'own', lambda dev, role: made.setdefault(role, Stream(role)))
    monkeypatch.setattr(torch.cuda, 'stream', on)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda device=None: Stream('caller'))
    monkeypatch.setattr(torch.cuda, 'CUDAGraph', Graph)
    monkeypatch.setattr(torch.cuda, 'graph', capture)
    monkeypatch.setattr(torch.cuda, 'graph_pool_handle', lambda: (0, 0))
    monkeypatch.setattr(torch.cuda, 'synchronize', lambda device=None: None)
    monkeypatch.setattr(graphs, '_prepare_capture', lambda dev: None)
    monkeypatch.setattr(graphs.GraphedChain, '_body', body)

    def make(model, n=N):
        data = PlaceHolder(X=torch.zeros(B, n, KX), E=torch.zeros(B, n, n, KE), y=torch.zeros(B, 1), node_mask=torch.ones(B, n, dtype=torch.bool))
        got = graphs.GraphedChain.get(model, data, (torch.ones(B, n, KX), torch.ones(B, n, n, KE)), None, (1.0, 1.0), None, None, False, 0)
        got.warm = True
        return got
    return ns(make=make, log=log)


def test_a_dropped_model_takes_its_graphs_with_it(chain):
    model = Model()
    c = chain.make(model)
    c.run()
    assert chain.log.replays == T_EVAL and chain.make(model) is c and c.model is model
    held, first = weakref.ref(c), weakref.ref(next(iter(c.graphs.values())))
    on = gc.isenabled()
    gc.disable()
    try:
        del c, model
        assert held() is None and first() is None, 'left to the cycle collector'
    finally:
        if on:
            gc.enable()


def test_evicted_chains_die_at_once(chain):
    model = Model()
    gc.collect()
    gc.disable()
    try:
        refs = [weakref.ref(chain.make(model, n)) for n in range(2, 2 + graphs.CHAIN_GRAPH_CACHE + 1)]
        assert refs[0]() is None and all(r() is not None for r in refs[1:])
        model.packed = object()                                             # new weights: the shape's chain is built anew
        assert chain.make(model, 3) is not None and refs[1]() is None
    finally:
        gc.enable()


def test_no_collection_during_a_capture(chain):
    assert gc.isenabled()
    model = Model()
    chain.make(model).run()
    assert chain.log.collector == [False] * T_EVAL and gc.isenabled()
    with pytest.raises(ZeroDivisionError):
        with graphs._capture(torch.cuda.CUDAGraph(), 'cuda:0'):
            1 / 0
    assert gc.isenabled()
    gc.disable()
    try:
        with graphs._capture(torch.cuda.CUDAGraph(), 'cuda:0'):
            pass
        assert not gc.isenabled()                                           # the caller's setting stays
    finally:
        gc.enable()


def test_a_chain_without_its_model_refuses(chain):
    model = Model()
    c = chain.make(model)
    c.run()
    del model
    with pytest.raises(RuntimeError, match='model'):
        c.run()


def test_a_new_chain_takes_no_pooled_stream(chain, monkeypatch):
    """torch.cuda.Stream() walks through a pool of 32: a request per chain comes round to the capture stream.  Warm-up and capture each have a
    stream of their own, which no other role shares."""
    def pooled(*a, **k):
        raise AssertionError('a stream out of the pool')
    monkeypatch.setattr(torch.cuda, 'Stream', pooled)
    model = Model()
    for n in range(2, 40):
        c = chain.make(model, n)
        c.warm = False
        c.run()
    assert set(chain.log.ran) == {'warm', 'capture'} and chain.log.ran.count('warm') == 38
    assert set(chain.log.captured) == {'capture'}


def test_no_pooled_streams_in_the_package():
    root = os.path.dirname(graphs.__file__)
    for name in os.listdir(root):
        if name.endswith('.py'):
            text = open(os.path.join(root, name)).read()
            assert 'cuda.Stream(' not in re.sub(r'""".*?"""', '', text, flags=re.S), name
    assert len(set(streams.ROLES)) == len(streams.ROLES)


def test_streams_are_made_once_per_device(monkeypatch):
    made = []
    monkeypatch.setattr(streams, '_OWN', {})
    monkeypatch.setattr(streams, '_create', lambda index: made.append(index) or object())
    a = {r: streams.own('cuda:0', r) for r in streams.ROLES}
    b = {r: streams.own(torch.device('cuda', 1), r) for r in streams.ROLES}
    assert all(streams.own('cuda:0', r) is a[r] for r in streams.ROLES) and made == [0] * len(a) + [1] * len(b)
    assert len({id(s) for s in (*a.values(), *b.values())}) == 2 * len(streams.ROLES)
    with pytest.raises(KeyError):
        streams.own('cuda:0', 'another')


def test_stream_create_refuses_a_null_pointer_and_the_version_stays():
    from diffalign_amd import _lib as L
    assert L.lib().da_stream_create(None) != 0 and b'da_stream_create' in L.lib().da_last_error()
    assert L.lib().da_abi_version() == 3                # entry points were only added: a binding of version 3 keeps loading
