"""The framework's own HIP streams: one per device and purpose, made once and kept for the process, at the default priority.

torch.cuda.Stream() hands out the 32 streams of a per-device pool in turn: the 33rd call returns the first one's stream again.  A stream asked
for per chain or per call walks through the pool, and after 32 the 'new' stream is torch's graph capture stream, or one of the side
streams whose work it is meant to be ordered against -- eager work then runs on the stream a graph is recorded on next, and a captured fork
joins the stream it forked from.  (Graph launches ended the process, a segmentation fault in the runtime, three times: each after eager forked
work on the stream that earlier graphs had been recorded on and the next one was.  Most likely that is the cause; what the runtime does there
is not known.)  Streams made here are nobody else's."""
from __future__ import annotations

import ctypes as C
import threading

import torch

ROLES = ('y', 'node',          # engine: y chain, node chain of the inference forward
         'train_node',         # train_forward: node / y side of the training step
         'eig',                # extra_features: the eigensolver
         'pos',                # graphs.GraphedTrainStep: the next batch's positional encodings
         'warm',               # graphs: the eager run before a capture
         'capture')            # graphs: recording, and nothing else (no eager work ever runs on it)
_OWN = {}
_LOCK = threading.Lock()


def own(dev, role: str) -> torch.cuda.Stream:
    """The stream of `role` on device `dev`.  The first call for a device makes the streams of every role (not inside a capture then)."""
    dev = torch.device(dev)
    key = dev.index if dev.index is not None else torch.cuda.current_device()
    streams = _OWN.get(key)
    if streams is None:
        with _LOCK:
            streams = _OWN.get(key)
            if streams is None:
                streams = _OWN[key] = {r: _create(key) for r in ROLES}
    return streams[role]


def _create(index: int) -> torch.cuda.Stream:
    from . import _lib as L
    out = C.c_void_p()
    with torch.cuda.device(index):
        L.check(L.lib().da_stream_create(C.byref(out)), 'da_stream_create')
    return torch.cuda.ExternalStream(out.value, device=torch.device('cuda', index))
