"""Which steps an engine replays from a captured graph, on the host: the graph and the device stand-ins are the test's."""
import contextlib
import types

import pytest
import torch

from vlrf_b200.engine import step as step_module
from vlrf_b200.engine.step import Engine
from vlrf_b200.parts.context import Workspace


class Graph:
    def __init__(self):
        self.log, self.played = None, 0

    def replay(self):
        """A graph goes to the scratch that it was captured with: it has to be there still."""
        self.played += 1
        for ws, name, buf in self.log:
            assert ws._bufs[name] is buf, f"replayed with scratch '{name}' that has been given back"


class Model:
    """Takes as much scratch as a step's `room` says."""
    replayable = True

    def __init__(self):
        self.log = None

    def forward(self, ctx, cache):
        ctx.ws.get("scratch", ctx.room, 1, torch.float32)
        if self.log is not None:
            self.log.append((ctx.ws, "scratch", ctx.ws._bufs["scratch"]))
        return object()


@pytest.fixture
def engine(monkeypatch):
    eng = object.__new__(Engine)
    eng.model, eng.ws, eng.cache = Model(), Workspace("cpu"), None
    eng.capture_repeated_steps, eng._graphs, eng._seen, eng._graph_generation = True, {}, {}, -1

    @contextlib.contextmanager
    def capture_into(graph):
        eng.model.log = graph.log = []
        yield
        eng.model.log = None
    monkeypatch.setattr(step_module, "capture_into", capture_into)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    return eng


def run(eng, signature, room):
    return eng._forward(types.SimpleNamespace(max_new=5, ws=eng.ws, room=room), signature)


def test_a_step_seen_before_is_captured_and_replayed(engine):
    for _ in range(4):
        run(engine, "a", 10)
    assert engine._graphs["a"][0].played == 3


def test_a_graph_is_dropped_when_a_new_step_s_first_run_moves_the_scratch(engine):
    for _ in range(3):
        run(engine, "a", 10)
    run(engine, "b", 1000)                 # grows the scratch: what was captured goes to memory that is no longer there
    for _ in range(3):
        run(engine, "a", 10)
    assert engine._graphs["a"][0].played == 3


def test_a_graph_is_dropped_when_a_capture_moves_the_scratch(engine):
    for _ in range(3):
        run(engine, "a", 10)
    run(engine, "b", 5)
    run(engine, "b", 1000)                 # the capture itself had to allocate
    for _ in range(3):
        run(engine, "a", 10)
    for _ in range(2):
        run(engine, "b", 1000)
    assert engine._graphs["a"][0].played == 3 and engine._graphs["b"][0].played == 2
