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


class Layer:
    def __init__(self, mixer):
        self.mixer = mixer

    def cache_need(self):
        return self.mixer.cache_need()


@pytest.fixture
def stepping(monkeypatch):
    """An engine over layers of plain attention with a cache of 4 bits that says what it would go by: steps are planned and booked, not run."""
    from vlrf_b200.cache import SequenceCache
    from vlrf_b200.csrc import ops
    from vlrf_b200.engine.model import DecoderModel
    from vlrf_b200.parts.mixer import CausalSelfAttention
    monkeypatch.setattr(ops, "_SM_COUNT", 148)
    ops._packed_decode_shape.cache_clear(); ops._packed_prefill_shape.cache_clear()

    def make(heads, kv_heads, dim, kv_bits=4, window=0):
        mixers = [CausalSelfAttention(torch.zeros((heads + 2 * kv_heads) * dim, 1), None, torch.zeros(1, heads * dim), None, n_heads=heads,
                                      n_kv_heads=kv_heads, head_dim=dim, scale=0.125, window=window) for _ in range(2)]
        model = object.__new__(DecoderModel)
        model.layers, model.schedule, model.embedding, model.act_dtype = [Layer(m) for m in mixers], [], None, torch.bfloat16
        model.vocab_size, model.max_seq_len = 100, 100_000
        eng = object.__new__(Engine)
        eng.model, eng.ws, eng.dev_err, eng.steps_run = model, Workspace("cpu"), None, 0
        eng.cache = SequenceCache([m.cache_need() for m in mixers], max_tokens=200_000, max_seq_len=100_000, dtype=torch.bfloat16, device="cpu", n_slots=64,
                                  kv_bits=kv_bits)
        monkeypatch.setattr(eng.cache, "sync_tables", lambda: None)
        eng._meta_views, eng._meta_copied = {}, types.SimpleNamespace(synchronize=lambda: None, record=lambda: None)
        tables = torch.empty(100_000, dtype=torch.int32)
        eng._meta = lambda n: (tables, tables)
        eng.went_by = []
        eng._forward = lambda ctx, signature: eng.went_by.append(signature)
        return eng
    yield make
    ops._packed_decode_shape.cache_clear(); ops._packed_prefill_shape.cache_clear()


def goes_by(eng, new, past):
    """What a step is known by that brings new[i] tokens behind past[i]."""
    import numpy as np
    slots = [eng.start_sequence() for _ in new]
    for s, b in zip(slots, past):
        if b:
            eng.cache.reserve(s, b)
            eng.cache.advance(s, b)
    eng.step([step_module.StepEntry(s, np.ones(a, dtype=np.int64), [0]) for s, a in zip(slots, new)])
    for s in slots:
        eng.end_sequence(s)
    return eng.went_by[-1]


def test_steps_of_one_size_whose_contexts_ask_for_other_launches_are_captured_apart(stepping):
    eng = stepping(12, 12, 64)
    short, long = goes_by(eng, [256], [256]), goes_by(eng, [256], [20_000])              # the tiles whole; in parts
    assert short != long
    eng = stepping(32, 8, 128)
    short, long = goes_by(eng, [700] + [1] * 5, [1] + [10] * 5), goes_by(eng, [700] + [1] * 5, [1] + [2000] * 5)         # single tokens apart
    assert short != long


def test_steps_of_one_size_and_like_contexts_are_one_captured_step(stepping):
    eng = stepping(32, 8, 128)
    assert goes_by(eng, [700] + [1] * 30, [300] + [2000] * 30) == goes_by(eng, [700] + [1] * 30, [310] + [2005] * 30)
    assert goes_by(eng, [512], [7500]) == goes_by(eng, [512], [7600])
    assert len({goes_by(eng, [512], [512 * i]) for i in range(1, 65)}) <= step_module.MAX_CAPTURED       # one long prompt in pieces
    for eng in (stepping(3, 3, 32), stepping(2, 2, 192)):                                # (sizes that the general kernel takes)
        assert goes_by(eng, [70, 1], [0, 500]) == goes_by(eng, [70, 1], [9, 5000]) != goes_by(eng, [70, 1], [0, 0])
    plain = stepping(32, 8, 128, kv_bits=None)
    assert goes_by(plain, [512], [7500]) == goes_by(plain, [512], [100])


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
