"""Scratch that outlives a step: what a capture may leave behind."""
import pytest
import torch

from vlrf_b200.parts.context import Workspace


class Capture:
    """Stands for a stream that is capturing: a fill is recorded, and memory holds what it held."""

    def __init__(self, monkeypatch):
        self.on = False
        zeros, fill = torch.zeros, torch.Tensor.zero_
        monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.on)
        monkeypatch.setattr(torch, "zeros", lambda *a, **kw: zeros(*a, **kw).fill_(7) if self.on else zeros(*a, **kw))
        monkeypatch.setattr(torch.Tensor, "zero_", lambda t: t if self.on else fill(t))


def test_counters_first_made_in_a_capture_that_never_runs_are_zero_afterwards(monkeypatch):
    ws, capture = Workspace("cpu"), Capture(monkeypatch)
    capture.on = True
    ws.get_zeroed("counters", 5, torch.int32)
    ws.get_zeroed("counters", 3, torch.int32)              # (the step's other layers)
    capture.on = False
    assert not ws.get_zeroed("counters", 5, torch.int32).any()
    ws.get_zeroed("counters", 5, torch.int32)[2] = 9       # whoever uses it leaves it zero: it is not filled again and again
    assert int(ws.get_zeroed("counters", 5, torch.int32)[2]) == 9


def test_counters_that_grow_in_a_capture_that_never_runs_are_zero_afterwards(monkeypatch):
    ws, capture = Workspace("cpu"), Capture(monkeypatch)
    ws.get_zeroed("counters", 2, torch.int32)
    capture.on = True
    ws.get_zeroed("counters", 8, torch.int32)
    capture.on = False
    assert not ws.get_zeroed("counters", 8, torch.int32).any()


def test_a_workspace_without_a_device():
    ws = Workspace("cpu")
    assert not ws.get_zeroed("counters", 4, torch.int32).any() and not ws.get_zeroed("counters", 9, torch.int32).any()


@pytest.mark.gpu
def test_counters_made_in_a_dropped_capture_on_the_device():
    """Two captures that are dropped unplayed, one that is kept, and a plain step behind them."""
    from vlrf_b200.engine.capture import capture_into
    ws = Workspace("cuda:0")
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with capture_into(graph):
            ws.get_zeroed("counters", 1 << 20, torch.int32)
        del graph
        buf = ws._bufs["counters"]
        buf.fill_(3)                                       # as whatever lay there before
    seen = torch.empty(1 << 20, dtype=torch.int32, device="cuda:0")
    kept = torch.cuda.CUDAGraph()
    with capture_into(kept):
        seen.copy_(ws.get_zeroed("counters", 1 << 20, torch.int32))
    kept.replay()
    assert not bool(seen.any())
    ws._bufs["counters"].fill_(3)
    assert not bool(ws.get_zeroed("counters", 1 << 20, torch.int32).any())
