"""When a model's captured graphs go: at once with the model, and never inside another model's capture, where
destroying a graph or freeing pinned memory is illegal and ends the process."""
import contextlib
import copy
import gc
import pickle
import weakref
from types import SimpleNamespace

import pytest
import torch

from src.model import graph_decode
from src.model.transformer import TinyTransformerLM


def _model():
    return TinyTransformerLM(16, 32, 2, 1, 64, 32, attention_backend="paged_reference").eval()


@contextlib.contextmanager
def _collector(on):
    was, limits = gc.isenabled(), gc.get_threshold()
    (gc.enable if on else gc.disable)()
    try:
        yield
    finally:
        gc.set_threshold(*limits)
        (gc.enable if was else gc.disable)()


def test_a_dropped_model_takes_its_runner_with_it():
    with _collector(False):
        model = _model()
        runner = weakref.ref(model._graph_runner())
        assert runner().model is model
        del model
        assert runner() is None


def test_a_copied_model_makes_its_own_runner():
    model = _model()
    runner = model._graph_runner()
    for other in (copy.deepcopy(model), pickle.loads(pickle.dumps(model))):
        assert other._graph_runner().model is other
        assert other._graph_runner() is not runner
    assert model._graph_runner() is runner and runner.model is model


class _Owner:
    """Stands for what owns a graph, in a cycle that only the collector can free."""

    def __init__(self, freed):
        self.me = self
        weakref.finalize(self, freed.append, True)


@pytest.mark.parametrize("fails", [False, True])
def test_nothing_is_collected_inside_a_capture(monkeypatch, fails):
    stream = SimpleNamespace(wait_stream=lambda other: None)
    monkeypatch.setattr(torch.cuda, "Stream", lambda **kw: stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: object())
    freed, capturing, seen = [], [], []

    @contextlib.contextmanager
    def graph(g):
        capturing.append(g)
        _Owner(freed)  # garbage from the capture's begin on
        try:
            yield
        finally:
            seen.append(list(freed))
            capturing.clear()

    monkeypatch.setattr(torch.cuda, "graph", graph)
    model = _model()
    runner = model._graph_runner()

    def forward(cap, pools):
        if capturing:
            kept = [[i] for i in range(20000)]  # container objects: what starts a collection
            if fails:
                raise ValueError("no step")
            return len(kept)

    monkeypatch.setattr(runner, "_static_forward", forward)
    cap = SimpleNamespace(ids=torch.zeros(1), graph=None, logits=None)
    with _collector(True):
        gc.set_threshold(50, 2, 2)
        with pytest.raises(ValueError, match="no step") if fails else contextlib.nullcontext():
            runner._capture(cap, [])
        assert seen == [[]]
        assert gc.isenabled()
    gc.collect()
    assert freed == [True]
    if not fails:
        assert cap.graph is not None and runner.captures == 1


def test_a_collector_that_was_off_stays_off(monkeypatch):
    stream = SimpleNamespace(wait_stream=lambda other: None)
    monkeypatch.setattr(torch.cuda, "Stream", lambda **kw: stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: object())
    monkeypatch.setattr(torch.cuda, "graph", lambda g: contextlib.nullcontext())
    model = _model()
    runner = model._graph_runner()
    monkeypatch.setattr(runner, "_static_forward", lambda cap, pools: None)
    with _collector(False):
        runner._capture(SimpleNamespace(ids=torch.zeros(1), graph=None, logits=None), [])
        assert not gc.isenabled()


def test_a_shallow_copy_makes_its_own_runner():
    """A shallow copy (module replication makes such) holds the original's runner, whose model may be gone."""
    model = _model()
    model._graph_runner()
    other = copy.copy(model)
    assert other._graph_runner().model is other
    assert model._graph_runner().model is model
    del model
    gc.collect()
    assert other._graph_runner().model is other
