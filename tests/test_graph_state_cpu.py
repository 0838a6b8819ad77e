"""What a captured graph replays over has to live as long as the graph.  Without
a GPU: capture and replay are stand-ins, the ownership is the real one."""

import contextlib
import gc
import weakref
from types import SimpleNamespace

import pytest
import torch

from peco_b200.graph import PecoCallGraph, PecoStepGraph


@pytest.fixture
def no_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: SimpleNamespace(replay=lambda: None))
    monkeypatch.setattr(torch.cuda, "graph", lambda graph: contextlib.nullcontext())


def _processor():
    return SimpleNamespace(config=SimpleNamespace(warmup_steps=0, warmup_layers=0), layer_idx=0, stage_events=None,
                           context=SimpleNamespace(step=1, text_length=0, valid_text_length=0),
                           q_centroids=torch.randn(1, 2, 4, 8), k_centroids=torch.randn(1, 2, 4, 8),
                           update_centroids_in_place=False, attention=lambda q, k, v: q + 1)


def test_step_graph_keeps_centroids_and_tables(no_capture):
    class Model:
        def __call__(self, x):
            return x + 1

    model = Model()
    processor = _processor()
    model._peco_processors, model._peco_context = [processor], processor.context
    model._rope = {"grid": (torch.zeros(4, 8), torch.zeros(4, 8))}
    first = PecoStepGraph(model, torch.zeros(3))
    used = [weakref.ref(t) for t in (processor.q_centroids, processor.k_centroids, *model._rope["grid"])]
    PecoStepGraph(model, torch.zeros(3))         # captures over centroids of its own
    processor.q_centroids = processor.k_centroids = None  # a new video
    model._rope = {"other grid": (torch.zeros(2, 8), torch.zeros(2, 8))}
    gc.collect()
    assert all(r() is not None for r in used)
    first(torch.zeros(3))
    del first
    gc.collect()
    assert all(r() is None for r in used)        # and no longer


def test_call_graph_keeps_its_centroids(no_capture, monkeypatch):
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    processor = _processor()
    q = torch.zeros(1, 2, 6, 8)
    first = PecoCallGraph(processor, q, q, q)
    used = [weakref.ref(t) for t in (processor.q_centroids, processor.k_centroids)]
    second = PecoCallGraph(processor, q, q, q)
    processor.q_centroids = processor.k_centroids = None
    gc.collect()
    assert all(r() is not None for r in used)
    assert all(a is b() for a, b in zip(first.centroids, used))
    assert all(a is not b for a, b in zip(first.centroids, second.centroids))
    first.set_centroids(torch.ones(1, 2, 4, 8), torch.ones(1, 2, 4, 8))
    assert (first.centroids[0] == 1).all() and not (second.centroids[0] == 1).all()
