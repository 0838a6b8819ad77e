"""8-bit weights that are kept with layers: what owns them, and what replays over them.  Without a GPU."""

import contextlib
from types import SimpleNamespace

import pytest
import torch
import torch.nn as nn

from peco_b200 import int8
from peco_b200.graph import PecoStepGraph
from peco_b200.hunyuan import HunyuanConfig, build_transformer, use_block_operators


@pytest.fixture
def no_capture(monkeypatch):
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: SimpleNamespace(replay=lambda: None))
    monkeypatch.setattr(torch.cuda, "graph", lambda graph: contextlib.nullcontext())


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.layer = nn.Linear(16, 8)
        keep(self.layer)
        ctx = SimpleNamespace(step=1, text_length=0, valid_text_length=0)
        self._peco_context = ctx
        self._peco_processors = [SimpleNamespace(config=SimpleNamespace(warmup_steps=0, warmup_layers=0), layer_idx=0, context=ctx,
                                                 q_centroids=torch.zeros(1, 1, 2, 4), k_centroids=torch.zeros(1, 1, 2, 4))]

    def forward(self, x):
        return x + 1


def keep(layer):
    rows = int8.QuantizedRows(torch.zeros(layer.weight.shape, dtype=torch.int8), torch.ones(layer.weight.shape[0]))
    layer.int8 = int8._layer_int8(rows, layer.weight)


def scale(layer):
    with torch.no_grad():
        layer.weight.mul_(2)


def replace(layer):
    layer.weight = nn.Parameter(layer.weight.detach() * 2)


def repoint(layer):
    layer.weight.data = layer.weight.data * 2


@pytest.mark.parametrize("again", [False, True])
@pytest.mark.parametrize("change", [scale, replace, repoint])
def test_a_graph_over_8_bit_weights_notices_their_change(no_capture, change, again):
    """Also where the layer was quantised again: the graph has the values of its capture."""
    model = Model()
    graph = PecoStepGraph(model, torch.zeros(3))
    assert (graph(torch.zeros(3)) == 1).all()
    change(model.layer)
    if again:
        keep(model.layer)
    with pytest.raises(RuntimeError, match="capture"):
        graph(torch.zeros(3))
    if again:
        assert (PecoStepGraph(model, torch.zeros(3))(torch.zeros(3)) == 1).all()


def test_a_graph_outlives_the_8_bit_form(no_capture):
    model = Model()
    graph = PecoStepGraph(model, torch.zeros(3))
    del model.layer.int8  # 16 bits again: the weights are the same
    assert (graph(torch.zeros(3)) == 1).all()


def test_an_attribute_of_that_name_stays():
    """use_block_operators drops what it keeps with layers, not what others keep there under the same name."""
    model = build_transformer(HunyuanConfig(hidden=32, heads=2, head_dim=16, dual_blocks=1, single_blocks=1, text_dim=8, pooled_dim=8),
                              device="cpu", dtype=torch.bfloat16)
    block = model.transformer_blocks[0]
    block.attn.to_q.int8 = block.ff[0].int8 = True
    keep(block.attn.to_k)
    for args in ({}, dict(enabled=False), dict(int8=True)):
        use_block_operators(model, **args)
        assert block.attn.to_q.int8 is True and block.ff[0].int8 is True
        assert "int8" not in vars(block.attn.to_k)
