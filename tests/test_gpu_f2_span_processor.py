"""Exact attention of a model on the package's kernels: the forms of a module that one prompt and several have in common.

Paths differ in where they round (2^-9 a step): cosine >= 0.9995 against each other.
"""

import pytest
import torch
import torch.nn as nn
import torch.nn as nn

from peco_b200 import _native
from peco_b200.hunyuan import HunyuanConfig, build_transformer, use_block_operators, use_dense_attention
from peco_b200.processor import InferenceContext

pytestmark = pytest.mark.gpu


def prompts(cfg, batch):
    g = torch.Generator().manual_seed(4)
    def make(*shape):
        return torch.randn(*shape, generator=g).to("cuda", torch.bfloat16).repeat(batch, *[1] * (len(shape) - 1))
    return make(1, 16, 2, 16, 16), torch.tensor([500.0] * batch, device="cuda"), make(1, 16, cfg.text_dim), \
        torch.ones(batch, 16, dtype=torch.bool, device="cuda"), make(1, cfg.pooled_dim)


def close(a, b):
    return torch.nn.functional.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0).item() >= 0.9995


@pytest.mark.parametrize("operators", [False, True])
@pytest.mark.parametrize("axes", [(8, 12, 12), (16, 40, 40), (16, 56, 56)])
def test_head_dimensions(axes, operators):
    cfg = HunyuanConfig(hidden=2 * sum(axes), heads=2, head_dim=sum(axes), dual_blocks=1, single_blocks=1, text_dim=64, pooled_dim=32,
                        rope_axes=axes)
    model = build_transformer(cfg, device="cuda", dtype=torch.bfloat16)
    use_block_operators(model, operators)
    use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=12), spans=True)
    with torch.no_grad():
        one, two = model(*prompts(cfg, 1)), model(*prompts(cfg, 2))
    assert one.isfinite().all() and close(one, two[:1]) and close(one, two[1:])
    assert _native.device_status(clear=True) == 0


def test_modules_without_norms():
    cfg = HunyuanConfig(hidden=128, heads=2, head_dim=64, dual_blocks=1, single_blocks=1, text_dim=64, pooled_dim=32,
                        rope_axes=(16, 24, 24))
    model = build_transformer(cfg, device="cuda", dtype=torch.bfloat16)
    for block in [*model.transformer_blocks, *model.single_transformer_blocks]:
        for name in ("norm_q", "norm_k", "norm_added_q", "norm_added_k"):
            setattr(block.attn, name, None)
    use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=12), spans=True)
    with torch.no_grad():
        one, two = model(*prompts(cfg, 1)), model(*prompts(cfg, 2))
    assert one.isfinite().all() and close(one, two[:1]) and close(one, two[1:])


@pytest.mark.parametrize("batch", [1, 2])
def test_modules_without_output_layers(batch):
    """As single-stream modules of other libraries: no such attributes at all."""
    class Single(nn.Module):
        def __init__(self):
            super().__init__()
            self.heads = 2
            self.to_q, self.to_k, self.to_v = (nn.Linear(128, 128) for _ in range(3))
            self.norm_q = self.norm_k = self.add_q_proj = None

    from peco_b200.hunyuan import SpanProcessor
    module = Single().to("cuda", torch.bfloat16)
    call = SpanProcessor(InferenceContext(step=0, text_length=16, valid_text_length=12))
    x, text = (torch.randn(1, n, 128, device="cuda").bfloat16().repeat(batch, 1, 1) for n in (40, 16))
    with torch.no_grad():
        video, words = call(module, x, text)
    assert video.shape == x.shape and words.shape == text.shape and video.isfinite().all()
