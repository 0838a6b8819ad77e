"""Several step graphs of one model: each replays over tensors of its own."""

import pytest
import torch

from peco_b200 import _native
from peco_b200.graph import PecoStepGraph
from peco_b200.hunyuan import HunyuanConfig, Pipe, build_transformer, use_block_operators
from peco_b200.model import install_attention, reset_state
from peco_b200.processor import PecoConfig

pytestmark = pytest.mark.gpu

CFG = HunyuanConfig(hidden=256, heads=2, head_dim=128, dual_blocks=2, single_blocks=2, text_dim=64, pooled_dim=32)


def test_an_older_graph_replays_after_a_newer_one_and_a_reset():
    model = build_transformer(CFG, device="cuda", dtype=torch.bfloat16)
    install_attention(Pipe(model), PecoConfig(num_q_centroids=8, num_k_centroids=16, top_p=1.0, min_kc_ratio=1.0,
                                              kmeans_iter_init=3, kmeans_iter_step=2, warmup_steps=0, base_offset_bits=0))
    g = torch.Generator().manual_seed(0)
    mask = torch.ones(1, 16, dtype=torch.bool, device="cuda")
    args = (torch.randn(1, 16, 2, 16, 16, generator=g).to("cuda", torch.bfloat16), torch.tensor([500.0], device="cuda"),
            torch.randn(1, 16, CFG.text_dim, generator=g).to("cuda", torch.bfloat16), mask,
            torch.randn(1, CFG.pooled_dim, generator=g).to("cuda", torch.bfloat16))
    wider = (torch.randn(1, 16, 2, 16, 32, generator=g).to("cuda", torch.bfloat16), *args[1:])
    with torch.no_grad():
        model(*args)
        want = model(*args)
        first = PecoStepGraph(model, *args)
        use_block_operators(model)
        second = PecoStepGraph(model, *args)
        reset_state(Pipe(model))
        model(*wider)  # other centroids and other tables
        torch.cuda.empty_cache()
        for graph in (first, second, first):
            got = graph(*args)
            # every pair is kept, so only rounding separates the two: bf16 over four blocks
            assert torch.nn.functional.cosine_similarity(got.double().flatten(), want.double().flatten(), dim=0) >= 0.999
    assert _native.device_status(clear=True) == 0
