"""A model whose blocks run through the block operators (norms, linears,
rotary positions) against the same model in plain torch.

Both compute in bf16 with fp32 accumulation and differ in where they round:
the operators round once per fused step, the torch path after every
elementwise step.  Tolerance: cosine >= 0.9995 of the model's output, the level
at which bf16's 2^-9 roundings of a few dozen steps per block accumulate as
noise (relative error about 2^-9 sqrt(steps * blocks) ~ 2e-2).
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.hunyuan import HunyuanConfig, Pipe, build_transformer, use_block_operators, use_dense_attention
from peco_b200.linear import linear_act, linear_act_backward
from peco_b200.model import install_attention
from peco_b200.norms import modulated_norm, modulated_norm_backward
from peco_b200.processor import InferenceContext, PecoConfig
from peco_b200.rotary import AxialPositions, rotate

pytestmark = pytest.mark.gpu

CFG = HunyuanConfig(hidden=256, heads=2, head_dim=128, dual_blocks=2, single_blocks=2, text_dim=64, pooled_dim=32)


def _inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(1, 16, 2, 16, 16, generator=g).to("cuda", torch.bfloat16)
    txt = torch.randn(1, 16, CFG.text_dim, generator=g).to("cuda", torch.bfloat16)
    mask = torch.zeros(1, 16, dtype=torch.bool)
    mask[0, :12] = True
    return x, torch.tensor([500.0], device="cuda"), txt, mask.cuda(), \
        torch.randn(1, CFG.pooled_dim, generator=g).to("cuda", torch.bfloat16)


def _model():
    model = build_transformer(CFG, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():  # biases and modulation at sizes a trained model has
        g = torch.Generator(device="cuda").manual_seed(1)
        for name, p in model.named_parameters():
            if p.ndim == 1 and "norm_" not in name:
                p.copy_(0.2 * torch.randn(p.shape, generator=g, device="cuda"))
    return model


def _cosine(a, b):
    return torch.nn.functional.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0).item()


def test_blocks_through_the_operators_match_the_torch_path():
    model = _model()
    use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=12))
    args = _inputs()
    with torch.no_grad():
        ref = model(*args)
        launches = _native.load().peco_launch_count()
        use_block_operators(model)
        got = model(*args)
        assert _native.load().peco_launch_count() - launches >= 2 * 12 + 2 * 5  # the operators ran
        use_block_operators(model, False)
        assert torch.equal(model(*args), ref)  # and switch off
    assert got.shape == ref.shape and torch.isfinite(got).all()
    assert _cosine(got, ref) >= 0.9995
    assert _native.device_status(clear=True) == 0


def test_operators_around_the_sparse_call_and_in_a_step_graph():
    from peco_b200.graph import PecoStepGraph
    cfg = PecoConfig(num_q_centroids=8, num_k_centroids=16, top_p=1.0, min_kc_ratio=1.0, kmeans_iter_init=3,
                     kmeans_iter_step=2, warmup_steps=1, base_offset_bits=0)
    model, dense = _model(), _model()
    install_attention(Pipe(model), cfg)
    use_block_operators(model)
    use_dense_attention(dense, InferenceContext(step=0, text_length=16, valid_text_length=12))
    args = _inputs()
    with torch.no_grad():
        torch.manual_seed(0)
        model(*args)                # dense warm-up, centroids initialised
        got = model(*args)          # sparse path, every pair kept
        assert _cosine(got, dense(*args)) >= 0.999
    graph = PecoStepGraph(model, *args)
    first = graph(*args).clone()
    assert _cosine(first, got) >= 0.9999


def test_processor_takes_positions():
    model = _model()
    use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=12))
    attn = model.transformer_blocks[0].attn
    from peco_b200.hunyuan import rope_3d
    grid = (2, 8, 8)
    x = torch.randn(1, 128, 256, device="cuda").to(torch.bfloat16)
    txt = torch.randn(1, 16, 256, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        ref = attn(x, txt, None, rope_3d(grid, CFG.rope_axes, CFG.rope_theta, "cuda"))
        got = attn(x, txt, None, AxialPositions(CFG.rope_axes, CFG.rope_theta, grid=grid))
        for a, b in zip(got, ref):
            assert _cosine(a, b) >= 0.9999
        with pytest.raises(ValueError, match="rotary positions"):
            attn(x, txt, None, AxialPositions(CFG.rope_axes, CFG.rope_theta, grid=(2, 8, 7)))


@pytest.mark.parametrize("width", [64, 1001])
def test_launches_in_a_row_are_ordered(width):
    # every kernel may start before the one in front of it has ended and has to wait for its results
    g = torch.Generator(device="cuda").manual_seed(3)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    rows, heads = 150, 2
    w1, w2 = normal(heads * 64, width, std=width ** -0.5), normal(width, heads * 64, std=0.1)
    gate, scale, b = normal(2, width), normal(2, width), normal(width)

    def chain(x, wait):
        kept = []
        for _ in range(6):
            h = modulated_norm(x, scale=scale, shift=gate)
            wait()
            q = linear_act(h, w1, activation="silu")
            wait()
            q = rotate(q.view(2, rows, heads, 64).transpose(1, 2), axes=(16, 24, 24), grid=(1, 10, 15))
            wait()
            y = linear_act(q.transpose(1, 2).reshape(2, rows, heads * 64), w2, b, gate=gate, residual=x)
            wait()
            d = linear_act_backward(q.transpose(1, 2).reshape(2, rows, heads * 64), h, w1, bias=True)
            wait()
            n = modulated_norm_backward(d.x, y, x, y, gate=gate, scale=scale)
            wait()
            x = modulated_norm(y, n.x, gate=n.gate)[1]
            wait()
            kept += [y, d.weight, d.bias, n.scale, x]
        torch.cuda.synchronize()
        return kept

    x = normal(2, rows, width)
    for a, c in zip(chain(x, torch.cuda.synchronize), chain(x, lambda: None)):
        assert torch.equal(a, c)
    assert _native.device_status(clear=True) == 0
