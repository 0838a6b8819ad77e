"""The model's blocks through 8-bit linear layers and through attention over key spans.

Against the same model through the 16-bit operators, and against plain torch.
8-bit products: rows and weights are off by half a step of max / 127 each.  For
normal values (max about 4 deviations over these widths) a step is 4 / 127 of a
deviation, its rounding sqrt(1/12) of that: 0.9% noise a factor, 1.3% a layer; some
30 layers in residual branches of a four-block model stay under 10% in all:
cosine >= 0.995.  16-bit paths that differ in where they round: cosine >= 0.9995
(2^-9 sqrt(steps) each); gradients through the whole model >= 0.998.
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.hunyuan import HunyuanConfig, Pipe, build_transformer, use_block_operators, use_dense_attention
from peco_b200.int8 import int8_weight, quantize_layer
from peco_b200.model import install_attention
from peco_b200.processor import InferenceContext, PecoConfig

pytestmark = pytest.mark.gpu

CFG = HunyuanConfig(hidden=256, heads=2, head_dim=128, dual_blocks=2, single_blocks=2, text_dim=64, pooled_dim=32)


def _inputs(batch=1, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, 16, 2, 16, 16, generator=g).to("cuda", dtype)
    txt = torch.randn(batch, 16, CFG.text_dim, generator=g).to("cuda", dtype)
    return x, torch.tensor([500.0] * batch, device="cuda"), txt, torch.ones(batch, 16, dtype=torch.bool, device="cuda"), \
        torch.randn(batch, CFG.pooled_dim, generator=g).to("cuda", dtype)


def _model(dtype=torch.bfloat16):
    model = build_transformer(CFG, device="cuda", dtype=dtype)
    with torch.no_grad():  # biases and modulation at sizes a trained model has
        g = torch.Generator(device="cuda").manual_seed(1)
        for name, p in model.named_parameters():
            if p.ndim == 1 and "norm_" not in name:
                p.copy_(0.2 * torch.randn(p.shape, generator=g, device="cuda"))
    return model


def _cosine(a, b):
    return torch.nn.functional.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0).item()


def test_blocks_in_8_bits():
    model = _model()
    use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=12))
    args = _inputs()
    with torch.no_grad():
        use_block_operators(model)
        ref = model(*args)
        before = model(*args)
        assert torch.equal(before, ref)
        use_block_operators(model, int8=True)
        got = model(*args)
        assert not torch.equal(got, ref) and _cosine(got, ref) >= 0.995
        assert torch.equal(model(*args), got)
        use_block_operators(model)           # and off again
        assert torch.equal(model(*args), ref)
        assert int8_weight(model.transformer_blocks[0].attn.to_q) is None
    assert _native.device_status(clear=True) == 0


def test_8_bits_around_the_sparse_call_and_in_a_step_graph():
    from peco_b200.graph import PecoStepGraph
    cfg = PecoConfig(num_q_centroids=8, num_k_centroids=16, top_p=1.0, min_kc_ratio=1.0, kmeans_iter_init=3,
                     kmeans_iter_step=2, warmup_steps=1, base_offset_bits=0)
    model = _model()
    install_attention(Pipe(model), cfg)
    use_block_operators(model, int8=True)
    args = _inputs()
    with torch.no_grad():
        torch.manual_seed(0)
        model(*args)                # dense warm-up, centroids initialised
        got = model(*args)          # sparse path, every pair kept
    graph = PecoStepGraph(model, *args)
    assert _cosine(graph(*args).clone(), got) >= 0.9999
    dense = _model()
    use_dense_attention(dense, InferenceContext(step=0, text_length=16, valid_text_length=16), spans=True)
    use_block_operators(dense, int8=True)
    with torch.no_grad():
        assert _cosine(got, dense(*args)) >= 0.995


def test_a_graph_keeps_the_weights_it_replays_over():
    from peco_b200.graph import PecoStepGraph
    cfg = PecoConfig(num_q_centroids=8, num_k_centroids=16, top_p=1.0, min_kc_ratio=1.0, kmeans_iter_init=3,
                     kmeans_iter_step=2, warmup_steps=0, base_offset_bits=0)
    model = _model()
    install_attention(Pipe(model), cfg)
    use_block_operators(model, int8=True)
    args = _inputs()
    with torch.no_grad():
        model(*args)
        model(*args)
    graph = PecoStepGraph(model, *args)
    first = graph(*args).clone()
    use_block_operators(model)             # the layers drop their 8-bit weights
    torch.cuda.empty_cache()
    junk = [torch.full((1 << 20,), 77, dtype=torch.int8, device="cuda") for _ in range(64)]
    assert _cosine(graph(*args), first) >= 0.9999  # (the centroids moved on by a step)
    del junk


def test_changed_weights_are_noticed():
    layer = torch.nn.Linear(64, 32, device="cuda", dtype=torch.bfloat16)
    assert quantize_layer(layer) and int8_weight(layer) is not None
    with torch.no_grad():
        layer.weight.mul_(2)
    with pytest.raises(RuntimeError, match="changed"):
        int8_weight(layer)
    assert quantize_layer(layer)
    layer.weight = torch.nn.Parameter(layer.weight.detach().clone())
    with pytest.raises(RuntimeError, match="changed"):
        int8_weight(layer)
    hooked = torch.nn.Linear(64, 32, device="cuda", dtype=torch.bfloat16)
    quantize_layer(hooked)
    hooked.register_forward_hook(lambda *_: None)
    assert int8_weight(hooked) is None and not quantize_layer(hooked)  # called instead
    assert not quantize_layer(torch.nn.Linear(8, 8, device="cuda")) and not quantize_layer(torch.nn.GELU())


@pytest.mark.parametrize("operators", [False, True])
def test_span_attention_of_one_and_of_several_prompts(operators):
    model = _model()
    ctx = InferenceContext(step=0, text_length=16, valid_text_length=12)
    args = _inputs()
    with torch.no_grad():
        use_dense_attention(model, ctx)
        ref = model(*args)
        use_block_operators(model, operators)
        use_dense_attention(model, ctx, spans=True)
        launches = _native.load().peco_launch_count()
        assert _cosine(model(*args), ref) >= 0.9995
        assert _native.load().peco_launch_count() - launches >= 8  # every layer's spans and attention
        # several prompts of their own lengths: each as if alone
        both = _inputs(batch=3, seed=3)
        lengths = torch.tensor([16, 5, 0], device="cuda")
        use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=lengths), spans=True)
        got = model(*both)
        for i, n in enumerate(lengths.tolist()):
            use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=n), spans=True)
            assert _cosine(got[i:i + 1], model(*(t[i:i + 1] for t in both))) >= 0.9999
    assert _native.device_status(clear=True) == 0


def test_training_through_the_operators():
    """Gradients of a loss over two prompts against the same model in fp32 torch."""
    lengths = torch.tensor([16, 7], device="cuda")
    model, plain = _model(), _model(torch.float32)
    with torch.no_grad():
        for p, r in zip(model.parameters(), plain.parameters()):
            r.copy_(p)
    use_block_operators(model)
    use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=lengths), spans=True)
    args = _inputs(batch=2, seed=5)
    target = torch.randn(args[0].shape, generator=torch.Generator().manual_seed(9)).to("cuda", torch.bfloat16)
    out = model(*args)
    grads = torch.autograd.grad((out * target).sum(), list(model.parameters()), allow_unused=True)
    total = None
    for i, n in enumerate(lengths.tolist()):  # a prompt at a time, as the fp32 processor takes them
        use_dense_attention(plain, InferenceContext(step=0, text_length=16, valid_text_length=n))
        one = [t[i:i + 1].float() if t.is_floating_point() and t.dim() > 1 else t[i:i + 1] for t in args]
        g = torch.autograd.grad((plain(*one) * target[i:i + 1].float()).sum(), list(plain.parameters()), allow_unused=True)
        total = g if total is None else [a if b is None else b if a is None else a + b for a, b in zip(total, g)]
    checked = 0
    for (name, _), a, b in zip(model.named_parameters(), grads, total):
        assert (a is None) == (b is None), name
        if a is None or b.abs().max() == 0:
            continue
        assert torch.isfinite(a).all(), name
        # small gradients are differences of large ones: their noise is that of bf16 rows
        assert _cosine(a, b) >= (0.998 if b.ndim > 1 else 0.98), (name, _cosine(a, b))
        checked += 1
    assert checked > 60
    with pytest.raises(RuntimeError, match="no gradient"):
        use_block_operators(model, int8=True)
        model(*args)
    assert _native.device_status(clear=True) == 0
