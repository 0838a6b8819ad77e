"""A model on the block operators whose layers carry hooks and adapters: they run, and the result follows them."""

import pytest
import torch

from peco_b200.hunyuan import HunyuanConfig, build_transformer, use_block_operators, use_dense_attention
from peco_b200.processor import InferenceContext

pytestmark = pytest.mark.gpu

CFG = HunyuanConfig(hidden=256, heads=2, head_dim=128, dual_blocks=2, single_blocks=2, text_dim=64, pooled_dim=32)


def _model_and_inputs(dtype=torch.bfloat16):
    model = build_transformer(CFG, device="cuda", dtype=dtype)
    use_dense_attention(model, InferenceContext(step=0, text_length=16, valid_text_length=12))
    g = torch.Generator().manual_seed(0)
    mask = torch.zeros(1, 16, dtype=torch.bool)
    mask[0, :12] = True
    with torch.no_grad():  # modulation and gates at sizes that let every block count
        gd = torch.Generator(device="cuda").manual_seed(1)
        for name, p in model.named_parameters():
            if p.ndim == 1 and "norm_" not in name:
                p.copy_(0.2 * torch.randn(p.shape, generator=gd, device="cuda"))
    return model, (torch.randn(1, 16, 2, 16, 16, generator=g).to("cuda", dtype), torch.tensor([500.0], device="cuda"),
                   torch.randn(1, 16, CFG.text_dim, generator=g).to("cuda", dtype), mask.cuda(),
                   torch.randn(1, CFG.pooled_dim, generator=g).to("cuda", dtype))


def _cosine(a, b):
    return torch.nn.functional.cosine_similarity(a.double().flatten(), b.double().flatten(), dim=0).item()


def test_hooks_run_and_change_the_result():
    # tolerance: cosine 0.9995, the level at which bf16's 2^-9 roundings of a few dozen steps a block gather as noise
    model, args = _model_and_inputs()
    dual, single = model.transformer_blocks[0], model.single_transformer_blocks[1]
    layers = dict(q=dual.attn.to_q, text_v=dual.attn.add_v_proj, out=dual.attn.to_out[0], text_out=dual.attn.to_add_out,
                  mod=dual.img_mod, first=dual.ff[0], second=dual.ff_context[2], mlp=model.transformer_blocks[1].ff,
                  act=model.transformer_blocks[1].ff_context[1], single_mod=single.mod, single_mlp=single.proj_mlp,
                  single_out=single.proj_out)
    with torch.no_grad():
        plain = model(*args)
        seen = []
        for name, layer in layers.items():
            layer.register_forward_hook(lambda module, inputs, out, name=name: (seen.append(name), 1.5 * out)[1])
        want = model(*args)
        assert set(seen) == set(layers)
        use_block_operators(model)
        seen.clear()
        got = model(*args)
        assert set(seen) == set(layers)
    assert _cosine(got, want) >= 0.9995 > _cosine(plain, want)


def test_rotary_tables_stay_unless_positions_are_asked_for():
    from peco_b200 import _native
    model, args = _model_and_inputs()
    blocks = CFG.dual_blocks + CFG.single_blocks
    count = _native.load().peco_launch_count

    def run():
        before = count()
        with torch.no_grad():
            out = model(*args)
        return out, count() - before

    use_block_operators(model)
    tables, launches = run()
    use_block_operators(model, positions=True)
    positions, more = run()
    assert more == launches + blocks  # one pass over Q and K more in every block
    # the fused pass rounds Q and K once, the two passes twice: one more bf16 rounding of Q and K
    assert _cosine(tables, positions) >= 0.9995
    use_block_operators(model, False)
    assert torch.equal(run()[0], model(*args)) and not model.rotary_positions


@pytest.mark.parametrize("positions", [False, True])
def test_float16_model(positions):
    # the processor computes a float16 module in plain torch; tolerance as above, float16 rounds finer
    model, args = _model_and_inputs(torch.float16)
    with torch.no_grad():
        want = model(*args)
        use_block_operators(model, positions=positions)
        got = model(*args)
        assert torch.isfinite(got).all() and _cosine(got, want) >= 0.9995
        with pytest.raises(ValueError, match="rotary positions"):
            from peco_b200.rotary import AxialPositions
            short = AxialPositions(CFG.rope_axes, CFG.rope_theta, grid=(2, 8, 7))
            model.transformer_blocks[0].attn(torch.zeros(1, 128, 256, device="cuda", dtype=torch.float16), None, None, short)
