"""Which layers of a model the block operators may stand for: a layer that is
more than a plain linear map is called, so that its own work and its hooks
happen.  Without a GPU (the operators themselves refuse CPU tensors, so a layer
that was read instead of called shows as that refusal)."""

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from peco_b200 import hunyuan, processor
from peco_b200.hunyuan import RowParallelLinear, SINGLE
from peco_b200.linear import is_plain_linear


class Adapted(nn.Module):
    """A low-rank adapter around a layer, showing the layer's weight and bias."""

    def __init__(self, base):
        super().__init__()
        self.base = base
        self.down, self.up = nn.Linear(base.in_features, 2, bias=False), nn.Linear(2, base.out_features, bias=False)

    @property
    def weight(self):
        return self.base.weight

    @property
    def bias(self):
        return self.base.bias

    def forward(self, x):
        return self.base(x) + self.up(self.down(x))


class Scaled(nn.Linear):
    def forward(self, x):
        return 2 * super().forward(x)


class Marked(torch.Tensor):
    """Stands for a quantised weight: a tensor subclass with arithmetic of its own."""


def _row_parallel(n, k, cls=RowParallelLinear):
    layer = cls(n, k, [(0, k)], SINGLE)
    layer.in_features, layer.out_features = k, n
    return layer


def _others(n, k):
    """Layers that show a 2-D weight and compute more than its product."""
    class RowScaled(RowParallelLinear):
        def forward(self, x):
            return 2 * super().forward(x)

    hooked, before, back, patched = (nn.Linear(k, n) for _ in range(4))
    hooked.register_forward_hook(lambda module, args, out: 2 * out)
    before.register_forward_pre_hook(lambda module, args: (2 * args[0],))
    back.register_full_backward_hook(lambda module, gi, go: None)
    patched.forward = lambda x: F.linear(x, patched.weight) * 3
    reparametrised = nn.Linear(k, n)
    nn.utils.parametrizations.weight_norm(reparametrised)
    quantised = nn.Linear(k, n)
    quantised.weight = nn.Parameter(quantised.weight.detach().as_subclass(Marked))
    row_hooked = _row_parallel(n, k)
    row_hooked.register_forward_hook(lambda module, args, out: out + 1)
    return [Adapted(nn.Linear(k, n)), Adapted(_row_parallel(n, k)), Scaled(k, n), _row_parallel(n, k, RowScaled), hooked,
            before, back, patched, reparametrised, quantised, row_hooked]


def test_plain_layers():
    assert is_plain_linear(nn.Linear(8, 4)) and is_plain_linear(nn.Linear(8, 4, bias=False))
    assert is_plain_linear(_row_parallel(4, 8))
    assert not is_plain_linear(nn.Identity()) and not is_plain_linear(nn.Embedding(4, 8))
    handle = nn.modules.module.register_module_forward_hook(lambda *a: None)
    try:
        assert not is_plain_linear(nn.Linear(8, 4))
    finally:
        handle.remove()
    assert is_plain_linear(nn.Linear(8, 4))


def test_other_layers_are_called():
    torch.manual_seed(0)
    x, x2, gate, residual = torch.randn(1, 5, 8), torch.randn(1, 5, 4), torch.randn(1, 8), torch.randn(1, 5, 8)
    with torch.no_grad():
        for layer in _others(8, 8):
            assert not is_plain_linear(layer), type(layer)
            assert torch.equal(processor._project(layer, x), layer(x))
            assert torch.equal(hunyuan._linear(layer, x, "gelu_tanh"), F.gelu(layer(x), approximate="tanh"))
            assert torch.equal(hunyuan._row_operator(layer, x, gate, residual), residual + gate[:, None] * layer(x))
            assert torch.equal(torch.cat(hunyuan._modulation(layer, x[:, 0], 2), -1), layer(x[:, 0]))
        for layer in _others(8, 12):
            assert torch.equal(hunyuan._row_operator(layer, x, gate, residual, x2=x2),
                               residual + gate[:, None] * layer(torch.cat((x, x2), -1)))
        assert torch.equal(processor._project(nn.Identity(), x), x)


def test_other_mlps_are_called():
    torch.manual_seed(1)
    x, gate, residual = torch.randn(1, 5, 8), torch.randn(1, 8), torch.randn(1, 5, 8)

    def mlp(act=None):
        return nn.Sequential(nn.Linear(8, 16), act or nn.GELU(approximate="tanh"), _row_parallel(8, 16))

    hooked, inner = mlp(), mlp()
    hooked.register_forward_hook(lambda module, args, out: 2 * out)
    inner[1].register_forward_hook(lambda module, args, out: 2 * out)
    longer = nn.Sequential(*mlp(), nn.Dropout(0.0))
    with torch.no_grad():
        for ff in (mlp(nn.GELU()), mlp(nn.SiLU()), hooked, inner, longer):
            assert torch.equal(hunyuan._mlp_operator(ff, x, gate, residual), residual + gate[:, None] * ff(x))
        both = nn.Sequential(Adapted(nn.Linear(8, 16)), nn.GELU(approximate="tanh"), Scaled(16, 8))
        assert torch.equal(hunyuan._mlp_operator(both, x, gate, residual), residual + gate[:, None] * both(x))
        with pytest.raises(RuntimeError, match="CUDA"):  # as built: the operators
            hunyuan._mlp_operator(mlp().bfloat16(), x.bfloat16(), gate.bfloat16(), residual.bfloat16())
