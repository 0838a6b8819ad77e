"""The erf form of GELU over its whole negative side, value and gradient, on the GPU against 64 bits.

One product per output (K = 1, factor 1), so that nothing but the activation
and the rounding of the result stands between z and it.  Tolerance: u of the
result (2^-8 bf16, 2^-11 fp16) and 2^-16 of the size of the terms, what fp32 can
give where exp(-z^2 / 2) is formed from an exponent of up to 2^7; half the
smallest subnormal of fp16, and the smallest normal fp32 (2^-126) in bf16.
"""

import math

import pytest
import torch

from peco_b200.linear import linear_act, linear_act_backward

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def _values(dtype):
    """Every value of the type between -12.5 and 12.5 in steps of at least 2^-9."""
    z = torch.arange(-12.5, 12.5, 2.0 ** -9, device=DEV, dtype=torch.float64).to(dtype)
    return z.unique()


def _phi(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2)), torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _near(got, ref, size, dtype):
    err = (got.double() - ref).abs()
    bound = U[dtype] * ref.abs() + 2.0 ** -16 * size * (1 + U[dtype]) + TINY[dtype]
    worst = (err - bound).argmax()
    assert (err <= bound).all(), (ref[worst].item(), err[worst].item(), bound[worst].item())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_tail(dtype):
    z = _values(dtype)
    one = torch.ones(1, 1, device=DEV, dtype=dtype)
    cdf, _ = _phi(z.double())
    for x, w in ((z[:, None], one), (one, z[:, None])):  # down the rows, and along the columns
        _near(linear_act(x, w, activation="gelu").flatten(), z.double() * cdf, (z.double() * cdf).abs(), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_gradient_tail(dtype):
    z = _values(dtype)
    n = z.numel()
    one = torch.ones(1, 1, device=DEV, dtype=dtype)
    cdf, pdf = _phi(z.double())
    slope, size = cdf + z.double() * pdf, cdf + (z.double() * pdf).abs()
    ones = torch.ones(1, n, device=DEV, dtype=dtype)
    for gate in (None, ones[0]):
        g = linear_act_backward(ones, one, ones.t().contiguous(), preact=z[None], activation="gelu", gate=gate, bias=True)
        _near(g.bias, slope, size, dtype)
        _near(g.weight[:, 0], slope, size, dtype)  # dz, rounded for the product with x = 1
        if gate is not None:
            _near(g.gate, z.double() * cdf, (z.double() * cdf).abs(), dtype)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("gated", [False, True])
def test_gradient_past_the_range_of_the_saved_preactivation(act, gated):
    # float16 saves a pre-activation of -90000 as -infinity: the slope there is 0 and the value 0, far above it is 1
    x = torch.tensor([[-300.0], [300.0], [-1.0]], device=DEV, dtype=torch.float16, requires_grad=True)
    w = torch.tensor([[300.0], [-300.0]], device=DEV, dtype=torch.float16)
    gate = torch.tensor([0.5, 0.5], device=DEV, dtype=torch.float16, requires_grad=True) if gated else None
    out = linear_act(x, w, activation=act, gate=gate)
    down, up = (out[0, 0], out[1, 1]), (out[1, 0], out[0, 1])  # at -90000 and at 90000
    assert all(v == 0 for v in down) and all(v.isinf() if not gated else v > 44000 for v in up)
    pick = torch.zeros_like(out)
    pick[0, 0] = pick[1, 1] = 1.0
    grads = torch.autograd.grad(out, (x, gate) if gated else (x,), pick, retain_graph=True)
    assert all((g == 0).all() for g in grads)
    pick = torch.zeros_like(out)
    pick[1, 0] = 1.0
    (gx,) = torch.autograd.grad(out, x, pick)
    assert torch.equal(gx[:, 0], torch.tensor([0.0, 150.0 if gated else 300.0, 0.0], device=DEV, dtype=torch.float16))
    # a pre-activation that is no number stays none
    one = torch.ones(1, 1, device=DEV, dtype=torch.float16)
    g = linear_act_backward(one, one, one, preact=one * float("nan"), activation=act, gate=one[0], bias=True)
    assert g.bias.isnan().all() and g.gate.isnan().all() and g.x.isnan().all()
