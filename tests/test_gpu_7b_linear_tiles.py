"""linear_act where one CTA finishes several tiles, on the GPU against the definition in 64 bits.

Tolerances as in test_gpu_7_linear: one rounding of the result (u |out|), the
fp32 sum of K products (K 2^-24 sum |x||w|, times the gate) and 2^-23 of the
value for the steps after it.
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.linear import linear_act, linear_act_backward

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _normal(seed, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return lambda *shape, std=1.0: (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _within(got, ref, slack, u):
    err = (got.double() - ref).abs()
    assert (err <= u * ref.abs() + slack * (1 + u) + 2.0 ** -24).all(), (err - u * ref.abs() - slack).max().item()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,k,n", [(600, 64, 24576), (6750, 128, 12288), (300, 64, 40000)])
def test_gate_without_bias_past_the_last_rows(rows, k, n, residual):
    # the last row tile leaves the second CTA of a pair without rows (and without a gate row) between tiles that have
    # them; each tile's columns take their own piece of the gate
    assert 0 < rows % 256 <= 128
    normal = _normal(rows)
    x, w, gate = normal(rows, k), normal(n, k, std=k ** -0.5), normal(n)
    r = normal(rows, n) if residual else None
    got = linear_act(x, w, gate=gate, residual=r)
    y = (x.double() @ w.double().t()) * gate.double()
    slack = (k + 2) * 2.0 ** -24 * (x.double().abs() @ w.double().abs().t()) * gate.double().abs()
    if residual:
        y += r.double()
    _within(got, y, slack + 2.0 ** -23 * y.abs(), U[torch.bfloat16])
    del y, slack
    for _ in range(50):
        assert torch.equal(linear_act(x, w, gate=gate, residual=r), got)
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("rows", [1, 31, 33, 97, 127, 130, 161, 255])
@pytest.mark.parametrize("k,n", [(4096, 700), (2048, 5000)])
def test_sums_shared_out_over_ragged_rows(rows, k, n):
    # K over the groups of a cluster, with warps some of whose lanes have no row
    normal = _normal(rows + k)
    x, w, b = normal(rows, k), normal(n, k, std=k ** -0.5), normal(n)
    got = linear_act(x, w, b)
    y = x.double() @ w.double().t() + b.double()
    slack = (k + 2) * 2.0 ** -24 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    _within(got, y, slack + 2.0 ** -23 * y.abs(), U[torch.bfloat16])
    for _ in range(10):
        assert torch.equal(linear_act(x, w, b), got)
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("samples,rows", [(65535, 1), (65536, 1), (70001, 2)])
def test_gradient_of_many_samples(samples, rows):
    # a gate row for every sample.  Sums of one or two rows (gate) and of all (bias): fp32 in runs, 2^-16 of their terms
    normal = _normal(samples)
    k, n = 16, 24
    x, w, gate = normal(samples, rows, k), normal(n, k, std=0.25), normal(samples, n)
    z, g = normal(samples, rows, n), normal(samples, rows, n)
    got = linear_act_backward(g, x, w, preact=z, activation="silu", gate=gate, bias=True)
    u = U[torch.bfloat16]
    zd, gd = z.double(), g.double()
    s = torch.sigmoid(zd)
    dz, value = gd * gate.double()[:, None] * (s * (1 + zd * (1 - s))), gd * zd * s
    _within(got.gate, value.sum(1), 2.0 ** -16 * value.abs().sum(1), u)
    _within(got.bias, dz.sum((0, 1)), 2.0 ** -16 * dz.abs().sum((0, 1)), u)
    _within(got.x, dz @ w.double(), (u + 2.0 ** -16) * (dz.abs() @ w.double().abs()), u)  # dz is rounded for the products
    flat, rows_x = dz.flatten(0, 1), x.double().flatten(0, 1)
    _within(got.weight, flat.t() @ rows_x, (u + (samples * rows) * 2.0 ** -24) * (flat.abs().t() @ rows_x.abs()), u)
    assert _native.device_status(clear=True) == 0
