"""linear_act and its gradient at sizes whose tiles outnumber the CTA groups: a
group walks several tiles, so that accumulators, barrier phases, the ring and
the staged vectors pass from one tile to the next, on one CTA and on pairs, on
tiles of one and of two accumulators, with ragged rows, columns and bands.
test_linear_tiles_cpu checks that the sizes are cut as they are meant to be.

Tolerances as in test_gpu_7_linear.
"""

import pytest
import torch
from test_gpu_7_linear import U, _case, _check, _check_grads, _forward64, _grads64

from peco_b200 import _native
from peco_b200.linear import linear_act, linear_act_backward

pytestmark = pytest.mark.gpu

# (samples, rows of each, k, k2, n), activation, bias, gate, residual; CTAs per tile, columns per accumulator,
# accumulators per tile, tile rows left over in the last band
FORWARD = [
    ((1, 100, 128, 0, 60000), None, False, "shared", True, (1, 128, 1, 0)),
    ((1, 37, 64, 0, 50000), "gelu", True, None, False, (1, 128, 1, 0)),
    ((2, 500, 200, 0, 24600), "silu", True, "sample", True, (2, 224, 1, 0)),
    ((1, 8348, 256, 0, 2500), None, False, "shared", True, (2, 256, 1, 1)),
    ((1, 700, 200, 320, 30000), "gelu_tanh", True, None, True, (2, 256, 1, 0)),
    ((1, 12500, 4096, 0, 12400), None, True, "shared", False, (2, 256, 1, 1)),
    ((1, 3330, 4160, 0, 10000), None, False, "shared", False, (2, 256, 2, 0)),
    ((1, 6750, 2000, 2160, 7000), None, True, "shared", True, (2, 224, 2, 0)),
    ((3, 3000, 3200, 0, 2600), None, True, "sample", True, (2, 224, 2, 0)),
    ((1, 808, 3136, 0, 5000), "gelu", True, None, False, (2, 160, 2, 0)),
]

# rows, k, n; the cut of the gradient of the rows (or, rows and n exchanged, of the weight)
BACKWARD = [
    ((12000, 3000, 1600), (2, 256, 2, 1)),
    ((9000, 4200, 1600), (2, 224, 2, 0)),
    ((8000, 6000, 2000), (2, 192, 2, 0)),
    ((15000, 4000, 1664), (2, 256, 1, 1)),
    ((7501, 2048, 1536), (2, 256, 2, 0)),
    ((20000, 4096, 1600), (2, 256, 2, 1)),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,act,bias,gate,residual,cut", FORWARD)
def test_forward(shape, act, bias, gate, residual, cut, dtype):
    b, rows, k, k2, n = shape
    c = _case(rows + k, b, rows, k, n, k2=k2, dtype=dtype, bias=bias, gate=gate, residual=residual)
    got = linear_act(**c, activation=act)
    _check(got, *_forward64(c, act), U[dtype])
    for _ in range(5):
        assert torch.equal(linear_act(**c, activation=act), got)
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("of", ["rows", "weight"])
@pytest.mark.parametrize("shape,cut", BACKWARD)
def test_backward(shape, cut, of):
    rows, k, n = shape if of == "rows" else shape[::-1]
    dtype = torch.float16 if shape[0] % 2000 else torch.bfloat16
    c = _case(rows, 1, rows, k, n, dtype=dtype, gate=None, residual=False)
    g = torch.Generator(device="cuda").manual_seed(n)
    grad, preact = (torch.randn((1, rows, n), generator=g, device="cuda").to(dtype) for _ in range(2))
    args = dict(preact=preact, activation="gelu_tanh", bias=True)
    got = linear_act_backward(grad, c["x"], c["weight"], **args)
    _check_grads(got, _grads64(c, "gelu_tanh", grad, preact), U[dtype], rows, n)
    for _ in range(5):
        again = linear_act_backward(grad, c["x"], c["weight"], **args)
        assert torch.equal(again.x, got.x) and torch.equal(again.weight, got.weight) and torch.equal(again.bias, got.bias)
    assert _native.device_status(clear=True) == 0
