"""quantize_rows and linear_int8 on the GPU against the definition in 64 bits.

The integers are those of the exact quotients, compared for equality.  The
products of integers are exact, so with u the unit roundoff of the output type
(2^-8 bf16, 2^-11 fp16) and e = 2^-24: a sum of up to 2^31 rounds to fp32 (e), is
multiplied by two rounded scales (4 e with theirs), the bias is added (e of the
result), the activation's slope is at most 1.13 and its fp32 value within 2^-18
(the erf and tanh forms at these sizes), gate and residual add e each: altogether
8 e of the sum of magnitudes, times the gate, and u of the result.
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.int8 import QuantizedRows, linear_int8, quantize_rows

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _rounded64(x):
    """(integers, scales) of [..., K] rows by the definition: whole part and remainder of 127 |x| / max."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    size = x.abs() * 127
    whole = torch.floor(size / top)
    rest = 2 * (size - whole * top)
    up = (rest > top) | ((rest == top) & (whole % 2 == 1))
    return torch.where(top > 0, torch.sign(x) * (whole + up), torch.zeros_like(x)), top[..., 0] / 127


def _act64(z, act):
    fn = torch.nn.functional
    return {None: lambda t: t, "gelu_tanh": lambda t: fn.gelu(t, approximate="tanh"), "gelu": fn.gelu, "silu": fn.silu}[act](z)


def _expected(values, scales, w, bias, act, gate, residual):
    z = (values.double() @ w.values.double().t()) * scales.double()[..., None] * w.scales.double()
    size = z.abs()
    if bias is not None:
        z, size = z + bias.double(), size + bias.double().abs()
    y = _act64(z, act)
    slack = 8 * 2.0 ** -24 * 1.13 * size + 2.0 ** -18 * y.abs()
    if gate is not None:
        g = gate.double() if gate.dim() != 2 else gate.double()[:, None]
        y, slack = y * g, slack * g.abs()
    if residual is not None:
        y = y + residual.double()
    return y, slack + 2.0 ** -23 * y.abs()


def _check(got, ref, slack):
    u = U[got.dtype]
    err = (got.double() - ref).abs()
    assert (err <= u * ref.abs() + slack * (1 + u) + 2.0 ** -24).all(), (err - u * ref.abs() - slack).max().item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 64), (300, 1000), (9, 1024), (9, 1032), (17, 2048), (33, 2056),
                                    (33, 4096), (6, 4104), (5, 8192), (3, 8200), (2, 16384), (2, 16392), (4, 1001),
                                    (2501, 2047), (7, 2049), (5, 4095), (3, 4097), (5000, 1024), (2700, 3000)])
def test_integers_are_those_of_the_exact_quotient(rows, k, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows * k)
    x = _normal(g, rows, k, std=0.3, dtype=dtype)
    x[0, 0] = 2 * x[0].abs().amax()  # some rows with one large element
    x[-1] = x[-1].abs().amax() * torch.randint(-256, 257, (k,), generator=g, device=DEV).to(dtype) / 254  # ties
    got = quantize_rows(x)
    values, scales = _rounded64(x)
    assert got.values.shape == (rows, k) and got.scales.shape == (rows,)
    assert torch.equal(got.values.double(), values)
    assert torch.equal(got.scales, (x.abs().amax(-1).double() / 127).float())
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_every_pair_of_significands(dtype):
    bits = 8 if dtype is torch.bfloat16 else 11
    top = torch.arange(1 << (bits - 1), 1 << bits, device=DEV, dtype=torch.float64)
    if dtype is torch.float16:
        top = top[::3]
    part = torch.arange(1 << (bits - 1), 1 << bits, device=DEV, dtype=torch.float64)
    for s in range(10):
        x = (part * 2.0 ** -s).expand(len(top), -1)
        x = torch.where(x <= top[:, None], x, torch.zeros_like(x))
        x = torch.cat((x, top[:, None], -x), 1).to(dtype)
        assert torch.equal(quantize_rows(x).values.double(), _rounded64(x)[0])


def test_special_rows():
    for dtype in (torch.bfloat16, torch.float16):
        for width in (64, 67):
            x = torch.ones(7, width, device=DEV, dtype=dtype)
            x[0] = 0
            x[1, 5] = float("inf")
            x[2, 6] = float("-inf")
            x[3, 7] = float("nan")
            x[4] *= torch.finfo(dtype).smallest_normal / 2 ** 6  # subnormal
            x[5] *= torch.finfo(dtype).max
            x[5, ::2] *= -1
            values, scales = quantize_rows(x)
            assert torch.equal(scales[0].cpu(), torch.tensor(0.0)) and values[:4].abs().max() == 0
            assert scales[1:4].isnan().all()
            assert (values[4:7].abs() == 127).all() and (values[5, ::2] == -127).all()
            assert torch.equal(scales[4:], (x[4:].abs().amax(-1).double() / 127).float())
            w = quantize_rows(torch.ones(40, width, device=DEV, dtype=dtype))
            for out in (linear_int8(x, w), linear_int8(QuantizedRows(values, scales), w, dtype=dtype)):
                assert (out[0] == 0).all() and out[1:4].isnan().all() and not out[4].isnan().any()
                assert not out[6].isnan().any()


def test_rows_side_by_side_and_strided():
    g = torch.Generator(device=DEV).manual_seed(0)
    for k, k2, pad in ((64, 192, 8), (1001, 40, 3), (24, 1000, 0), (3, 5, 1)):
        x = _normal(g, 4, 25, k + pad)[..., :k]
        x2 = _normal(g, 100, k2 + pad, std=3.0)[:, :k2].view(4, 25, k2) if pad == 0 else _normal(g, 4, 25, k2, std=3.0)
        got = quantize_rows(x, x2)
        values, scales = _rounded64(torch.cat((x, x2), -1))
        assert got.values.shape == (4, 25, k + k2) and torch.equal(got.values.double(), values)
        assert ((got.scales.double() - scales).abs() <= 2.0 ** -24 * scales).all()


SHAPES = [(1, 1, 64, 8), (1, 1, 1, 1), (1, 1, 1001, 77), (1, 5, 1, 3), (1, 17, 40, 24), (1, 128, 128, 128),
          (1, 129, 144, 136), (2, 65, 400, 130), (3, 33, 1001, 77), (1, 300, 520, 264), (4, 256, 1536, 1032),
          (1, 1, 4096, 3000), (1, 1500, 272, 2056), (1, 250, 8208, 520), (2, 1021, 528, 1288), (1, 256, 12288, 1024),
          (1, 128, 6144, 512), (1, 6400, 144, 3080), (1, 4500, 1000, 1536)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear(shape, dtype):
    b, t, k, n = shape
    for i, act in enumerate((None, "gelu_tanh", "gelu", "silu")):
        g = torch.Generator(device=DEV).manual_seed(i)
        x = _normal(g, b, t, k, dtype=dtype)
        w = quantize_rows(_normal(g, n, k, std=k ** -0.5, dtype=dtype))
        bias = _normal(g, n, dtype=dtype) if i != 1 else None
        gate = (_normal(g, b, 1, n, dtype=dtype), None, _normal(g, n, dtype=dtype), _normal(g, b, 3, n, dtype=dtype)[:, 1])[i]
        residual = _normal(g, b, t, n, dtype=dtype) if i % 2 == 0 else None
        args = dict(activation=act, gate=gate, residual=residual)
        values, scales = _rounded64(x)
        ref, slack = _expected(values, scales, w, bias, act, gate, residual)
        got = linear_int8(x, w, bias, **args)
        _check(got, ref, slack)
        assert torch.equal(linear_int8(quantize_rows(x), w, bias, dtype=dtype, **args), got)
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("k,k2,n", [(64, 128, 96), (1001, 55, 77), (512, 2048, 520)])
def test_linear_of_joined_rows(k, k2, n):
    g = torch.Generator(device=DEV).manual_seed(k)
    x, x2 = _normal(g, 2, 70, k), _normal(g, 2, 70, k2, std=2.0)
    w = quantize_rows(_normal(g, n, k + k2, std=0.05))
    values, scales = _rounded64(torch.cat((x, x2), -1))
    _check(linear_int8(x, w, x2=x2), *_expected(values, scales, w, None, None, None, None))


def test_largest_sums_stay_exact():
    """Integers at their bounds over the longest rows: sums near 2^31."""
    k = 131071
    values = torch.full((3, k), -128, dtype=torch.int8, device=DEV)
    values[1] = 127
    ones = torch.ones(3, device=DEV)
    w = QuantizedRows(torch.full((33, k), -128, dtype=torch.int8, device=DEV), torch.full((33,), 2.0 ** -20, device=DEV))
    out = linear_int8(QuantizedRows(values, ones), w, dtype=torch.bfloat16).double()
    ref = torch.tensor([128.0 * 128 * k, -127.0 * 128 * k, 128.0 * 128 * k], device=DEV, dtype=torch.float64) * 2.0 ** -20
    assert ((out - ref[:, None]).abs() <= 2.0 ** -8 * ref.abs()[:, None]).all()


def test_unaligned_and_strided_integers():
    g = torch.Generator(device=DEV).manual_seed(4)
    x, wide = _normal(g, 90, 333), _normal(g, 50, 333)
    q, w = quantize_rows(x), quantize_rows(wide)
    ref = linear_int8(q, w, dtype=torch.bfloat16)
    loose = QuantizedRows(q.values.contiguous(), q.scales)              # rows 333 bytes apart
    tight = QuantizedRows(w.values.contiguous(), w.scales)
    shifted = QuantizedRows(torch.cat((w.values[:, :1], w.values), 1)[:, 1:], w.scales)
    column = QuantizedRows(w.values.t().contiguous().t(), w.scales)     # columns adjacent
    for a in (q, loose):
        for b in (w, tight, shifted, column):
            assert torch.equal(linear_int8(a, b, dtype=torch.bfloat16), ref)


def test_streams_capture_and_empty_rows():
    g = torch.Generator(device=DEV).manual_seed(5)
    x, bias = _normal(g, 64, 256), _normal(g, 96)
    w = quantize_rows(_normal(g, 96, 256))
    ref = linear_int8(x, w, bias, activation="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_int8(x, w, bias, activation="silu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    static = torch.zeros_like(x)
    graphs = []
    for _ in range(2):  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = linear_int8(static, w, bias, activation="silu")
        graphs.append((graph, out))
    static.copy_(x)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, ref) for _, out in graphs)
    assert linear_int8(x[:0], w).shape == (0, 96)
    empty = quantize_rows(x[:0])
    assert empty.values.shape == (0, 256) and empty.scales.shape == (0,)
    assert linear_int8(empty, w, dtype=torch.bfloat16).shape == (0, 96)
