"""linear_act and its gradient on the GPU against the definition in 64 bits.

Tolerances.  u is the unit roundoff of the output type (2^-8 bf16, 2^-11 fp16).
Forward, element by element: one rounding of the result (u |out|), the fp32
sum of K products (K 2^-24 sum |x||w|, times the gate and the activation's
slope, at most 1.13) and the fp32 activation (2^-18 of its value).  Gradients
add the rounding of grad * gate * act' to the operands' type: u of the sum of
absolute products, element by element; over all elements, two independent
roundings of at most u each with zero mean stay below u in relative 2-norm.
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.linear import linear_act, linear_act_backward

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _act64(z, act):
    fn = torch.nn.functional
    return {None: lambda t: t, "gelu_tanh": lambda t: fn.gelu(t, approximate="tanh"), "gelu": fn.gelu,
            "silu": fn.silu}[act](z)


def _case(seed, b, t, k, n, k2=0, dtype=torch.bfloat16, bias=True, gate="sample", residual=True):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)

    return dict(x=normal(b, t, k), weight=normal(n, k + k2, std=(k + k2) ** -0.5), bias=normal(n) if bias else None,
                gate={"sample": lambda: normal(b, 1, n), "shared": lambda: normal(n), None: lambda: None}[gate](),
                residual=normal(b, t, n) if residual else None, x2=normal(b, t, k2) if k2 else None)


def _gate64(gate):
    return gate if gate is None or gate.dim() != 2 else gate[:, None]


def _forward64(c, act):
    d = {k: None if v is None else v.double() for k, v in c.items()}
    x = d["x"] if d["x2"] is None else torch.cat((d["x"], d["x2"]), -1)
    z = x @ d["weight"].t()
    size = x.abs() @ d["weight"].abs().t()
    if d["bias"] is not None:
        z, size = z + d["bias"], size + d["bias"].abs()
    y = _act64(z, act)
    slack = 1.13 * (x.shape[-1] + 2) * 2.0 ** -24 * size + 2.0 ** -18 * y.abs()
    if d["gate"] is not None:
        y, slack = y * _gate64(d["gate"]), slack * _gate64(d["gate"]).abs()
    if d["residual"] is not None:
        y = y + d["residual"]
    return y, slack + 2.0 ** -23 * y.abs()


def _check(got, ref, slack, u):
    err = (got.double() - ref).abs()
    # 2^-24: half the smallest step of a subnormal fp16
    assert (err <= u * ref.abs() + slack * (1 + u) + 2.0 ** -24).all(), (err - u * ref.abs() - slack).max().item()


SHAPES = [(1, 1, 64, 8), (1, 1, 1, 1), (1, 1, 1001, 77), (1, 5, 1, 3), (1, 17, 40, 24), (1, 128, 64, 128),
          (1, 129, 72, 136), (2, 65, 200, 130), (3, 33, 1001, 77), (1, 300, 520, 264), (4, 256, 1536, 1032),
          (1, 1, 4096, 3000), (1, 1500, 136, 2056), (1, 250, 4104, 520), (2, 1021, 264, 1288)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dtype):
    for i, act in enumerate((None, "gelu_tanh", "gelu", "silu")):
        c = _case(i, *shape, dtype=dtype, bias=i != 1, gate=("sample", None, "shared", "sample")[i], residual=i % 2 == 0)
        _check(linear_act(**c, activation=act), *_forward64(c, act), U[dtype])
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("k,k2", [(64, 128), (72, 40), (33, 31), (1000, 24), (8, 3000), (128, 1)])
@pytest.mark.parametrize("rows", [3, 200, 1100])
def test_two_inputs(k, k2, rows):
    c = _case(k + rows, 2, rows, k, 200, k2=k2)
    _check(linear_act(**c, activation="silu"), *_forward64(c, "silu"), U[torch.bfloat16])
    joined = dict(c, x=torch.cat((c["x"], c["x2"]), -1), x2=None)
    _check(linear_act(**joined, activation="silu"), *_forward64(c, "silu"), U[torch.bfloat16])


@pytest.mark.parametrize("rows", [1, 40, 700])
def test_strided_operands_and_their_surroundings(rows):
    """Views into wider buffers whose other entries are NaN: nothing outside a view is read into a result."""
    k, n = 200, 136
    c = _case(5, 1, rows, k, n, gate="shared")

    def inside(t, left, right):
        buf = torch.full((*t.shape[:-1], t.shape[-1] + left + right), float("nan"), device=DEV, dtype=t.dtype)
        view = buf[..., left:left + t.shape[-1]]
        view.copy_(t)
        return view

    for left, right in ((8, 16), (3, 2)):  # aligned and unaligned rows
        v = {key: inside(t, left, right) if key in ("x", "weight", "residual") else t for key, t in c.items()}
        out = torch.full((1, rows, n + 16), 7.0, device=DEV, dtype=torch.bfloat16)
        linear_act(**v, activation="gelu_tanh", out=out[..., 8:8 + n])
        _check(out[..., 8:8 + n], *_forward64(c, "gelu_tanh"), U[torch.bfloat16])
        assert (out[..., :8] == 7).all() and (out[..., 8 + n:] == 7).all()
    # transposed weight, and a batch of rows that no single stride walks
    w = c["weight"].t().contiguous().t()
    _check(linear_act(**dict(c, weight=w)), *_forward64(c, None), U[torch.bfloat16])
    wide = torch.randn(2, rows + 3, k, device=DEV).to(torch.bfloat16)
    d = dict(_case(6, 2, rows, k, n), x=wide[:, :rows])
    _check(linear_act(**d), *_forward64(d, None), U[torch.bfloat16])


def test_in_place_residual_and_flat_shapes():
    c = _case(9, 1, 300, 128, 256)
    ref = linear_act(**c, activation="gelu")
    r = c["residual"].clone()
    assert linear_act(**dict(c, residual=r), activation="gelu", out=r) is r
    assert torch.equal(r, ref)
    x2d = dict(x=c["x"][0], weight=c["weight"], bias=c["bias"], gate=c["gate"].reshape(1, -1), residual=c["residual"][0])
    assert torch.equal(linear_act(**x2d, activation="gelu"), ref[0])
    one = linear_act(c["x"][0, 0], c["weight"])
    assert one.shape == (256,)
    assert linear_act(c["x"][:, :0], c["weight"]).shape == (1, 0, 256)


def test_special_values_stay_in_their_rows_and_columns():
    for rows in (40, 1000):
        c = _case(11, 1, rows, 192, 264, gate="shared")
        clean = linear_act(**c, activation="silu")
        c["x"][0, 7] = float("nan")
        c["x"][0, rows - 1, 3] = float("inf")
        c["weight"][100] = float("nan")
        got = linear_act(**c, activation="silu")
        keep = torch.ones(rows, 264, dtype=torch.bool, device=DEV)
        keep[7], keep[rows - 1], keep[:, 100] = False, False, False
        assert torch.equal(got[0][keep], clean[0][keep])
        assert got[0, 7].isnan().all() and got[0, :, 100].isnan().all()
    # large pre-activations: the activations saturate instead of overflowing
    x = torch.tensor([[200.0, -200.0, 60000.0, -60000.0]], device=DEV, dtype=torch.float16).t().contiguous()
    w = torch.ones(1, 1, device=DEV, dtype=torch.float16)
    for act in ("gelu_tanh", "gelu", "silu"):
        assert torch.equal(linear_act(x, w, activation=act)[:, 0], torch.relu(x[:, 0]))


def test_other_stream():
    c = _case(13, 1, 500, 512, 512)
    ref = linear_act(**c, activation="gelu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear_act(**c, activation="gelu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)


# ---- gradient ------------------------------------------------------------------

def _grads64(c, act, grad, preact):
    """Gradients by differentiation in 64 bits at the saved pre-activation, and their slack."""
    d = {k: None if v is None else v.double() for k, v in c.items()}
    x = d["x"] if d["x2"] is None else torch.cat((d["x"], d["x2"]), -1)
    z = preact.double().reshape(grad.shape).requires_grad_()
    gate = None if d["gate"] is None else d["gate"].requires_grad_()
    y = _act64(z, act) * (1 if gate is None else _gate64(gate))
    dz, dgate = torch.autograd.grad(y, (z, gate), grad.double()) if gate is not None else \
        (torch.autograd.grad(y, z, grad.double())[0], None)
    k, rows = c["x"].shape[-1], x.flatten(0, 1)
    dzf = dz.flatten(0, 1)
    dx, dw = dz @ d["weight"], dzf.t() @ rows
    sx, sw = dz.abs() @ d["weight"].abs(), dzf.abs().t() @ rows.abs()
    out = {"x": (dx[..., :k], sx[..., :k]), "weight": (dw, sw), "bias": (dzf.sum(0), dzf.abs().sum(0))}
    if d["x2"] is not None:
        out["x2"] = (dx[..., k:], sx[..., k:])
    if gate is not None:
        size = (grad.double() * _act64(z, act)).abs()
        out["gate"] = (dgate, size.sum(1).reshape(dgate.shape) if gate.dim() == 3 or gate.dim() == 2 else size.sum((0, 1)))
    return out


def _check_grads(got, ref, u, rows, n):
    for name, (value, size) in ref.items():
        g = getattr(got, name)
        assert g.shape == value.shape, name
        fresh = 0.0 if name in ("bias", "gate") else u  # dz is rounded for the products only
        _check(g, value, (fresh + (rows + n) * 2.0 ** -24 + 2.0 ** -17) * size, u)
        if value.norm() > 0:
            assert ((g.double() - value).norm() <= u * value.norm() + 2.0 ** -24 * value.numel() ** 0.5).item(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape,k2", [((1, 1, 64, 8), 0), ((1, 1, 33, 7), 5), ((2, 65, 200, 130), 0),
                                      ((3, 33, 101, 77), 0), ((1, 300, 136, 264), 72), ((1, 129, 64, 128), 0),
                                      ((4, 256, 520, 392), 0), ((1, 2100, 72, 1032), 0), ((2, 3, 2000, 24), 0)])
def test_backward(shape, k2, dtype):
    for i, act in enumerate((None, "gelu_tanh", "gelu", "silu")):
        c = _case(i, *shape, k2=k2, dtype=dtype, gate=("sample", None, "shared", "sample")[i], residual=False)
        g = torch.Generator(device=DEV).manual_seed(77 + i)
        grad = torch.randn((*shape[:2], shape[3]), generator=g, device=DEV).to(dtype)
        preact = torch.randn(grad.shape, generator=g, device=DEV).to(dtype)
        got = linear_act_backward(grad, c["x"], c["weight"], preact=preact, activation=act, gate=c["gate"], x2=c["x2"],
                                  bias=True)
        _check_grads(got, _grads64(c, act, grad, preact), U[dtype], shape[0] * shape[1], shape[3])
        again = linear_act_backward(grad, c["x"], c["weight"], preact=preact, activation=act, gate=c["gate"],
                                    x2=c["x2"], bias=True)
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))  # a fixed order of sums
    assert _native.device_status(clear=True) == 0


def test_backward_plain_layer_reads_the_gradient_in_place():
    """No activation and no gate: no pre-activation is needed, and an expanded gradient is taken too."""
    c = _case(3, 2, 50, 96, 88, gate=None, residual=False)
    for grad in (torch.randn(2, 50, 88, device=DEV).to(torch.bfloat16),
                 torch.ones((), device=DEV, dtype=torch.bfloat16).expand(2, 50, 88),
                 torch.randn(2, 50, 91, device=DEV).to(torch.bfloat16)[..., 1:89]):
        got = linear_act_backward(grad, c["x"], c["weight"], bias=True)
        _check_grads(got, _grads64(c, None, grad, torch.zeros_like(grad)), U[torch.bfloat16], 100, 88)
    only = linear_act_backward(grad, c["x"], c["weight"], bias=True, needs=("bias",))
    assert only.x is None and only.weight is None and torch.equal(only.bias, got.bias)
    empty = linear_act_backward(grad[:, :0], c["x"][:, :0], c["weight"], bias=True)
    assert empty.x.shape == (2, 0, 96) and not empty.weight.any() and not empty.bias.any()


def test_autograd_against_differences():
    """loss = <grad, out>: each gradient against central differences of the 64-bit definition along a random
    direction.  The forward saves a rounded pre-activation: one more rounding of size u |z act''| <= u |z|."""
    act, dtype = "gelu_tanh", torch.float16
    c = _case(21, 2, 40, 72, 56, k2=24, dtype=dtype)
    leaves = {k: v.clone().requires_grad_() for k, v in c.items()}
    grad = torch.randn(2, 40, 56, device=DEV).to(dtype)
    out = linear_act(**leaves, activation=act)
    assert torch.equal(out, linear_act(**c, activation=act))
    got = dict(zip(leaves, torch.autograd.grad(out, list(leaves.values()), grad)))
    assert torch.equal(got["residual"], grad)
    g = torch.Generator(device=DEV).manual_seed(4)
    for name, value in c.items():
        v = torch.randn(value.shape, generator=g, device=DEV, dtype=torch.float64)
        h = 1e-5

        def loss(sign):
            d = {k: t.double() for k, t in c.items()}
            d[name] = d[name] + sign * h * v
            return (_forward64(d, act)[0] * grad.double()).sum()

        diff = ((loss(1) - loss(-1)) / (2 * h)).item()
        # roundings of the gradient's elements (its own, dz's and the pre-activation's: 4u of an element's size in
        # all) are independent: their sum along v stays within 6 standard deviations of the 2-norm, which for dz's
        # part is taken at the size of the gradient itself
        bound = 6 * 4 * U[dtype] * (got[name].double() * v).norm().item() + 1e-6 * abs(diff)
        assert abs((got[name].double() * v).sum().item() - diff) <= bound, name


def test_refusals():
    c = _case(1, 2, 8, 16, 24)
    x, w = c["x"], c["weight"]
    with pytest.raises(ValueError):
        linear_act(x, w, activation="relu6")
    with pytest.raises(ValueError):
        linear_act(x, w[:, :8])
    with pytest.raises(ValueError):
        linear_act(x, w, bias=c["bias"][:-1])
    with pytest.raises(ValueError):
        linear_act(x, w, gate=c["gate"][:, 0, :][:1])  # one row for two samples
    with pytest.raises(ValueError):
        linear_act(x, w, residual=c["residual"][:1])
    with pytest.raises(ValueError):
        linear_act(x, w, x2=x[:1])
    with pytest.raises(ValueError):
        linear_act(x, w, out=torch.empty(2, 8, 23, device=DEV, dtype=x.dtype))
    with pytest.raises(ValueError):
        linear_act(x, w, out=torch.empty(2, 24, 8, device=DEV, dtype=x.dtype).transpose(1, 2))
    with pytest.raises(TypeError):
        linear_act(x.float(), w.float())
    with pytest.raises(TypeError):
        linear_act(x, w.half())
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_act(x.cpu(), w.cpu())
    with pytest.raises(RuntimeError):
        linear_act(x.clone().requires_grad_(), w, out=torch.empty(2, 8, 24, device=DEV, dtype=x.dtype))
    with pytest.raises(ValueError, match="preact"):
        linear_act_backward(c["residual"], x, w, activation="silu")
    with pytest.raises(ValueError):
        linear_act_backward(c["residual"], x, w, needs=("gate",))
    lib, p, z = _native.load(), _native.ptr(x), _native.P(0)
    s = _native.stream_of(x.device, x)
    launches = lib.peco_launch_count()
    # unsupported type, unknown activation, row stride below a row, missing second input, workspace too small
    assert lib.peco_linear_forward(p, 16, z, 0, p, 16, z, z, 0, z, 0, p, 8, z, 1, 2, 16, 0, 8, 0, 2, z, 0, s) == 20001
    assert lib.peco_linear_forward(p, 16, z, 0, p, 16, z, z, 0, z, 0, p, 8, z, 1, 2, 16, 0, 8, 9, 1, z, 0, s) == 1
    assert lib.peco_linear_forward(p, 8, z, 0, p, 16, z, z, 0, z, 0, p, 8, z, 1, 2, 16, 0, 8, 0, 1, z, 0, s) == 1
    assert lib.peco_linear_forward(p, 16, z, 0, p, 16, z, z, 0, z, 0, p, 8, z, 1, 2, 8, 8, 8, 0, 1, z, 0, s) == 1
    assert lib.peco_linear_forward(p, 15, z, 0, p, 16, z, z, 0, z, 0, p, 8, z, 1, 2, 15, 0, 8, 0, 1, z, 0, s) == 20005
    assert lib.peco_launch_count() == launches


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 256, 1536, 12288), (1, 200, 1000, 6000), (2, 80, 3000, 999), (1, 256, 4096, 2688),
                                   (1, 129, 2048, 5000), (3, 170, 2048, 2050), (1, 100, 2048, 9000), (1, 7, 4096, 700),
                                   (1, 256, 8192, 2048)])
def test_few_rows_over_long_sums(shape, dtype):
    # the sum over K is shared out among CTAs, on tiles of one and of two accumulators
    for i, act in enumerate(("gelu_tanh", None)):
        c = _case(7 + i, *shape, dtype=dtype, gate="sample" if i else "shared", residual=i == 0)
        _check(linear_act(**c, activation=act), *_forward64(c, act), U[dtype])
    assert _native.device_status(clear=True) == 0
