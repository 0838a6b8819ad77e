"""modulated_norm and rotate, with their gradients, on the GPU against the definitions in 64 bits.

Tolerances.  u is the unit roundoff of the output type (2^-8 bf16, 2^-11 fp16,
2^-24 fp32).  norm: r and h are fp32 chains of a few operations on values of
known size, rounded once: u |value| plus 2^-18 of the sizes of the terms that
are added (fp32 sums of up to 16384 terms taken as trees of short runs: about
2^-20, and the square root).  A row without variance has rstd = 1/sqrt(eps) =
1000, which multiplies the fp32 error of r - mean: eps = 1 is used where a
width of 1 or a constant row makes that the whole value.  rotary: two fp32
products and a sum (3 * 2^-24 of |a| + |b|), sine and cosine to 2^-22, one
rounding.
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.hunyuan import rope_3d, rotate_pairs
from peco_b200.norms import modulated_norm, modulated_norm_backward
from peco_b200.rotary import rotate

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _near(got, ref, size, u, fine=2.0 ** -18):
    err = (got.double() - ref).abs()
    bound = u * ref.abs() + fine * size + 2.0 ** -24
    assert (err <= bound).all(), (err - bound).max().item()


# ---- norm ------------------------------------------------------------------------

def _inputs(seed, b, t, c, dtype=torch.bfloat16, branch=True, gate="sample", modulate="sample", weight=True, post="rms"):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dtype)

    def vec(kind):
        return {"sample": lambda: normal(b, 3 * c, std=0.5)[:, c:2 * c], "shared": lambda: normal(c, std=0.5),
                None: lambda: None}[kind]()

    return dict(x=normal(b, t, c, std=2.0, mean=0.5), branch=normal(b, t, c) if branch else None,
                gate=vec(gate if branch else None), scale=vec(modulate), shift=vec(modulate),
                weight=normal(c, std=0.1, mean=1.0) if weight else None,
                post_weight=normal(c, std=0.1, mean=1.0) if branch and post else None)


def _row(v):
    return None if v is None else v[:, None] if v.dim() == 2 else v


def _norm64(x, kind, eps):
    m = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    rstd = ((x - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    return (x - m) * rstd, rstd


def _forward64(c, norm, post, eps, rs):
    d = {k: None if v is None else v.double() if v.dtype != torch.float64 else v for k, v in c.items()}
    r, size = rs * d["x"], (rs * d["x"]).abs()
    if d["branch"] is not None:
        y = d["branch"] if post is None else _norm64(d["branch"], post, eps)[0]
        if d["post_weight"] is not None:
            y = y * d["post_weight"]
        if d["gate"] is not None:
            y = y * _row(d["gate"])
        r, size = r + y, size + y.abs()
    n, rstd = _norm64(r, norm, eps)
    h, hsize = n, size.amax(-1, keepdim=True) * rstd + n.abs()
    for v in (d["weight"], None if d["scale"] is None else 1 + _row(d["scale"])):
        if v is not None:
            h, hsize = h * v, hsize * v.abs()
    if d["shift"] is not None:
        h, hsize = h + _row(d["shift"]), hsize + _row(d["shift"]).abs()
    return r, size, h, hsize


WIDTHS = [1, 2, 7, 8, 64, 100, 512, 520, 1000, 1001, 1024, 1032, 2048, 2056, 3072, 3080, 5001, 6144, 6152, 16384, 16383]


@pytest.mark.parametrize("width", WIDTHS)
def test_norm_forward(width):
    eps = 1.0 if width < 4 else 1e-6
    for i, (norm, post, dtype) in enumerate([("layer", None, torch.bfloat16), ("rms", "rms", torch.float16),
                                             ("layer", "layer", torch.bfloat16), ("rms", None, torch.bfloat16)]):
        for b, t in ((1, 1), (3, 37)):
            c = _inputs(i, b, t, width, dtype, gate=("sample", "shared", None, "sample")[i],
                        modulate=("sample", "shared", "sample", None)[i], weight=i != 0, post=post if i == 1 else None)
            rs = (1.0, 0.5, 1.0, -2.0)[i]
            r, h = modulated_norm(**c, norm=norm, post_norm=post, eps=eps, residual_scale=rs)
            r64, rsize, h64, hsize = _forward64(c, norm, post, eps, rs)
            _near(r, r64, rsize, U[dtype])
            _near(h, h64, hsize, U[dtype])
            alone = dict(c, branch=None, gate=None, post_weight=None)
            h = modulated_norm(**alone, norm=norm, eps=eps)
            _near(h, *_forward64(alone, norm, None, eps, 1.0)[2:], U[dtype])


def test_norm_strides_shapes_and_special_rows():
    c = _inputs(3, 2, 20, 256)
    r, h = modulated_norm(**c, post_norm="rms")
    wide = torch.full((2, 25, 300), float("nan"), device=DEV, dtype=torch.bfloat16)
    for left in (8, 3):  # aligned and unaligned views whose surroundings are NaN
        wide[:, 2:22, left:left + 256] = c["x"]
        view = wide[:, 2:22, left:left + 256]
        r2, h2 = modulated_norm(**dict(c, x=view), post_norm="rms")
        # the unaligned form sums a row in another order: one rounding step at most
        assert (r2.float() - r.float()).abs().max() <= 2.0 ** -7 * r.float().abs().max()
        _near(h2, *_forward64(c, "layer", "rms", 1e-6, 1.0)[2:], U[torch.bfloat16])
        wide.fill_(float("nan"))
    flat = modulated_norm(c["x"][0], scale=c["scale"][:1], shift=c["shift"][:1])
    assert torch.equal(flat, modulated_norm(c["x"][:1], scale=c["scale"][:1], shift=c["shift"][:1])[0])
    v = modulated_norm(c["x"][0, 0])
    assert v.shape == (256,) and torch.equal(v, modulated_norm(c["x"])[0, 0])
    assert modulated_norm(c["x"][:, :0]).shape == (2, 0, 256)
    four = modulated_norm(c["x"].reshape(2, 4, 5, 256), scale=c["scale"], shift=c["shift"])
    assert torch.equal(four.reshape(2, 20, 256), modulated_norm(c["x"], scale=c["scale"], shift=c["shift"]))
    x = c["x"].clone()
    x[0, 3], x[1, 5, 9], x[0, 0] = 4.0, float("inf"), float("nan")
    clean, got = modulated_norm(c["x"]), modulated_norm(x)
    assert not got[0, 3].any()  # a constant row has no deviation
    assert got[1, 5].isnan().any() and got[0, 0].isnan().all()
    keep = torch.ones(2, 20, dtype=torch.bool, device=DEV)
    keep[0, 3] = keep[1, 5] = keep[0, 0] = False
    assert torch.equal(got[keep], clean[keep])
    # a mean far above the deviation: the variance is taken around the mean
    far = (1024.0 + torch.randn(1, 64, 512, device=DEV)).half()
    n64, _ = _norm64(far.double(), "layer", 1e-6)
    _near(modulated_norm(far), n64, 2.0 ** 6 * n64.abs().clamp_min(1.0), U[torch.float16])


def _norm_grads64(c, gh, gr, norm, post, eps, rs):
    leaves = {k: v.double().requires_grad_() for k, v in c.items() if v is not None}
    r, _, h, _ = _forward64({**dict.fromkeys(c), **leaves}, norm, post, eps, rs)
    outs, grads = ([h, r], [gh.double(), gr.double()]) if gr is not None else ([h], [gh.double()])
    return dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads)))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [(1, 1), (3, 37), (2, 400)])
def test_norm_backward(width, rows):
    """Row gradients: u |value| plus 2^-16 of the largest term of the row (a difference of fp32 means).  Vector
    gradients: u |value| plus 2^-16 of the sum of the absolute terms, bounded by sqrt(rows * width) norms."""
    eps = 1.0 if width < 4 else 1e-6
    for i, (norm, post, dtype) in enumerate([("layer", None, torch.bfloat16), ("rms", "rms", torch.float16),
                                             ("layer", "layer", torch.bfloat16)]):
        c = _inputs(i, *rows, width, dtype, gate=("sample", "shared", None)[i], modulate=("sample", "shared", "sample")[i],
                    weight=i != 0, post=post if i == 1 else None)
        g = torch.Generator(device=DEV).manual_seed(50 + i)
        gh, gr = (torch.randn(c["x"].shape, generator=g, device=DEV).to(dtype) for _ in range(2))
        opts = dict(norm=norm, post_norm=post, eps=eps, residual_scale=0.5)
        got = modulated_norm_backward(gh, gr, **c, **opts)
        ref = _norm_grads64(c, gh, gr, norm, post, eps, 0.5)
        for name, value in c.items():
            mine = getattr(got, name)
            if value is None:
                assert mine is None
                continue
            assert mine.shape == value.shape and mine.dtype == dtype
            v = ref[name]
            if name in ("x", "branch"):
                _near(mine, v, v.abs().amax(-1, keepdim=True) + 1.0, U[dtype], 2.0 ** -16)
            else:
                _near(mine, v, 10.0 * rows[0] * rows[1], U[dtype], 2.0 ** -16)
            if v.norm() > 1e-3:
                assert (mine.double() - v).norm() <= U[dtype] * v.norm(), name
        again = modulated_norm_backward(gh, gr, **c, **opts)
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))
        part = modulated_norm_backward(gh, None, **c, **opts, needs=("x",))
        v = _norm_grads64(c, gh, None, norm, post, eps, 0.5)["x"]
        _near(part.x, v, v.abs().amax(-1, keepdim=True) + 1.0, U[dtype], 2.0 ** -16)
        assert all(t is None for t in part[1:])


def test_norm_autograd_against_differences():
    """Central differences of the 64-bit definition along random directions; the only roundings are of the gradient's
    elements (u each, independent: 6 standard deviations of their sum)."""
    dtype = torch.float16
    c = _inputs(5, 2, 30, 200, dtype)
    opts = dict(norm="layer", post_norm="rms", eps=1e-5, residual_scale=0.7)
    leaves = {k: v.clone().requires_grad_() for k, v in c.items()}
    gr, gh = (torch.randn(c["x"].shape, device=DEV).to(dtype) for _ in range(2))
    r, h = modulated_norm(**leaves, **opts)
    got = dict(zip(leaves, torch.autograd.grad([r, h], list(leaves.values()), [gr, gh])))
    g = torch.Generator(device=DEV).manual_seed(2)
    for name, value in c.items():
        v = torch.randn(value.shape, generator=g, device=DEV, dtype=torch.float64)

        def loss(step):
            d = {k: t.double() for k, t in c.items()}
            d[name] = d[name] + step * v
            r64, _, h64, _ = _forward64(d, "layer", "rms", 1e-5, 0.7)
            return ((r64 * gr.double()).sum() + (h64 * gh.double()).sum()).item()

        diff = (loss(1e-5) - loss(-1e-5)) / 2e-5
        mine = got[name].double() * v
        assert abs(mine.sum().item() - diff) <= 6 * U[dtype] * mine.norm().item() + 1e-6 * (abs(diff) + 1), name
    # only one output used, and none of the vectors
    x = c["x"].clone().requires_grad_()
    r, h = modulated_norm(x, c["branch"], gate=c["gate"], norm="rms")
    (gx,) = torch.autograd.grad(r, x, gr)
    assert torch.equal(gx, gr)


def test_norm_refusals():
    c = _inputs(1, 2, 8, 16)
    x = c["x"]
    for bad in (dict(norm="batch"), dict(post_norm="batch"), dict(gate=c["gate"]), dict(post_norm="rms"),
                dict(scale=c["scale"][:, :8]), dict(scale=c["scale"][:1]), dict(weight=c["weight"][:3]),
                dict(branch=x[:1]), dict(branch=c["branch"], post_weight=c["post_weight"]), dict(eps=-1.0),
                dict(residual_scale=float("nan"))):
        with pytest.raises(ValueError):
            modulated_norm(x, **bad)
    with pytest.raises(ValueError):
        modulated_norm(torch.zeros(1, 2, 16385, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        modulated_norm(x.float())
    with pytest.raises(TypeError):
        modulated_norm(x, scale=c["scale"].float())
    with pytest.raises(RuntimeError, match="CUDA"):
        modulated_norm(x.cpu())
    with pytest.raises(ValueError):
        modulated_norm_backward(x, x, x)  # a gradient of r without a branch
    with pytest.raises(ValueError):
        modulated_norm_backward(x, None, x, needs=("gate",))


# ---- rotary ------------------------------------------------------------------------

def _rotate64(x, pos, axes, theta, interleaved, inverse):
    """x [B, H, N, D], pos [B or 1, N', A]: (value, size of its terms)."""
    ang = torch.cat([pos[..., a:a + 1].double() * theta ** (-torch.arange(0, d, 2, device=DEV).double() / max(d, 1))
                     for a, d in enumerate(axes)], -1)[:, None]
    if inverse:
        ang = -ang
    n, p = ang.shape[2], ang.shape[3]
    out = x.double().clone()
    size = torch.zeros_like(out)
    rows = x.double()[:, :, :n, :2 * p]
    a, b = (rows[..., 0::2], rows[..., 1::2]) if interleaved else (rows[..., :p], rows[..., p:])
    new = torch.stack((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()), -1)
    terms = (a.abs() + b.abs())[..., None].expand(new.shape)
    if interleaved:
        out[:, :, :n, :2 * p], size[:, :, :n, :2 * p] = new.flatten(-2), terms.flatten(-2)
    else:
        out[:, :, :n, :2 * p] = new.transpose(-1, -2).flatten(-2)
        size[:, :, :n, :2 * p] = terms.transpose(-1, -2).flatten(-2)
    return out, size


def _grid_pos(grid):
    return torch.cartesian_prod(*(torch.arange(s, device=DEV) for s in grid)).reshape(1, -1, len(grid))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,axes", [(128, (16, 56, 56)), (64, (16, 24, 24)), (40, (8, 12, 12)), (128, (44, 42, 42)),
                                    (96, (22, 22, 20)), (256, (64, 64, 64, 64)), (6, (2,)), (80, (10, 0, 62)), (2, (2,)),
                                    (64, (32,))])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary(d, axes, dtype, interleaved):
    grid = {1: (37,), 3: (3, 5, 9), 4: (2, 3, 2, 7)}[len(axes)]
    n = torch.Size(grid).numel()
    g = torch.Generator(device=DEV).manual_seed(d)
    for b, heads, kv, text, inverse in ((1, 1, 1, 0, False), (2, 6, 2, 11, True), (1, 5, 0, 3, False)):
        def rand(h, token_major):
            if token_major:
                return torch.randn((b, n + text, h, d), generator=g, device=DEV).to(dtype).transpose(1, 2)
            return torch.randn((b, h, n + text, d), generator=g, device=DEV).to(dtype)

        for token_major in (False, True):
            q, k = rand(heads, token_major), rand(kv, token_major) if kv else None
            opts = dict(axes=axes, theta=100.0, interleaved=interleaved, inverse=inverse)
            got = rotate(q, k, **opts, grid=grid)
            got = got if k is not None else (got,)
            pos = torch.randint(-50, 5000, (b, n, len(axes)), generator=g, device=DEV)
            for x, y in zip((q, k), got):
                assert y.stride() == x.stride()  # the layout is kept
                v, size = _rotate64(x, _grid_pos(grid), axes, 100.0, interleaved, inverse)
                _near(y, v, size, U[dtype], 2.0 ** -21)
            for positions in (pos, pos[0], pos.int(), pos.float() + 0.25):
                y = rotate(q, k, **opts, positions=positions)
                p3 = positions if positions.dim() == 3 else positions[None]
                _near(y[0] if k is not None else y, *_rotate64(q, p3, axes, 100.0, interleaved, inverse), U[dtype], 2.0 ** -21)
            q2, k2 = q.clone(memory_format=torch.preserve_format), None if k is None else k.clone()
            back = rotate(q2, k2, **opts, grid=grid, inplace=True)
            assert (back[0] if k is not None else back) is q2 and torch.equal(q2, got[0])
            if k is not None:
                assert torch.equal(k2, got[1])


def test_rotary_far_positions_and_views():
    q = torch.randn(1, 2, 9, 128, device=DEV)
    pos = torch.full((9, 3), 2 ** 24 + 12345, device=DEV, dtype=torch.int64)
    _near(rotate(q, axes=(16, 56, 56), positions=pos), *_rotate64(q, pos[None], (16, 56, 56), 256.0, True, False),
          U[torch.float32], 2.0 ** -21)
    wide = torch.full((1, 2, 12, 140), float("nan"), device=DEV, dtype=torch.bfloat16)
    for left in (8, 5):
        view = wide[:, :, 1:10, left:left + 128]
        view.copy_(q)
        v, size = _rotate64(view, pos[None], (16, 56, 56), 256.0, True, False)
        got = rotate(view, axes=(16, 56, 56), positions=pos)
        _near(got, v, size, U[torch.bfloat16], 2.0 ** -21)
        rotate(view, axes=(16, 56, 56), positions=pos, inplace=True)
        assert torch.equal(view, got)
        wide.fill_(float("nan"))
    assert torch.equal(rotate(q, axes=(16, 56, 56), positions=pos[:0]), q)
    assert rotate(q[:, :, :0], axes=(16,), grid=(0,)).shape == (1, 2, 0, 128)


def test_rotary_agrees_with_the_model_tables():
    grid, axes = (3, 6, 10), (16, 56, 56)
    x = torch.randn(1, 4, 180, 128, device=DEV)
    cos, sin = rope_3d(grid, axes, 256.0, DEV)
    # the tables hold fp32 angles: up to 10 * 2^-24 off
    assert (rotate(x, axes=axes, grid=grid) - rotate_pairs(x, cos, sin)).abs().max() <= 2.0 ** -19 * x.abs().max() * 2


def test_rotary_gradient_is_the_inverse():
    q = torch.randn(2, 3, 60, 64, device=DEV, dtype=torch.float32, requires_grad=True)
    k = torch.randn(2, 1, 60, 64, device=DEV, dtype=torch.float32, requires_grad=True)
    opts = dict(axes=(16, 24, 24), grid=(3, 4, 5), interleaved=False)
    a, b = rotate(q, k, **opts)
    ga, gb = torch.randn_like(a), torch.randn_like(b)
    gq, gk = torch.autograd.grad([a, b], [q, k], [ga, gb])
    back = rotate(ga, gb, **opts, inverse=True)
    assert torch.equal(gq, back[0]) and torch.equal(gk, back[1])
    # differences along a random direction: the operator is linear, so any step is exact but for fp32 rounding
    v = torch.randn_like(q)
    with torch.no_grad():
        diff = ((rotate(q + v, **opts) - rotate(q - v, **opts)).double() * ga.double()).sum() / 2
    mine = (gq.double() * v.double()).sum()
    assert abs(mine - diff) <= 6 * 8 * 2.0 ** -24 * (ga.double().norm() * (q.double().norm() + v.double().norm()))
    (only,) = torch.autograd.grad(rotate(q.detach(), k, **opts)[1], k, gb)
    assert torch.equal(only, gk)


def test_rotary_refusals():
    q = torch.randn(2, 3, 12, 64, device=DEV).to(torch.bfloat16)
    pos = torch.zeros(2, 12, 3, device=DEV, dtype=torch.int32)
    ok = dict(axes=(16, 24, 24), positions=pos)
    for bad in (dict(ok, axes=(16, 24, 26)), dict(ok, axes=(15, 25, 24)), dict(ok, axes=(16, 48)), dict(ok, grid=(1, 2, 3)),
                dict(axes=(16, 24, 24)), dict(axes=(64,), grid=(13,)), dict(axes=(64,), grid=(3, 4)), dict(ok, theta=0.0),
                dict(ok, positions=pos[:, :, :2]), dict(ok, positions=pos[:, :1].expand(2, 13, 3)),
                dict(ok, positions=pos[:1].expand(3, 12, 3)), dict(ok, k=q[:1]), dict(ok, k=q[:, :, :5])):
        with pytest.raises(ValueError):
            rotate(q, **bad)
    with pytest.raises(ValueError):
        rotate(q[..., :63], **ok)
    with pytest.raises(ValueError):
        rotate(q[:, :1].expand(2, 3, 12, 64), **ok, inplace=True)
    with pytest.raises(TypeError):
        rotate(q.double(), **ok)
    with pytest.raises(TypeError):
        rotate(q, q.half(), **ok)
    with pytest.raises(TypeError):
        rotate(q, axes=(16, 24, 24), positions=pos.to(torch.int16))
    with pytest.raises(RuntimeError, match="CUDA"):
        rotate(q.cpu(), axes=(64,), grid=(12,))
    with pytest.raises(RuntimeError):
        rotate(q.clone().requires_grad_(), **ok, inplace=True)


def test_second_epsilon_and_shared_operand_are_refused():
    x = torch.randn(1, 4, 16, device=DEV).to(torch.bfloat16)
    with pytest.raises(ValueError):
        modulated_norm(x, x, post_norm="rms", post_eps=-1.0)
    with pytest.raises(ValueError):
        modulated_norm_backward(x, None, x, x, post_norm="rms", post_eps=float("nan"))
    q = torch.randn(1, 2, 4, 16, device=DEV).to(torch.bfloat16)
    with pytest.raises(ValueError):
        rotate(q, q, axes=(16,), grid=(4,), inplace=True)
