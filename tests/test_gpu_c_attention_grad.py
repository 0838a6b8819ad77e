"""attention's gradients on the GPU against the formula in 64 bits, and against differences.

Tolerances, element by element, with u the unit roundoff of the type (2^-8 bf16,
2^-11 fp16) and e = 2^-20 (1 + the magnitudes a score is made of):
probabilities p are rounded to 16 bits (u, with their error 2 e), so
  |dv| error <= u |dv| + (u + 2 e + N 2^-24) sum p |g|;
ds = p (g.v - delta) s', where delta = g.out takes the 16-bit out (off by its
rounding u |out| and its probabilities' (u + 2 e) sum p |v|), is off by (2 e +
2^-20) p (|g.v| + |delta|) s' (g.v of D products in fp32), plus p times delta's
error, and is rounded (u |ds|): summed over the products with |k| or |q|, and u
of the result.  In fp16 a ds below 2^-14 rounds by up to 2^-25
absolutely (p, held 2^10 times larger, by 2^-35).
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.attention import attention, attention_backward
from span_reference import attend, score_size
from test_gpu_b_attention import DEV, MASKS, SIZES, U, inputs, plan

pytestmark = pytest.mark.gpu


def formula(q, k, v, g, out, seen, pos, scale=None, softcap=None, slopes=None):
    """Gradients in 64 bits and the bounds of their errors; q, k, v, g, out in 16 bits."""
    u, group = U[q.dtype], q.shape[1] // k.shape[1]
    tiny = 2.0 ** -25 if q.dtype is torch.float16 else 0.0
    args = dict(scale=scale, softcap=softcap, slopes=slopes)
    q, k, v, g = (t.double() for t in (q, k, v, g))
    kg, vg = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    exact, _, p = attend(q, k, v, seen, pos, **args)
    e = 2.0 ** -20 * (1 + score_size(q, k, seen, pos, **args))
    factor = q.shape[-1] ** -0.5 if scale is None else scale
    slope = torch.ones_like(p)
    if softcap is not None:
        slope = 1 - torch.tanh(q @ kg.transpose(-1, -2) * factor / softcap) ** 2
    gv = g @ vg.transpose(-1, -2)
    delta = (g * exact).sum(-1, keepdim=True)
    ds = p * (gv - delta) * slope
    # out's own error: its rounding and its probabilities'
    loose = (g.abs() * (u * exact.abs() + (u + 2 * e) * (p @ vg.abs()))).sum(-1, keepdim=True)
    off = p * ((2 * e + 2.0 ** -20) * (g.abs() @ vg.abs().transpose(-1, -2) + delta.abs()) + loose) * slope \
        + u * ds.abs() + tiny * (p > 0)
    if softcap is not None:  # the slope's own error: a few 2^-23
        off = off + 2.0 ** -20 * p * (gv - delta).abs()

    def shared(t):  # sum over the query heads of a key head
        return t.unflatten(1, (k.shape[1], group)).sum(2)

    n, m = q.shape[2], k.shape[2]
    result = {"q": (factor * ds @ kg, factor * (off + m * 2.0 ** -24 * ds.abs()) @ kg.abs()),
              "k": (shared(factor * ds.transpose(-1, -2) @ q),
                    shared(factor * (off + n * group * 2.0 ** -24 * ds.abs()).transpose(-1, -2) @ q.abs())),
              "v": (shared(p.transpose(-1, -2) @ g),
                    shared(((u + 2 * e + n * group * 2.0 ** -24) * p + tiny * 2.0 ** -10 * (p > 0)).transpose(-1, -2) @ g.abs()))}
    return {name: (ref, slack + u * ref.abs() + 2.0 ** -25) for name, (ref, slack) in result.items()}


def check(got, expected):
    for name, t in zip("qkv", got):
        ref, slack = expected[name]
        assert torch.isfinite(t).all(), name
        over = (t.double() - ref).abs() - slack
        assert (over <= 0).all(), (name, over.max().item())
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_every_key(size, dtype):
    b, h, kv, n, m, d = size
    q, k, v = inputs(n + m, *size, dtype=dtype, token_major=n % 2 == 1)
    g = inputs(1, *size, dtype=dtype)[0]
    seen = torch.ones(b, n, m, dtype=torch.bool, device=DEV)
    pos = (torch.arange(n, device=DEV) + m - n).expand(b, n)
    slopes = torch.rand(h, device=DEV) * 0.2
    for args in ({}, dict(softcap=2.0), dict(softcap=30.0, slopes=slopes, scale=0.3)):
        out, lse = attention(q, k, v, return_lse=True, **args)
        got = attention_backward(g, q, k, v, out, lse, **args)
        assert [t.stride() for t in got] == [t.stride() for t in (q, k, v)]
        check(got, formula(q, k, v, g, out, seen, pos, **args))


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("form", [(4, 4, 128), (4, 1, 64), (15, 5, 40)])
def test_masks(mask, form):
    b, n, m, words = mask
    h, kv, d = form
    spans, seen, pos = plan(b, n, m, **words)
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(n, b, h, kv, n, m, d, dtype=dtype)
        g = inputs(n + 1, b, h, kv, n, m, d, dtype=dtype)[0]
        slopes = torch.rand(h, device=DEV) * 0.1
        for args in ({}, dict(softcap=5.0, slopes=slopes)):
            out, lse = attention(q, k, v, spans=spans, return_lse=True, **args)
            got = attention_backward(g, q, k, v, out, lse, spans=spans, **args)
            check(got, formula(q, k, v, g, out, seen, pos, **args))


# heads on shared keys whose sums several CTAs share: unequal shares, one head each, a share for every two; causal over more tiles
@pytest.mark.parametrize("size", [(1, 13, 1, 300, 5100, 24), (2, 10, 2, 259, 130, 128), (1, 12, 2, 390, 4600, 64),
                                  (1, 36, 3, 700, 4000, 16)])
def test_shared_keys_in_parts(size):
    b, h, kv, n, m, d = size
    spans, seen, pos = plan(b, n, m, causal=True) if m == 4000 else (
        None, torch.ones(b, n, m, dtype=torch.bool, device=DEV), (torch.arange(n, device=DEV) + m - n).expand(b, n))
    bits = 1 if spans is not None else 0
    lib = _native.load()
    assert lib.peco_span_attention_backward_workspace(b, h, kv, n, m, d, bits) > 8 * b * h * ((n + 127) // 128 * 128)
    q, k, v = inputs(n, *size, dtype=torch.float16)
    g = inputs(1, *size, dtype=torch.float16)[0]
    out, lse = attention(q, k, v, spans=spans, return_lse=True)
    got = attention_backward(g, q, k, v, out, lse, spans=spans)
    check(got, formula(q, k, v, g, out, seen, pos))
    for name in "kv":
        alone = attention_backward(g, q, k, v, out, lse, spans=spans, needs=[name])
        assert torch.equal(getattr(alone, name), getattr(got, name))
    inner = torch.zeros(b, m, kv, d, device=DEV, dtype=torch.float16).transpose(1, 2)  # another layout of k's gradient
    again = attention_backward(g, q, inner.copy_(k), v, out, lse, spans=spans)
    assert again.k.stride() == inner.stride() and all(torch.equal(x, y) for x, y in zip(again, got))


def test_differences_of_the_loss():
    """The gradient along a direction against the loss's difference quotient in 64 bits (central, step 2^-13: the
    quotient is off by about 2^-26 of third derivatives), to the gradient's rounding."""
    spans, seen, pos = plan(1, 90, 90, documents=[0, 50, 85], causal=True, prefix=10)
    h, kv, d = 4, 2, 64
    q, k, v = inputs(11, 1, h, kv, 90, 90, d)
    g = inputs(12, 1, h, kv, 90, 90, d)[0]
    slopes = torch.rand(h, device=DEV) * 0.1
    args = dict(softcap=4.0, slopes=slopes)
    out, lse = attention(q, k, v, spans=spans, return_lse=True, **args)
    got = attention_backward(g, q, k, v, out, lse, spans=spans, **args)
    expected = formula(q, k, v, g, out, seen, pos, **args)
    step = 2.0 ** -13

    def loss(*qkv):
        return (attend(*qkv, seen, pos, **args)[0] * g.double()).sum()

    for i, name in enumerate("qkv"):
        turn = torch.randn(got[i].shape, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV, dtype=torch.float64)
        ends = []
        for s in (step, -step):
            x = [q.double(), k.double(), v.double()]
            x[i] = x[i] + s * turn
            ends.append(loss(*x))
        quotient = (ends[0] - ends[1]) / (2 * step)
        along = (got[i].double() * turn).sum()
        bound = (expected[name][1] * turn.abs()).sum() + 1e-4 * (expected[name][0] * turn).abs().sum()
        assert (along - quotient).abs() <= bound


def test_autograd():
    spans, seen, pos = plan(2, 150, 150, causal=True, lengths=[150, 60])
    q, k, v = (t.requires_grad_() for t in inputs(13, 2, 4, 2, 150, 150, 64))
    g = inputs(14, 2, 4, 2, 150, 150, 64)[0]
    out, lse = attention(q, k, v, spans=spans, softcap=3.0, return_lse=True)
    assert not lse.requires_grad
    got = torch.autograd.grad(out, (q, k, v), g, retain_graph=True)
    direct = attention_backward(g, q.detach(), k.detach(), v.detach(), out.detach(), lse, spans=spans, softcap=3.0)
    assert all(torch.equal(a, b) for a, b in zip(got, direct))
    (only,) = torch.autograd.grad(out, (k,), g, retain_graph=True)
    assert torch.equal(only, got[1])
    broadcast = torch.autograd.grad(out, (q,), g[:, :, :1].expand_as(g), retain_graph=True)[0]  # a gradient with strides of 0
    assert torch.equal(broadcast, torch.autograd.grad(out, (q,), g[:, :, :1].expand_as(g).contiguous(), retain_graph=True)[0])
    # a shared leaf, and a leaf that wants no gradient
    x = inputs(15, 1, 2, 2, 64, 64, 64)[0].requires_grad_()
    (dx,) = torch.autograd.grad(attention(x, x, x).sum(), (x,))
    parts = [t.detach().requires_grad_() for t in (x, x, x)]
    split = torch.autograd.grad(attention(*parts).sum(), parts)
    assert torch.allclose(dx.double(), sum(t.double() for t in split), rtol=2.0 ** -6, atol=2.0 ** -6 * split[2].abs().max().item())
    frozen = attention(parts[0], parts[1].detach(), parts[2].detach())
    assert torch.equal(torch.autograd.grad(frozen.sum(), (parts[0],))[0], split[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out = attention(q, k, v, spans=spans)
        spans.rows[0, 0, 1] = 0
        out.sum().backward()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_nobody_sees_may_hold_anything(bad):
    for h, kv, n, m, words in ((2, 2, 300, 300, dict(documents=[0, 150, 290])), (4, 2, 300, 300, dict(lengths=[131])),
                               (2, 1, 200, 100, dict(causal=True)), (2, 2, 140, 500, dict(documents=[0, 60, 80], key_documents=[0, 250, 400]))):
        spans, seen, pos = plan(1, n, m, **words)
        q, k, v = inputs(16, 1, h, kv, n, m, 64)
        g = inputs(17, 1, h, kv, n, m, 64)[0]
        out, lse = attention(q, k, v, spans=spans, return_lse=True)
        clean = attention_backward(g, q, k, v, out, lse, spans=spans)
        blind, unseen = ~seen[0].any(1), ~seen[0].any(0)
        assert blind.any() or unseen.any()
        q, k, v, g = (t.clone() for t in (q, k, v, g))
        q[:, :, blind] = g[:, :, blind] = bad
        k[:, :, unseen] = v[:, :, unseen] = bad
        out2, lse2 = attention(q, k, v, spans=spans, return_lse=True)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        for a, c in zip(attention_backward(g, q, k, v, out, lse, spans=spans), clean):
            assert torch.equal(a, c)
        assert (clean.q[:, :, blind] == 0).all() and (clean.k[:, :, unseen] == 0).all() and (clean.v[:, :, unseen] == 0).all()
    assert _native.device_status(clear=True) == 0


def test_no_rows_no_keys_and_layouts():
    q, k, v = inputs(18, 2, 4, 2, 6, 9, 64)
    g = attention_backward(q[:, :, :0], q[:, :, :0], k, v, q[:, :, :0], torch.empty(2, 4, 0, device=DEV))
    assert g.q.shape == (2, 4, 0, 64) and (g.k == 0).all() and (g.v == 0).all()
    none = torch.full((2, 4, 6), -torch.inf, device=DEV)
    g = attention_backward(q, q, k[:, :, :0], v[:, :, :0], torch.zeros_like(q), none)
    assert (g.q == 0).all() and g.k.shape == (2, 2, 0, 64)
    out, lse = attention(q, k, v, return_lse=True)
    ref = attention_backward(q, q, k, v, out, lse)
    odd = torch.zeros(2, 4, 6, 65, device=DEV, dtype=torch.bfloat16)
    odd[..., 1:] = q
    got = attention_backward(odd[..., 1:], odd[..., 1:], k.transpose(-1, -2).contiguous().transpose(-1, -2), v, out, lse)
    assert all(torch.equal(a, c) for a, c in zip(got, ref))
    assert attention_backward(q, q, k, v, out, lse, needs=[]) == (None, None, None)
    some = attention_backward(q, q, k, v, out, lse, needs=iter(["v"]))
    assert some.q is None and some.k is None and torch.equal(some.v, ref.v)


def test_small_probabilities_and_large_gradients_in_fp16():
    """Probabilities near 1 / 20000 and gradients near the type's range."""
    q, k, v = inputs(19, 1, 1, 1, 130, 20000, 64, dtype=torch.float16, std=0.5)
    g = inputs(20, 1, 1, 1, 130, 20000, 64, dtype=torch.float16)[0] * 64
    out, lse = attention(q, k, v, return_lse=True)
    seen = torch.ones(1, 130, 20000, dtype=torch.bool, device=DEV)
    pos = (torch.arange(130, device=DEV) + 20000 - 130).expand(1, 130)
    check(attention_backward(g, q, k, v, out, lse), formula(q, k, v, g, out, seen, pos))


def test_repeats_streams_and_capture():
    spans, _, _ = plan(1, 500, 500, documents=[0, 130, 480], causal=True)
    q, k, v = inputs(21, 1, 6, 2, 500, 500, 128)
    g = inputs(22, 1, 6, 2, 500, 500, 128)[0]
    out, lse = attention(q, k, v, spans=spans, return_lse=True)
    ref = attention_backward(g, q, k, v, out, lse, spans=spans)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(attention_backward(g, q, k, v, out, lse, spans=spans), ref))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attention_backward(g, q, k, v, out, lse, spans=spans)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, ref))
    static = torch.zeros_like(g)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = attention_backward(static, q, k, v, out, lse, spans=spans)
        graphs.append((graph, made))
    static.copy_(g)
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for _, made in graphs:
        assert all(torch.equal(a, c) for a, c in zip(made, ref))
    assert _native.device_status(clear=True) == 0
