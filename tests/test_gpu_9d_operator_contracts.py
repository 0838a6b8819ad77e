"""What the block operators promise to autograd and about memory."""

import pytest
import torch

from peco_b200.linear import linear_act, linear_act_backward
from peco_b200.norms import modulated_norm_backward
from peco_b200.rotary import rotate

pytestmark = pytest.mark.gpu

DEV = "cuda"


def test_rotary_backward_turns_by_what_the_forward_turned_by():
    q = torch.randn(1, 2, 4, 16, device=DEV, requires_grad=True)
    pos = torch.arange(4, device=DEV)[:, None].clone()
    y = rotate(q, axes=(16,), positions=pos)
    pos += 1
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()
    axes, grid = [8, 8], [2, 2]
    y = rotate(q, axes=axes, grid=grid)
    axes[:], grid[:] = [4, 12], [1, 4]
    (g,) = torch.autograd.grad(y, q, torch.ones_like(y))
    assert torch.equal(g, rotate(torch.ones_like(y), axes=(8, 8), grid=(2, 2), inverse=True))
    pos = torch.rand(4, 1, device=DEV)
    y = rotate(q, axes=(16,), positions=pos)
    (g,) = torch.autograd.grad(y, q, torch.ones_like(y))
    assert torch.equal(g, rotate(torch.ones_like(y), axes=(16,), positions=pos, inverse=True))


def test_written_tensors_are_known_to_autograd():
    x, w = torch.randn(4, 16, device=DEV).bfloat16(), torch.randn(8, 16, device=DEV).bfloat16()
    buffer = torch.randn(4, 24, device=DEV).bfloat16()
    leaf = torch.randn(4, 8, device=DEV).bfloat16().requires_grad_()
    with_out = (leaf * buffer[:, 8:16]).sum()       # saves the buffer
    with torch.no_grad():
        linear_act(x, w, out=buffer[:, 8:16])
    with pytest.raises(RuntimeError, match="modified"):
        with_out.backward()
    q, k = torch.randn(1, 2, 4, 16, device=DEV), torch.randn(1, 2, 4, 16, device=DEV)
    scale = torch.randn(1, 2, 4, 16, device=DEV, requires_grad=True)
    with_q, with_k = (scale * q).sum(), (scale * k).sum()
    rotate(q, k, axes=(16,), grid=(4,), inplace=True)
    for loss in (with_q, with_k):
        with pytest.raises(RuntimeError, match="modified"):
            loss.backward()
    with_q = (scale * q).sum()
    rotate(q, axes=(16,), grid=(4,))                # not in place: nothing of the caller's is written
    linear_act(x, w, residual=buffer[:, :8])
    with_q.backward()
    with torch.inference_mode():                    # tensors without a version
        out = torch.empty(4, 8, device=DEV, dtype=torch.bfloat16)
        assert linear_act(x, w, out=out) is out
        rotate(torch.ones(1, 2, 4, 16, device=DEV), axes=(16,), grid=(4,), inplace=True)


def test_out_shares_no_memory_with_the_operands():
    m, k, n = 40, 16, 16
    x, w = torch.randn(m, k, device=DEV).bfloat16(), torch.randn(n, k, device=DEV).bfloat16()
    vec = torch.randn(n, device=DEV).bfloat16()
    wide = torch.randn(m + 1, 3 * n, device=DEV).bfloat16()
    left, mid, right = (wide[:m, i * n:(i + 1) * n] for i in range(3))
    below = wide[1:, n:2 * n]
    flat = torch.randn(2 * m * n, device=DEV).bfloat16()
    for kw in (dict(x=x, weight=w, out=x), dict(x=left, weight=w, out=left), dict(x=left, weight=w, out=wide[:m, 8:8 + n]),
               dict(x=left, weight=w, x2=mid, out=mid), dict(x=x[:n], weight=w, out=w), dict(x=x[:1], weight=w, bias=vec, out=vec[None]),
               dict(x=x[:1], weight=w, gate=vec, out=vec[None]), dict(x=x, weight=w, residual=mid, out=below),
               dict(x=x, weight=w, residual=flat[:m * n].view(m, n), out=flat[n:(m + 1) * n].view(m, n)),
               dict(x=x, weight=w, residual=flat[:m * n].view(m, n), out=flat.view(m, 2 * n)[:, :n])):
        kw = {key: torch.cat((t, t), 1) if key == "weight" and "x2" in kw else t for key, t in kw.items()}
        before = [t.clone() for t in kw.values()]
        with pytest.raises(ValueError, match="out shares memory with"):
            linear_act(**kw)
        assert all(torch.equal(a, b) for a, b in zip(before, kw.values()))
    # neighbours in one buffer, and the residual itself
    ref = linear_act(left, w, residual=right)
    assert linear_act(left, w, residual=right, out=mid) is mid and torch.equal(mid, ref)
    assert torch.equal(linear_act(left, w, residual=right, out=right), ref)
    ref = linear_act(x[:1], w, residual=wide[:1, :n])
    assert torch.equal(linear_act(x[:1], w, residual=wide[:1, :n], out=wide[0, :n][None]), ref)
    # an operand that has to be copied is read from its copy
    square = torch.randn(n, n, device=DEV).bfloat16()
    ref = linear_act(square.t(), w)
    assert torch.equal(linear_act(square.t(), w, out=square), ref)


def test_inplace_queries_and_keys_share_no_memory():
    opts = dict(axes=(8, 8), grid=(2, 3))
    qkv = torch.randn(2, 7, 10, 16, device=DEV)                   # token rows of 10 heads
    heads = qkv.transpose(1, 2)
    keep = qkv.clone()
    for q, k in ((heads[:, :4], heads[:, 3:6]), (heads[:, 2:6], heads[:, :3]), (heads, heads[:, 9:]), (heads[:1], heads[:1]),
                 (heads[:, :1], heads[:, 1:2].as_strided((2, 1, 7, 16), (1120, 160, 80, 1), 80))):
        with pytest.raises(ValueError, match="share memory"):
            rotate(q, k, **opts, inplace=True)
    assert torch.equal(qkv, keep)
    want_q, want_k = rotate(heads[:, :6], heads[:, 6:8], **opts)  # neighbours in one buffer
    q, k = rotate(heads[:, :6], heads[:, 6:8], **opts, inplace=True)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(qkv[:, :, 8:], keep[:, :, 8:])


def test_needs_may_be_any_iterable():
    x, w, g = (torch.randn(16, 16, device=DEV).bfloat16() for _ in range(3))
    got = linear_act_backward(g, x, w, bias=True, needs=iter(["weight", "x"]))
    assert got.x is not None and got.weight is not None and got.bias is None
    with pytest.raises(ValueError):
        linear_act_backward(g, x, w, needs=iter(["x", "gain"]))
    got = modulated_norm_backward(g, None, x, scale=x[0], shift=w[0], needs=iter(["shift", "x"]))
    assert got.x is not None and got.shift is not None and got.scale is None
    with pytest.raises(ValueError):
        modulated_norm_backward(g, None, x, needs=iter(["x", "scale"]))
