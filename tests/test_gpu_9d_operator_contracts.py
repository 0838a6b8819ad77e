"""What the block operators promise to autograd and about memory."""

import pytest
import torch

from peco_b200.linear import linear_act
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
