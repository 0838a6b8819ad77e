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
