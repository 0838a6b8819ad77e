"""Block operators without a GPU: they refuse CPU tensors, their C entry points
check their arguments before any launch, and the workspace sizes are host
arithmetic."""

import ctypes

import pytest
import torch

from peco_b200 import _native
from peco_b200.linear import linear_act, linear_act_backward
from peco_b200.norms import modulated_norm, modulated_norm_backward
from peco_b200.rotary import AxialPositions, rotate


@pytest.fixture(scope="module")
def lib():
    from peco_b200 import build
    build.build()
    return _native.load()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 4, 16, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_act(x, x[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_act_backward(x[..., :4], x, x[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        modulated_norm(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        modulated_norm_backward(x, None, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotate(x[:, None], axes=(16,), grid=(4,))
    with pytest.raises(RuntimeError, match="CUDA"):
        AxialPositions((16,), grid=(4,)).rotate(x[:, None])


def test_arguments_are_checked_before_the_device():
    x = torch.zeros(2, 4, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        linear_act(x, x[0], activation="tanh")
    with pytest.raises(TypeError):
        linear_act(x.float(), x[0].float())
    with pytest.raises(ValueError):
        modulated_norm(x, norm="batch")
    with pytest.raises(ValueError):
        rotate(x[:, None], axes=(15,), grid=(4,))


def test_linear_workspace(lib):
    f = lib.peco_linear_forward_workspace
    aligned = 1 << 20
    assert f(aligned, 64, 0, 0, aligned, 64, 1, 100, 64, 0, 32) == 0
    # one unaligned operand: its rows at 16-byte strides, in 256-byte pieces
    assert f(aligned + 2, 64, 0, 0, aligned, 64, 1, 100, 64, 0, 32) == 100 * 64 * 2
    assert f(aligned, 33, 0, 0, aligned, 33, 1, 100, 33, 0, 32) == -(-100 * 40 * 2 // 256) * 256 + -(-32 * 40 * 2 // 256) * 256
    # a second input that starts inside a 16-byte piece of the weight's rows
    assert f(aligned, 40, aligned, 40, aligned, 80, 1, 10, 36, 40, 8) == 8 * 40 * 2 // 256 * 256 + 256 * (8 * 40 * 2 % 256 > 0)
    assert f(aligned, 64, 0, 0, aligned, 64, 1, 100, 0, 0, 32) == -1
    b = lib.peco_linear_backward_workspace
    # dz [rows, n rounded up to 8] and two sets of column sums
    assert b(aligned, 30, aligned, 64, 0, 0, aligned, 64, 2, 50, 64, 0, 30, 1, 0) >= 100 * 32 * 2 + 2 * 4 * 2 * 30


def test_entry_points_refuse_without_launching(lib):
    p, z = _native.P(1 << 20), _native.P(0)
    launches = lib.peco_launch_count()
    assert lib.peco_linear_forward(p, 16, z, 0, p, 16, z, z, 0, z, 0, p, 8, z, 1, 2, 16, 0, 8, 0, 2, z, 0, z) == 20001
    assert lib.peco_linear_forward(p, 16, z, 0, p, 16, z, z, 0, z, 0, z, 8, z, 1, 2, 16, 0, 8, 0, 1, z, 0, z) == 1
    assert lib.peco_linear_forward(p, 16, z, 0, p, 16, z, z, 0, z, 0, p, 8, z, 1, 0, 16, 0, 8, 0, 1, z, 0, z) == 0
    # a gradient through an activation without its pre-activation, and over no rows
    assert lib.peco_linear_backward(p, 8, z, p, 16, z, 0, p, 16, z, 0, p, z, z, z, z, 1, 2, 16, 0, 8, 1, 1, p, 1 << 20, z) == 1
    assert lib.peco_linear_backward(p, 8, p, p, 16, z, 0, p, 16, z, 0, p, z, z, z, z, 1, 0, 16, 0, 8, 1, 1, p, 1 << 20, z) == 1
    norm = [p, 64, 16, z, 0, 0, z, 0, z, 0, z, 0, z, z, z, p, 1, 4, 16]
    assert lib.peco_gated_norm(*norm, 0, 0, 1e-6, 1e-6, 1.0, 1, z) == 1      # no such norm
    assert lib.peco_gated_norm(*norm, 1, 2, 1e-6, 1e-6, 1.0, 1, z) == 1      # a post norm without a branch
    assert lib.peco_gated_norm(*norm, 1, 0, 1e-6, 1e-6, 1.0, 2, z) == 20001  # fp32
    assert lib.peco_gated_norm(*norm[:-1], 16385, 1, 0, 1e-6, 1e-6, 1.0, 1, z) == 20001
    st, axes, grid = (ctypes.c_longlong * 6)(64, 64, 16, 64, 64, 16), (ctypes.c_int * 2)(8, 8), (ctypes.c_int * 2)(2, 2)
    rot = [p, p, 1, st, z, z, 0, None, 1, 4]
    assert lib.peco_rotary(*rot, 5, 16, axes, 2, 100.0, grid, z, 0, 0, 0, 1, 0, 1, z) == 1   # more turned rows than rows
    assert lib.peco_rotary(*rot, 3, 16, axes, 2, 100.0, grid, z, 0, 0, 0, 1, 0, 1, z) == 1   # not the grid's size
    assert lib.peco_rotary(*rot, 4, 12, axes, 2, 100.0, grid, z, 0, 0, 0, 1, 0, 1, z) == 1   # sections wider than the head
    assert lib.peco_rotary(*rot, 4, 258, axes, 2, 100.0, grid, z, 0, 0, 0, 1, 0, 1, z) == 20001
    assert lib.peco_rotary(*rot, 4, 16, axes, 2, 100.0, None, z, 0, 0, 0, 1, 0, 1, z) == 1   # neither grid nor positions
    assert lib.peco_launch_count() == launches
    assert lib.peco_gated_norm_backward_workspace(2, 10, 64) % (12 * 2 * 64) == 0
    assert lib.peco_gated_norm_backward_workspace(-1, 10, 64) == -1
