"""What the block operators' C entry points refuse before any launch: seen
without a GPU, where a call that passed its checks would return a CUDA error
and count a launch."""

import pytest

from peco_b200 import _native

WORKSPACE = 20005


@pytest.fixture(scope="module")
def lib():
    from peco_b200 import build
    build.build()
    return _native.load()


def test_workspaces_start_on_sixteen_bytes(lib):
    p, z, s = 1 << 20, 0, 0
    launches = lib.peco_launch_count()
    for at in (p + 4, p + 8, p + 1):
        # rows of 15 features are copied into the workspace
        assert lib.peco_linear_forward(p, 15, z, 0, p, 15, z, z, 0, z, 0, p, 8, z, 1, 2, 15, 0, 8, 0, 1, at, 1 << 20, s) == WORKSPACE
        # a gradient through an activation writes its product's operand there
        assert lib.peco_linear_backward(p, 8, p, p, 16, z, 0, p, 16, z, 0, p, z, p, p, z, 1, 2, 16, 0, 8, 1, 1, at, 1 << 20, s) == WORKSPACE
        # a norm's vector gradients their column sums
        assert lib.peco_gated_norm_backward(p, 64, 16, z, 0, 0, p, 64, 16, z, 0, 0, z, 0, p, 0, z, z, p, z, z, p, z, 0, z, z,
                                            1, 4, 16, 1, 0, 1e-6, 1e-6, 1.0, 1, at, 1 << 20, s) == WORKSPACE
    assert lib.peco_launch_count() == launches


def test_a_gate_gradient_needs_a_gate(lib):
    p, z = 1 << 20, 0
    launches = lib.peco_launch_count()
    # without one its sums would be read before they are written
    assert lib.peco_linear_backward(p, 8, p, p, 16, z, 0, p, 16, z, 0, z, z, z, z, p, 1, 2, 16, 0, 8, 1, 1, p, 1 << 20, 0) == 1
    assert lib.peco_launch_count() == launches
