"""modulated_norm and rotate where one block works through many rows or heads:
rows of later samples, refilled rings, prefetched rows and heads, and the
unaligned widths between 1025 and 4096.

Tolerances as in test_gpu_8_norm_rotary.
"""

import pytest
import torch
from test_gpu_8_norm_rotary import U, _forward64, _grid_pos, _inputs, _near, _norm_grads64, _rotate64

from peco_b200 import _native
from peco_b200.norms import modulated_norm, modulated_norm_backward
from peco_b200.rotary import rotate

pytestmark = pytest.mark.gpu

DEV = "cuda"
FORMS = [("layer", None, torch.bfloat16), ("rms", "rms", torch.float16), ("layer", "layer", torch.bfloat16),
         ("rms", None, torch.float16)]


def _case(i, b, t, width):
    norm, post, dtype = FORMS[i]
    return _inputs(i, b, t, width, dtype, gate=("sample", "shared", "sample", None)[i],
                   modulate=("sample", "sample", "shared", "sample")[i], weight=i != 0, post=post if i == 1 else None)


# a GPU of 148 SMs holds at most 148 x 16 blocks of four warps, of one to four rows each
@pytest.mark.parametrize("width,rows", [(64, 13001), (257, 13001), (512, 13001), (520, 13001), (1000, 5001), (1001, 5001),
                                        (1025, 5001), (1032, 5001), (2047, 3001), (2048, 3001), (2241, 3001), (3071, 3001),
                                        (3072, 3001), (3080, 3001), (3815, 3001), (4095, 3001), (4096, 3001), (5001, 2001),
                                        (6144, 2001), (6152, 2001), (8191, 1001), (8192, 1001), (9000, 1001), (16383, 501),
                                        (16384, 501)])
def test_norm_forward_walks(width, rows):
    for i, (norm, post, dtype) in enumerate(FORMS):
        c = _case(i, 3, rows, width)
        r, h = modulated_norm(**c, norm=norm, post_norm=post, residual_scale=0.5)
        r64, rsize, h64, hsize = _forward64(c, norm, post, 1e-6, 0.5)
        _near(r, r64, rsize, U[dtype])
        _near(h, h64, hsize, U[dtype])
        del r64, rsize, h64, hsize
        if i % 2:
            alone = dict(c, branch=None, gate=None, post_weight=None)
            _near(modulated_norm(**alone, norm=norm), *_forward64(alone, norm, None, 1e-6, 1.0)[2:], U[dtype])
        for _ in range(3):
            again = modulated_norm(**c, norm=norm, post_norm=post, residual_scale=0.5)
            assert torch.equal(again[0], r) and torch.equal(again[1], h)
    assert _native.device_status(clear=True) == 0


# a block takes the rows of one sample that are its number apart: three samples share 148 to 1776 blocks
@pytest.mark.parametrize("width,rows", [(64, 5001), (257, 5001), (512, 5001), (520, 2001), (1001, 2001), (1025, 1001), (1032, 1001),
                                        (2047, 1001), (2048, 1001), (2241, 1001), (3071, 1001), (3072, 1001), (3815, 1001),
                                        (4095, 1001), (4096, 1001), (5001, 501), (6144, 501), (8191, 501), (8192, 501),
                                        (9000, 501), (16383, 301), (16384, 301)])
def test_norm_backward_walks(width, rows):
    for i, (norm, post, dtype) in enumerate(FORMS):
        c = _case(i, 3, rows, width)
        g = torch.Generator(device=DEV).manual_seed(50 + i)
        gh, gr = (torch.randn(c["x"].shape, generator=g, device=DEV).to(dtype) for _ in range(2))
        opts = dict(norm=norm, post_norm=post, eps=1e-6, residual_scale=0.5)
        got = modulated_norm_backward(gh, gr, **c, **opts)
        ref = _norm_grads64(c, gh, gr, norm, post, 1e-6, 0.5)
        for name, value in c.items():
            mine = getattr(got, name)
            if value is None:
                assert mine is None
                continue
            v = ref[name]
            if name in ("x", "branch"):
                _near(mine, v, v.abs().amax(-1, keepdim=True) + 1.0, U[dtype], 2.0 ** -16)
            else:
                _near(mine, v, 10.0 * 3 * rows, U[dtype], 2.0 ** -16)
            assert (mine.double() - v).norm() <= U[dtype] * v.norm(), name
        del ref
        again = modulated_norm_backward(gh, gr, **c, **opts)
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, again))
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("aligned", [True, False])
def test_rotary_walks(dtype, interleaved, aligned):
    """Tokens enough for all blocks, so that a block takes all eleven heads (or, with fewer tokens, some of them)."""
    axes, theta = (16, 56, 56), 256.0
    for b, grid, text in ((1, (20, 40, 50), 77), (2, (4, 30, 41), 9)):
        n = torch.Size(grid).numel()
        g = torch.Generator(device=DEV).manual_seed(n)
        shift = 0 if aligned else 1
        wide = torch.randn((b, n + text, 11, 128 + 8), generator=g, device=DEV).to(dtype)
        heads = wide[..., shift:128 + shift].transpose(1, 2)
        q, k = heads[:, :7], heads[:, 7:]
        opts = dict(axes=axes, theta=theta, interleaved=interleaved)
        for inverse in (False, True):
            got = rotate(q, k, **opts, inverse=inverse, grid=grid)
            for x, y in zip((q, k), got):
                _near(y, *_rotate64(x, _grid_pos(grid), axes, theta, interleaved, inverse), U[dtype], 2.0 ** -21)
        keep = wide.clone()
        rotate(q, k, **opts, inverse=True, grid=grid, inplace=True)
        assert torch.equal(q, got[0]) and torch.equal(k, got[1])
        wide[..., shift:128 + shift] = keep[..., shift:128 + shift]
        assert torch.equal(wide, keep)  # and nothing beside the heads
        pos = torch.randint(0, 200, (b, n, 3), generator=g, device=DEV)
        for x, y in zip((q, k), rotate(q, k, **opts, positions=pos)):
            _near(y, *_rotate64(x, pos, axes, theta, interleaved, False), U[dtype], 2.0 ** -21)
