"""What the block operators refuse before they look for a device."""

import random

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from peco_b200 import _native
from peco_b200.linear import linear_act, linear_act_backward
from peco_b200.norms import modulated_norm, modulated_norm_backward
from peco_b200.rotary import _share_memory, rotate


def test_forward_mode_tangents_are_refused():
    x = torch.zeros(1, 4, 16, dtype=torch.bfloat16)
    w, v = torch.zeros(16, 16, dtype=torch.bfloat16), torch.zeros(16, dtype=torch.bfloat16)
    rot = dict(axes=(16,), grid=(4,))
    calls = [
        lambda dual: linear_act(dual(x), w), lambda dual: linear_act(x, dual(w)), lambda dual: linear_act(x, w, dual(v)),
        lambda dual: linear_act(x, w, gate=dual(v)), lambda dual: linear_act(x, w, residual=dual(x)),
        lambda dual: linear_act_backward(dual(x), x, w), lambda dual: linear_act_backward(x, x, w, preact=dual(x), activation="silu"),
        lambda dual: modulated_norm(dual(x)), lambda dual: modulated_norm(x, dual(x)), lambda dual: modulated_norm(x, scale=dual(v)),
        lambda dual: modulated_norm(x, weight=dual(v)), lambda dual: modulated_norm_backward(dual(x), None, x),
        lambda dual: modulated_norm_backward(x, None, x, shift=dual(v)),
        lambda dual: rotate(dual(x[None]), **rot), lambda dual: rotate(x[None], dual(x[None]), **rot),
    ]
    with forward_ad.dual_level():
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
            with pytest.raises(RuntimeError, match="CUDA"):  # an open level alone changes nothing
                call(lambda t: t)
    for call in calls:
        with pytest.raises(RuntimeError, match="CUDA"):
            call(lambda t: t)


def test_positions_that_want_a_gradient_are_refused():
    q, pos = torch.zeros(1, 1, 4, 16), torch.zeros(4, 1, requires_grad=True)
    for x in (q, q.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="gradient of positions"):
            rotate(x, axes=(16,), positions=pos)
        with pytest.raises(RuntimeError, match="CUDA"):
            rotate(x, axes=(16,), positions=pos.detach())
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        rotate(q, axes=(16,), positions=pos)


def test_out_that_wants_a_gradient_is_refused():
    x, w = torch.zeros(4, 16, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.bfloat16)
    out = torch.zeros(4, 8, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="does not record gradients"):
        linear_act(x, w, out=out)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        linear_act(x, w, out=out)


def test_rows_overlap_against_every_element():
    rng = random.Random(0)
    seen = [0, 0]
    for _ in range(4000):
        sets = []
        for _ in range(2):
            width = rng.randint(1, 6)
            sets.append((rng.randint(0, 60), rng.randint(1, 7), rng.randint(width, 14), width))
        if rng.random() < 0.5:  # columns of one buffer
            step = max(sets[0][2], sets[1][2])
            sets = [(p, n, step, w) for p, n, _, w in sets]
        a, b = ({p + i * s + j for i in range(n) for j in range(w)} for p, n, s, w in sets)
        assert _native.rows_overlap(*sets) == bool(a & b) == _native.rows_overlap(*sets[::-1]), sets
        seen[bool(a & b)] += 1
    assert min(seen) > 500
    big = 1 << 40  # rows of a long buffer
    assert not _native.rows_overlap((big, 1 << 20, 4096, 2048), (big + 2048, 1 << 20, 4096, 2048))
    assert _native.rows_overlap((big, 1 << 20, 4096, 2048), (big + 2047, 1 << 20, 4096, 2048))
    assert _native.rows_overlap((big, 1 << 20, 4096, 2049), (big + 2048, 7, 8192, 2048))


def test_shared_memory_of_queries_and_keys_against_every_element():
    """Views of one small buffer in the layouts of attention calls, and arbitrary ones."""
    rng = random.Random(1)
    buffer = torch.arange(4096, dtype=torch.float32)
    seen = [0, 0]

    def elements(t):
        return set(t.reshape(-1).tolist())

    def view(b, h, n, d):
        order = rng.sample(range(3), 3)     # which of batch, head and token runs innermost
        strides, step = [0, 0, 0], d + rng.choice((0, 0, 3))
        for axis in order:
            strides[axis] = step
            step *= (b, h, n)[axis] + rng.choice((0, 0, 1))
        return torch.as_strided(buffer, (b, h, n, d), (*strides, 1), rng.randint(0, 120))

    for _ in range(3000):
        b, n, d = rng.randint(1, 2), rng.randint(1, 4), 2 * rng.randint(1, 2)
        if rng.random() < 0.5:              # heads of one projection, [B, N, heads, D] or [B, heads, N, D]
            heads = 5
            whole = torch.as_strided(buffer, (b, n, heads, d), (n * heads * d, heads * d, d, 1)).transpose(1, 2) \
                if rng.random() < 0.5 else torch.as_strided(buffer, (b, heads, n, d), (heads * n * d, n * d, d, 1))
            cut, end = sorted(rng.sample(range(1, heads + 1), 2))
            start = rng.randint(0, cut)
            q, k = whole[:, :cut], whole[:, start if start < end else cut:end]
        else:
            q, k = view(b, rng.randint(1, 3), n, d), view(b, rng.randint(1, 3), n, d)
        common = bool(elements(q) & elements(k))
        assert _share_memory(q, k) == common == _share_memory(k, q), (q.shape, q.stride(), k.shape, k.stride())
        seen[common] += 1
    assert min(seen) > 300
    assert not _share_memory(buffer[:0].view(1, 0, 4, 2), buffer[:8].view(1, 1, 4, 2))
