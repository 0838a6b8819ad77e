"""What attention refuses whatever else its call asks for."""

import ctypes

import pytest
import torch

from peco_b200 import _native
from peco_b200.attention import KeySpans, attention, attention_backward

Q = torch.zeros(2, 4, 6, 64, dtype=torch.bfloat16)
K = torch.zeros(2, 2, 9, 64, dtype=torch.bfloat16)
LSE = torch.zeros(2, 4, 6)


@pytest.mark.parametrize("wants", ["", "q", "k", "v", "qkv"])
def test_a_gradient_of_slopes_is_refused(wants):
    """Also where the call is recorded for the other gradients: it would give none for slopes without a word."""
    slopes = torch.zeros(4, requires_grad=True)
    q, k, v = (t.clone().requires_grad_(name in wants) for name, t in zip("qkv", (Q, K, K)))
    with pytest.raises(RuntimeError, match="gradient of slopes"):
        attention(q, k, v, slopes=slopes)
    with pytest.raises(RuntimeError, match="gradient of slopes"):
        attention_backward(Q, q, k, v, Q, LSE, slopes=slopes)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        attention(q, k, v, slopes=slopes)
    with pytest.raises(RuntimeError, match="CUDA"):
        attention(q, k, v, slopes=slopes.detach())


@pytest.mark.parametrize("args", [dict(softcap=1e-50), dict(softcap=1e-31), dict(softcap=1e31), dict(softcap=1e300), dict(scale=1e-46),
                                  dict(scale=1e39), dict(scale=1e300), dict(scale=1e25, softcap=1e-10)])
def test_scales_and_caps_past_fp32_are_refused(args):
    """They would reach the kernels as 0 (a cap of 0 is none), as infinity, or make their quotient infinite."""
    with pytest.raises(ValueError, match="scale|softcap"):
        attention(Q, K, K, **args)
    with pytest.raises(ValueError, match="scale|softcap"):
        attention_backward(Q, Q, K, K, Q, LSE, **args)


@pytest.mark.parametrize("scale,cap", [(float("inf"), 0.0), (1e31, 0.0), (1e-31, 0.0), (1.0, float("inf")), (1.0, 1e31), (1.0, 1e-31),
                                       (1.0, float("nan")), (1e20, 1e-20)])
def test_entries_refuse_scales_and_caps_out_of_range(scale, cap):
    lib = _native.load()
    at = 0x10000  # never read: every call is refused
    strides = (ctypes.c_longlong * 24)(*[4 * 6 * 64, 6 * 64, 64] * 8)
    assert lib.peco_span_attention(at, at, at, strides, 0, 0, 0, 0, scale, cap, at, at, 2, 4, 2, 6, 9, 64, 1, 0, 0, 0) == 1
    assert lib.peco_span_attention_backward(at, at, at, at, at, at, strides, 0, 0, 0, 0, scale, cap, at, at, at, 2, 4, 2, 6, 9, 64, 1,
                                            at, 1 << 20, 0) == 1


def off_16_bytes(t):
    return torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape)


@pytest.mark.parametrize("which", [0, 1])
def test_plans_off_16_bytes_are_refused(which):
    """The kernels read them 16 bytes at a time: a misaligned address would be a fault."""
    rows, tiles = torch.zeros(2, 6, 4, dtype=torch.int32), torch.zeros(2, 1, 4, dtype=torch.int32)
    rows, tiles = (off_16_bytes(t) if i == which else t for i, t in enumerate((rows, tiles)))
    spans = KeySpans(rows, tiles, 6, 9)
    with pytest.raises(ValueError, match="spans"):
        attention(Q, K, K, spans=spans)
    with pytest.raises(ValueError, match="spans"):
        attention_backward(Q, Q, K, K, Q, LSE, spans=spans)


@pytest.mark.parametrize("rows,tiles", [(4, 0), (8, 0), (0, 4), (0, 12)])
def test_entries_refuse_plans_off_16_bytes(rows, tiles):
    lib = _native.load()
    at = 0x10000  # never read: every call is refused
    strides = (ctypes.c_longlong * 24)(*[4 * 6 * 64, 6 * 64, 64] * 8)
    assert lib.peco_span_attention(at, at, at, strides, at + rows, at + tiles, 1, 0, 1.0, 0.0, at, at, 2, 4, 2, 6, 9, 64, 1, 0, 0, 0) == 1
    assert lib.peco_span_attention_backward(at, at, at, at, at, at, strides, at + rows, at + tiles, 1, 0, 1.0, 0.0, at, at, at, 2, 4, 2,
                                            6, 9, 64, 1, at, 1 << 20, 0) == 1
