"""Capped scores whose cap is much larger than they are: cap tanh(s / cap) stays as exact as s itself.

Tolerances: as in the tests of attention and of its gradient, but a score is off by 2^-20 (1 + the
magnitudes it is made of) whatever the cap (below a quarter of the cap tanh is a series,
off by a few 2^-23 of its value; above, the form with exponentials is off by a few 2^-23 of the cap, four
times the value at most).
"""

import pytest
import torch

import span_reference
import test_gpu_b_attention
import test_gpu_c_attention_grad
from peco_b200.attention import attention, attention_backward
from test_gpu_b_attention import DEV, inputs

pytestmark = pytest.mark.gpu


def size_without_cap(q, k, seen, pos, scale=None, softcap=None, slopes=None):
    return span_reference.score_size(q, k, seen, pos, scale=scale, slopes=slopes)


@pytest.mark.parametrize("softcap", [100.0, 3e3, 1e4, 1e6, 1e12, 1e30])
@pytest.mark.parametrize("std", [1.0, 3.0])
def test_large_caps(softcap, std, monkeypatch):
    monkeypatch.setattr(test_gpu_b_attention, "score_size", size_without_cap)
    monkeypatch.setattr(test_gpu_c_attention_grad, "score_size", size_without_cap)
    for n, m, h, kv, d, dtype in ((200, 333, 4, 2, 128, torch.float16), (1, 3000, 8, 1, 64, torch.float16),
                                  (130, 130, 2, 2, 40, torch.bfloat16)):
        q, k, v = inputs(n, 1, h, kv, n, m, d, dtype=dtype, std=std)
        g = inputs(n + 1, 1, h, kv, n, m, d, dtype=dtype)[0]
        seen = torch.ones(1, n, m, dtype=torch.bool, device=DEV)
        pos = (torch.arange(n, device=DEV) + m - n).expand(1, n)
        for args in (dict(softcap=softcap), dict(softcap=softcap, slopes=torch.rand(h, device=DEV) * 0.05)):
            out, lse = attention(q, k, v, return_lse=True, **args)
            test_gpu_b_attention.check(q, k, v, out, lse, seen, pos, **args)
            got = attention_backward(g, q, k, v, out, lse, **args)
            test_gpu_c_attention_grad.check(got, test_gpu_c_attention_grad.formula(q, k, v, g, out, seen, pos, **args))
