"""attention's gradients of rows that see one key or a few.

A row that sees one key has p = 1 whatever its score: dq and its part of dk are 0.
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.attention import attention, attention_backward
from test_gpu_b_attention import DEV, inputs, plan
from test_gpu_c_attention_grad import check, formula

pytestmark = pytest.mark.gpu


def masked(b, n, m, words):
    """(spans or None, mask, positions)"""
    if words is not None:
        return plan(b, n, m, **words)
    return None, torch.ones(b, n, m, dtype=torch.bool, device=DEV), (torch.arange(n, device=DEV) + m - n).expand(b, n)


ONE_KEY = [
    (1, 1, 1, None), (2, 300, 1, None), (3, 1, 1, dict(lengths=[1, 0, 1])), (1, 129, 1, dict(causal=True)),
    (1, 300, 300, dict(window=1)), (2, 5, 700, dict(window=1, causal=True)), (1, 150, 150, dict(documents=list(range(0, 140)))),
    (1, 1, 129, dict(window=1)), (2, 90, 257, dict(lengths=[129, 1], window=1)),
    (1, 130, 400, dict(documents=[0, 127, 128, 130], key_documents=[0, 127, 128, 400], causal=True)),  # one-key rows among others
    (2, 260, 260, dict(documents=[[0, 1, 2, 200], [0, 128, 129, 260]], causal=True)),
    (1, 300, 3, dict(causal=True)),
]


@pytest.mark.parametrize("mask", ONE_KEY)
@pytest.mark.parametrize("form", [(4, 4, 128), (6, 1, 64), (16, 1, 40)])
def test_one_key_has_no_gradient_of_its_score(mask, form):
    b, n, m, words = mask
    h, kv, d = form
    spans, seen, pos = masked(b, n, m, words)
    alone = seen.sum(-1) == 1  # [b, n]
    assert alone.any()
    others = (seen & ~alone[..., None]).any(1)  # keys that a row with several sees
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(n + m, b, h, kv, n, m, d, dtype=dtype)
        g = inputs(n, b, h, kv, n, m, d, dtype=dtype)[0]
        slopes = torch.rand(h, device=DEV) * 0.1
        for args in ({}, dict(softcap=5.0, slopes=slopes)):
            out, lse = attention(q, k, v, spans=spans, return_lse=True, **args)
            got = attention_backward(g, q, k, v, out, lse, spans=spans, **args)
            assert (got.q.transpose(1, 2)[alone] == 0).all()
            assert (got.k.transpose(1, 2)[~others] == 0).all()
            check(got, formula(q, k, v, g, out, seen, pos, **args))


def test_nan_of_a_row_with_one_key():
    """A NaN gradient or score of such a row still reaches dv and the row's own dq."""
    spans, seen, pos = plan(1, 64, 64, window=1)
    q, k, v = inputs(3, 1, 2, 2, 64, 64, 64)
    g = inputs(4, 1, 2, 2, 64, 64, 64)[0]
    out, lse = attention(q, k, v, spans=spans, return_lse=True)
    g[0, 1, 5, 7] = float("nan")
    got = attention_backward(g, q, k, v, out, lse, spans=spans)
    assert got.q[0, 1, 5].isnan().all() and got.v[0, 1, 5, 7].isnan()
    assert (got.q[0, 0] == 0).all()
    assert _native.device_status(clear=True) == 0
