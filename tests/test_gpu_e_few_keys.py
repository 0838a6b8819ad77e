"""attention's gradients of rows that see one key or a few.

A row that sees one key has p = 1 whatever its score: dq and its part of dk are 0.
Rows of up to eight keys take delta = sum_j p_j (g.v_j) from their probabilities in fp32,
not from the rounded result: with e = 2^-20 (1 + the magnitudes a score is made of) and
A_ij = sum_d |g_id| |v_jd|, ds = p (g.v - delta) s' is off by
(2 e + 2^-20) p s' (A_ij + sum_j p_ij A_ij) and its rounding u |ds|, the rest as in the
gradient's tests.
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.attention import attention, attention_backward
from span_reference import attend, score_size
from test_gpu_b_attention import DEV, U, inputs, plan
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


def few_keys_formula(q, k, v, g, seen, pos, softcap=None, slopes=None):
    """dq and dk in 64 bits, and the bounds of their errors where no row sees more than eight keys."""
    u, group, n = U[q.dtype], q.shape[1] // k.shape[1], q.shape[2]
    tiny = 2.0 ** -25 if q.dtype is torch.float16 else 0.0
    args = dict(softcap=softcap, slopes=slopes)
    q, k, v, g = (t.double() for t in (q, k, v, g))
    kg, vg = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    _, _, p = attend(q, k, v, seen, pos, **args)
    e = 2.0 ** -20 * (1 + score_size(q, k, seen, pos, **args))
    factor = q.shape[-1] ** -0.5
    slope = torch.ones_like(p) if softcap is None else 1 - torch.tanh(q @ kg.transpose(-1, -2) * factor / softcap) ** 2
    gv = g @ vg.transpose(-1, -2)
    ds = p * (gv - (p * gv).sum(-1, keepdim=True)) * slope
    size = g.abs() @ vg.abs().transpose(-1, -2)
    size = size + (p * size).sum(-1, keepdim=True)
    off = p * (2 * e + 2.0 ** -20) * size * slope + u * ds.abs() + tiny * (p > 0)
    if softcap is not None:
        off = off + 2.0 ** -20 * p * size

    def shared(t):
        return t.unflatten(1, (k.shape[1], group)).sum(2)

    result = ((factor * ds @ kg, factor * (off + 8 * 2.0 ** -24 * ds.abs()) @ kg.abs()),
              (shared(factor * ds.transpose(-1, -2) @ q),
               shared(factor * (off + n * group * 2.0 ** -24 * ds.abs()).transpose(-1, -2) @ q.abs())))
    return [(ref, slack + u * ref.abs() + 2.0 ** -25) for ref, slack in result]


@pytest.mark.parametrize("mask", [(2, 70, 2, None), (1, 3, 8, None), (3, 40, 300, dict(lengths=[5, 8, 3])), (1, 300, 300, dict(window=4)),
                                  (1, 200, 7, dict(causal=True)), (2, 9, 200, dict(window=8, causal=True)),
                                  (1, 90, 90, dict(documents=[0, 2, 5, 9, 16, 24, 25, 33, 80], window=3))])
@pytest.mark.parametrize("form", [(4, 4, 128), (6, 1, 64), (4, 2, 40)])
def test_few_keys(mask, form):
    b, n, m, words = mask
    h, kv, d = form
    spans, seen, pos = masked(b, n, m, words)
    assert 1 < seen.sum(-1).max() <= 8
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(n + m, b, h, kv, n, m, d, dtype=dtype, token_major=True)
        g = inputs(n, b, h, kv, n, m, d, dtype=dtype)[0]
        for args in ({}, dict(softcap=5.0), dict(softcap=5.0, slopes=torch.rand(h, device=DEV) * 0.3)):
            out, lse = attention(q, k, v, spans=spans, return_lse=True, **args)
            got = attention_backward(g, q, k, v, out, lse, spans=spans, **args)
            for name, t, (ref, slack) in zip("qk", got, few_keys_formula(q, k, v, g, seen, pos, **args)):
                over = (t.double() - ref).abs() - slack
                assert (over <= 0).all(), (name, over.max().item())
            check(got, formula(q, k, v, g, out, seen, pos, **args))
