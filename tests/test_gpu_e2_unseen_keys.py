"""Keys that no row sees may hold anything: what attention's gradients make of NaN and infinities there."""

import pytest
import torch

from peco_b200 import _native
from peco_b200.attention import attention, attention_backward
from test_gpu_b_attention import DEV, inputs, plan

pytestmark = pytest.mark.gpu

SCORES = [{}, dict(softcap=5.0), dict(softcap=5.0, slopes=True), dict(slopes=True)]


def unseen_keys(bad, h, kv, n, m, words, d, dtype, args):
    spans, seen, pos = plan(1, n, m, **words)
    q, k, v = inputs(n, 1, h, kv, n, m, d, dtype=dtype)
    g = inputs(n + 1, 1, h, kv, n, m, d, dtype=dtype)[0]
    args = dict(args, spans=spans)
    if args.get("slopes"):
        args["slopes"] = torch.rand(h, device=DEV) * 0.1
    out, lse = attention(q, k, v, return_lse=True, **args)
    clean = attention_backward(g, q, k, v, out, lse, **args)
    assert all(t.isfinite().all() for t in clean)
    blind, unseen = ~seen[0].any(1), ~seen[0].any(0)
    assert unseen.any()
    q, k, v, g = (t.clone() for t in (q, k, v, g))
    q[:, :, blind] = g[:, :, blind] = bad
    k[:, :, unseen] = bad
    k[:, :, unseen, 1] = 1.0  # (infinities that do not meet: a score of infinity, not only NaN)
    v[:, :, unseen] = bad
    out2, lse2 = attention(q, k, v, return_lse=True, **args)
    assert torch.equal(lse, lse2) and out2.isfinite().all()
    for a, c in zip(attention_backward(g, q, k, v, out, lse, **args), clean):
        assert torch.equal(a, c)
    assert (clean.k[:, :, unseen] == 0).all() and (clean.v[:, :, unseen] == 0).all()
    assert _native.device_status(clear=True) == 0


@pytest.mark.parametrize("args", SCORES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_behind_the_last_key(bad, args):
    for h, kv, n, m, words in ((2, 2, 300, 300, dict(documents=[0, 150, 290])), (4, 2, 300, 300, dict(lengths=[131])),
                               (12, 1, 130, 300, dict(lengths=[131])), (2, 1, 1, 300, dict(lengths=[40])),
                               (2, 2, 140, 500, dict(documents=[0, 60, 80], key_documents=[0, 250, 400]))):
        for d, dtype in ((64, torch.bfloat16), (128, torch.float16)):
            unseen_keys(bad, h, kv, n, m, words, d, dtype, args)


# documents with keys and no rows, and more keys than rows under a window: what nobody sees lies between keys that are seen
GAPS = [
    (60, 300, dict(documents=[0, 30, 30, 60], key_documents=[0, 100, 200, 300])),
    (60, 300, dict(documents=[0, 30, 60], key_documents=[0, 150, 300], window=4)),
    (60, 2000, dict(documents=[0, 30, 60], key_documents=[0, 900, 2000], window=20, causal=True)),
    (300, 1500, dict(documents=[0, 100, 100, 250, 290], key_documents=[0, 130, 700, 1000, 1200])),
    (300, 400, dict(documents=[0, 128, 128, 300], key_documents=[0, 127, 129, 300])),
    (40, 400, dict(documents=list(range(0, 41)), key_documents=list(range(0, 401, 10)), window=2)),
    (200, 700, dict(documents=[0, 90, 90, 200], key_documents=[0, 200, 201, 700], causal=True, prefix=30)),
]


@pytest.mark.parametrize("args", SCORES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("gap", GAPS)
def test_between_the_spans_of_a_tile(gap, bad, args):
    n, m, words = gap
    for h, kv, d, dtype in ((2, 2, 128, torch.bfloat16), (4, 1, 40, torch.float16)):
        unseen_keys(bad, h, kv, n, m, words, d, dtype, args)
