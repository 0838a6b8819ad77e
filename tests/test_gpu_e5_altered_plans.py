"""Plans whose numbers the caller changed: whatever they say, only the call's own keys are read.  (The order of the tiles
stays: results of tiles that a plan does not name are not written.)"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.attention import attention, attention_backward
from test_gpu_b_attention import DEV, inputs, plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("column,value", [(1, 5000), (0, -700), (2, 1 << 30)])
@pytest.mark.parametrize("what", ["rows", "tiles"])
def test_altered_plans_read_no_other_memory(what, column, value):
    """Keys that lie in the middle of a buffer of infinities and NaN (read past either end they would show in the scores)."""
    b, h, kv, n, m, d = 1, 4, 2, 200, 300, 64
    spans, _, _ = plan(b, n, m, documents=[0, 90, 200], key_documents=[0, 140, 300], causal=True)
    getattr(spans, what)[..., column] = value
    q, k, v = inputs(7, b, h, kv, n, m, d)
    g = inputs(8, b, h, kv, n, m, d)[0]
    v[:, :, 100] = float("inf")  # rows that are summed again, key by key
    around = [torch.full((b, kv, 3 * m, d), float("nan"), device=DEV, dtype=q.dtype) for _ in range(2)]
    inside = [t[:, :, m:2 * m].copy_(x) for t, x in zip(around, (k, v))]
    for args in ({}, dict(softcap=5.0)):
        out, lse = attention(q, *inside, spans=spans, return_lse=True, **args)
        assert not lse.isnan().any()
        alone = attention(q, k, v, spans=spans, return_lse=True, **args)
        assert torch.equal(alone[1], lse) and torch.equal(torch.nan_to_num(alone[0]), torch.nan_to_num(out))
        got = attention_backward(g, q, *inside, alone[0], lse, spans=spans, **args)
        for a, c in zip(got, attention_backward(g, q, k, v, alone[0], lse, spans=spans, **args)):
            assert torch.equal(torch.nan_to_num(a), torch.nan_to_num(c))
    assert _native.device_status(clear=True) == 0
