"""attention on the GPU against the definition in 64 bits, its mask made from words.

Tolerances.  u: unit roundoff of the type (2^-8 bf16, 2^-11 fp16).  A score is
off by e = 2^-20 times the magnitudes it is made of (fp32 sums of D <= 128
products, two scalings, the cap within a few 2^-23 of its size, 2^x within
2^-22), which is the relative error of a probability before its rounding to 16
bits (u; in fp16 at least 2^-25, the largest being 1 or more).  So
  |out error| <= u |out| + (u + 2 e + M 2^-24) sum p |v| + 2^-25 sum |v|,
M keys summed in fp32; the logarithm is off by e + M 2^-24 and 2^-22 of itself.
"""

import pytest
import torch

from peco_b200 import _native
from peco_b200.attention import attention, key_spans
from span_reference import attend, score_size, visible

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def inputs(seed, b, h, kv, n, m, d, dtype=torch.bfloat16, std=1.0, token_major=False):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def heads(count, rows):
        if token_major:
            return (torch.randn(b, rows, count, d, generator=g, device=DEV) * std).to(dtype).transpose(1, 2)
        return (torch.randn(b, count, rows, d, generator=g, device=DEV) * std).to(dtype)

    return heads(h, n), heads(kv, m), heads(kv, m)


def plan(b, n, m, **words):
    """(KeySpans, mask, positions) from host lists."""
    on = {k: torch.tensor(v, dtype=torch.int32, device=DEV) if isinstance(v, (list, tuple)) else v for k, v in words.items()}
    seen, pos = visible(b, n, m, **{k: v for k, v in words.items() if v is not None})
    return key_spans(b, n, m, device=DEV, **on), seen.to(DEV), pos.to(DEV)


def check(q, k, v, got, lse, seen, pos, **args):
    q64, k64, v64 = q.double(), k.double(), v.double()
    ref, ref_lse, p = attend(q64, k64, v64, seen, pos, **args)
    u, m = U[q.dtype], k.shape[2]
    group = q.shape[1] // k.shape[1]
    e = 2.0 ** -20 * (1 + score_size(q64, k64, seen, pos, **args))
    size = p @ v64.abs().repeat_interleave(group, 1)
    total = v64.abs().sum(2, keepdim=True).repeat_interleave(group, 1)
    slack = u * ref.abs() + (u + 2 * e + m * 2.0 ** -24) * size + 2.0 ** -25 * (total + 1)
    assert torch.isfinite(got).all()
    over = (got.double() - ref).abs() - slack
    assert (over <= 0).all(), over.max().item()
    empty = ~seen.any(-1)[:, None].expand(ref_lse.shape)
    assert (got[empty] == 0).all() and (lse[empty] == -torch.inf).all()
    off = (lse.double() - ref_lse)[~empty].abs()
    bound = (e[..., 0] + m * 2.0 ** -24 + 2.0 ** -22 * ref_lse.abs())[~empty]
    assert (off <= bound).all(), (off - bound).max().item()
    assert _native.device_status(clear=True) == 0


SIZES = [  # batch, heads, key heads, rows, keys, dims
    (1, 1, 1, 1, 1, 8), (1, 2, 1, 1, 300, 64), (2, 3, 3, 5, 7, 40), (1, 2, 2, 128, 128, 128), (1, 2, 2, 129, 127, 64),
    (2, 4, 2, 200, 333, 80), (1, 8, 2, 64, 500, 128), (1, 8, 1, 16, 257, 128), (3, 6, 2, 1, 2049, 128), (1, 24, 24, 600, 640, 128),
    (1, 12, 4, 33, 4100, 96), (2, 40, 40, 257, 200, 64), (1, 2, 2, 1000, 3, 128), (2, 64, 32, 385, 385, 128),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", SIZES)
def test_every_key(size, dtype):
    b, h, kv, n, m, d = size
    q, k, v = inputs(n + m, *size, dtype=dtype, token_major=n % 2 == 1)
    out, lse = attention(q, k, v, return_lse=True)
    assert out.stride() == q.stride()
    seen = torch.ones(b, n, m, dtype=torch.bool, device=DEV)
    pos = (torch.arange(n, device=DEV) + m - n).expand(b, n)
    check(q, k, v, out, lse, seen, pos)
    slopes = torch.rand(h, device=DEV) * 0.2
    for args in (dict(softcap=2.0), dict(slopes=slopes), dict(softcap=30.0, slopes=slopes, scale=0.3)):
        out, lse = attention(q, k, v, return_lse=True, **args)
        check(q, k, v, out, lse, seen, pos, **args)


MASKS = [
    (2, 300, 300, dict(causal=True)),
    (2, 300, 300, dict(causal=True, prefix=40)),
    (1, 300, 300, dict(causal=True, prefix=1000)),
    (1, 300, 300, dict(causal=True, window=17)),
    (1, 700, 700, dict(window=1)),
    (1, 700, 700, dict(window=130)),
    (2, 100, 400, dict(causal=True)),
    (2, 400, 100, dict(causal=True)),                                  # the first 300 rows see nothing
    (2, 400, 100, dict(causal=True, prefix=3)),
    (3, 5, 300, dict(lengths=[300, 1, 129])),
    (3, 1, 3000, dict(lengths=[3000, 0, 129], causal=True)),
    (2, 260, 260, dict(lengths=[100, 260], causal=True)),
    (1, 520, 520, dict(documents=[0, 100, 101, 101, 400, 500])),        # empty document, rows behind the last
    (1, 520, 520, dict(documents=[20, 100, 101, 101, 400, 520], causal=True)),
    (1, 520, 520, dict(documents=[0, 100, 300, 520], causal=True, prefix=[10, 0, 500])),
    (2, 520, 520, dict(documents=[[0, 100, 520], [0, 519, 520]], causal=True, prefix=[[3, 90], [0, 7]])),
    (2, 150, 600, dict(documents=[0, 100, 150], key_documents=[[0, 300, 600], [10, 20, 30]], window=100)),
    (1, 256, 256, dict(documents=list(range(257)))),                    # a document a row
]


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("form", [(4, 4, 128), (4, 1, 64), (150, 50, 40)])
def test_masks(mask, form):
    b, n, m, words = mask
    h, kv, d = form
    spans, seen, pos = plan(b, n, m, **words)
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v = inputs(n, b, h, kv, n, m, d, dtype=dtype)
        slopes = torch.rand(h, device=DEV) * 0.1
        for args in ({}, dict(softcap=5.0, slopes=slopes)):
            out, lse = attention(q, k, v, spans=spans, return_lse=True, **args)
            check(q, k, v, out, lse, seen, pos, **args)


# few rows over caches of very unequal lengths, an empty one among them: their keys are shared out over the CTAs
@pytest.mark.parametrize("form", [(6, 1, 8, 2, 64), (9, 3, 16, 8, 128), (37, 1, 2, 2, 40), (1, 200, 8, 1, 128)])
def test_unequal_caches(form):
    b, n, h, kv, d = form
    lengths = [(7000, 0, 129, 1, 2500, 640)[i % 6] + i for i in range(b)]
    spans, seen, pos = plan(b, n, 7100, lengths=lengths, causal=True)
    q, k, v = inputs(b, b, h, kv, n, 7100, d)
    slopes = torch.rand(h, device=DEV) * 0.01
    for args in ({}, dict(softcap=5.0, slopes=slopes)):
        out, lse = attention(q, k, v, spans=spans, return_lse=True, **args)
        check(q, k, v, out, lse, seen, pos, **args)
    none = plan(b, n, 7100, lengths=[0] * b)[0]
    out, lse = attention(q, k, v, spans=none, return_lse=True)
    assert (out == 0).all() and (lse == -torch.inf).all()


@pytest.mark.parametrize("mask", [(1, 520, 520, dict(documents=[0, 100, 300, 500], causal=True)), (3, 1500, 700, dict(lengths=[700, 0, 9])),
                                  (2, 1000, 1000, dict(window=40, causal=True)), (1, 140000, 140000, dict(causal=True)), (1, 1, 5, {})])
def test_every_tile_has_its_turn(mask):
    """The plan names each tile of rows once, and no tile before one that sees more keys (of up to 1024 tiles)."""
    b, n, m, words = mask
    words = {k: torch.tensor(v, dtype=torch.int32, device=DEV) if isinstance(v, list) else v for k, v in words.items()}
    spans = key_spans(b, n, m, device=DEV, **words)
    tiles = -(-n // 128)
    turn = spans.rows[:, :tiles, 3].long()
    assert (turn.sort(1).values == torch.arange(tiles, device=DEV)).all() and (spans.rows[:, tiles:, 3] == 0).all()
    sizes = ((spans.tiles[..., 1].long() - spans.tiles[..., 0]).clamp(min=0) + 127) // 128
    if tiles <= 1024:
        assert (sizes.gather(1, turn).diff(dim=1) <= 0).all()


def test_one_plan_for_all_samples():
    spans, seen, pos = plan(1, 200, 200, causal=True)
    q, k, v = inputs(0, 3, 2, 2, 200, 200, 64)
    out, lse = attention(q, k, v, spans=spans, return_lse=True)
    check(q, k, v, out, lse, seen.expand(3, -1, -1), pos.expand(3, -1))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_masked_keys_and_values_may_hold_anything(bad):
    """Rows whose mask leaves a key out are what they are with a finite key there."""
    for h, kv, n, m, words in ((2, 2, 300, 300, dict(documents=[0, 150, 290])), (2, 1, 300, 300, dict(causal=True)),
                               (8, 2, 1, 3000, dict(lengths=[1500])), (2, 2, 300, 300, dict(lengths=[131])),
                               (2, 2, 70, 600, dict(documents=[0, 30, 60], key_documents=[0, 250, 600]))):
        spans, seen, pos = plan(1, n, m, **words)
        for d in (128, 40):
            q, k, v = inputs(1, 1, h, kv, n, m, d)
            at = torch.tensor([j for j in (m - 1, m - 3, 170, 270) if j < m and (n > 1 or j >= 1500)], device=DEV)
            clean = attention(q, k, v, spans=spans, return_lse=True, softcap=9.0)
            dirty_v, dirty_k = v.clone(), k.clone()
            dirty_v[:, :, at, ::3] = bad
            dirty_k[:, :, at] = bad
            apart = ~seen[0][:, at].any(-1)
            assert apart.any()
            for k2, v2 in ((k, dirty_v), (dirty_k, v), (dirty_k, dirty_v)):
                out, lse = attention(q, k2, v2, spans=spans, return_lse=True, softcap=9.0)
                assert torch.equal(lse[:, :, apart], clean[1][:, :, apart])
                # (a value's row may be summed again in fp32, without the 16-bit probabilities)
                near = (out[:, :, apart].double() - clean[0][:, :, apart].double()).abs()
                assert (near <= 4 * U[q.dtype] * v.double().abs().amax()).all() and not near.isnan().any()
            out = attention(q, k, dirty_v, spans=spans)
            hit = seen[0][:, at].any(-1)
            assert not torch.isfinite(out[:, :, hit][..., ::3]).any()
    assert _native.device_status(clear=True) == 0


def test_what_a_row_sees_reaches_it():
    """NaN in a query row, or in a key that a row sees, makes that row NaN and no other; also in parts of split keys."""
    for h, kv, n, m in ((2, 2, 300, 500), (4, 1, 2, 5000), (2, 2, 3, 60), (2, 1, 130, 129)):
        spans, seen, pos = plan(1, n, m, causal=True, window=200)
        q, k, v = inputs(23, 1, h, kv, n, m, 64)
        clean = attention(q, k, v, spans=spans, return_lse=True)
        for args in ({}, dict(softcap=9.0)):
            bad_q, bad_k = q.clone(), k.clone()
            bad_q[:, 0, n // 2, 3] = float("nan")
            out, lse = attention(bad_q, k, v, spans=spans, return_lse=True, **args)
            row = torch.zeros(1, h, n, dtype=torch.bool, device=DEV)
            row[:, 0, n // 2] = seen[0, n // 2].any()
            assert torch.equal(lse.isnan(), row) and torch.equal(out.isnan().all(-1), row) and torch.equal(out.isnan().any(-1), row)
            bad_k[:, :, m - 20, 5] = float("nan")
            out, lse = attention(q, bad_k, v, spans=spans, return_lse=True, **args)
            row = seen[:, None, :, m - 20].expand(1, h, n)
            assert row.any() and torch.equal(lse.isnan(), row) and torch.equal(out.isnan().all(-1), row)
            if not args:
                assert torch.equal(out[~row], clean[0][~row]) and torch.equal(lse[~row], clean[1][~row])


def test_wide_offsets():
    ends = torch.tensor([0, 70, 2 ** 40], device=DEV)  # the last document ends with the sequence
    spans = key_spans(1, 100, 100, documents=ends, causal=True, prefix=torch.tensor([2 ** 33, 5], device=DEV))
    same = key_spans(1, 100, 100, documents=torch.tensor([0, 70, 100], dtype=torch.int32, device=DEV), causal=True,
                     prefix=torch.tensor([100, 5], device=DEV))
    assert torch.equal(spans.rows, same.rows) and torch.equal(spans.tiles, same.tiles)
    lengths = key_spans(2, 3, 50, lengths=torch.tensor([2 ** 35, -2 ** 40], device=DEV))
    assert lengths.rows[0, :, 1].tolist() == [50] * 3 and lengths.rows[1, :, 1].tolist() == [0] * 3


def test_scores_at_the_ends_of_their_range():
    q, k, v = inputs(2, 1, 2, 2, 140, 200, 64, std=8.0)  # scores of some hundreds
    spans, seen, pos = plan(1, 140, 200, causal=True)
    out, lse = attention(q, k, v, spans=spans, return_lse=True, scale=1.0)
    check(q, k, v, out, lse, seen, pos, scale=1.0)
    k[:, :, 5] = -torch.inf * q[:, :1, :1].sign()[:, :, 0, :1]  # one key infinitely far for some rows
    out = attention(q.abs(), -k.abs(), v)  # every key but none infinite positive: finite results
    assert torch.isfinite(out).all()
    out, lse = attention(torch.ones_like(q), torch.full_like(k, -torch.inf), v, return_lse=True)
    assert (out == 0).all() and (lse == -torch.inf).all()  # all scores -inf: as if nothing were visible


def test_layouts():
    b, h, kv, n, m, d = 2, 4, 2, 150, 170, 64
    q, k, v = inputs(3, b, h, kv, n, m, d)
    ref = attention(q, k, v)
    joined = torch.randn(b, m, (kv + kv) * d + 8, device=DEV).to(torch.bfloat16)  # keys and values of one projection
    joined[..., :kv * d] = k.transpose(1, 2).flatten(2)
    joined[..., kv * d:2 * kv * d] = v.transpose(1, 2).flatten(2)
    k2, v2 = (joined[..., s * kv * d:(s + 1) * kv * d].unflatten(-1, (kv, d)).transpose(1, 2) for s in (0, 1))
    assert torch.equal(attention(q, k2, v2), ref)
    odd = torch.zeros(b, h, n, d + 1, device=DEV, dtype=torch.bfloat16)
    odd[..., 1:] = q
    assert torch.equal(attention(odd[..., 1:], k, v), ref)                       # rows off 16 bytes
    assert torch.equal(attention(q.transpose(-1, -2).contiguous().transpose(-1, -2), k, v), ref)
    one = q[:, :1].expand(b, h, n, d)                                             # a broadcast head
    assert torch.equal(attention(one, k, v), attention(one.contiguous(), k, v))
    # one row, and rows of one sample of a larger cache
    cache = torch.randn(4, kv, 4096, d, device=DEV).to(torch.bfloat16)
    spans = key_spans(2, 1, 4000, lengths=torch.tensor([4000, 77], device=DEV))
    a = attention(q[:, :, :1], cache[1:3, :, 5:4005], cache[2:, :, :4000], spans=spans)
    c = attention(q[:, :, :1].contiguous(), cache[1:3, :, 5:4005].contiguous(), cache[2:, :, :4000].contiguous(), spans=spans)
    assert torch.equal(a, c)


def test_no_rows_and_no_keys():
    q, k, v = inputs(4, 2, 4, 2, 6, 9, 64)
    out, lse = attention(q[:, :, :0], k, v, return_lse=True)
    assert out.shape == (2, 4, 0, 64) and lse.shape == (2, 4, 0)
    out, lse = attention(q, k[:, :, :0], v[:, :, :0], return_lse=True)
    assert (out == 0).all() and (lse == -torch.inf).all()
    spans = key_spans(2, 6, 0, causal=True, device=DEV)
    assert (attention(q, k[:, :, :0], v[:, :, :0], spans=spans) == 0).all()
    assert attention(q[:0], k[:0], v[:0]).shape == (0, 4, 6, 64)
    key_spans(1, 0, 5, device=DEV)
    assert _native.device_status(clear=True) == 0


def test_offsets_are_held_to_the_sequence():
    for words in (dict(documents=torch.tensor([-5, 1000, 3, 90], device=DEV)), dict(lengths=torch.tensor([5000], device=DEV)),
                  dict(lengths=torch.tensor([-3], device=DEV)), dict(documents=torch.tensor([300, 200, 100, 0], device=DEV)),
                  dict(documents=torch.tensor([0, 50], device=DEV), key_documents=torch.tensor([90, 2 ** 31 - 1], device=DEV))):
        spans = key_spans(1, 100, 200, causal=True, prefix=2 ** 31 - 1, **words)
        lo, hi = spans.rows[..., 0], spans.rows[..., 1]
        assert (lo >= 0).all() and (hi <= 200).all() and (lo <= hi).all()
        q, k, v = inputs(5, 1, 2, 2, 100, 200, 64)
        assert torch.isfinite(attention(q, k, v, spans=spans)).all()


def test_long_keys_split_over_ctas():
    for h, kv, n, m in ((2, 2, 3, 20000), (6, 1, 1, 70001), (1, 1, 200, 9000)):
        q, k, v = inputs(6, 1, h, kv, n, m, 128)
        spans, seen, pos = plan(1, n, m, lengths=[m - 77], causal=True)
        out, lse = attention(q, k, v, spans=spans, return_lse=True)
        check(q, k, v, out, lse, seen, pos)


def test_streams_and_capture():
    b, h, n = 1, 2, 260
    q, k, v = inputs(7, b, h, h, n, n, 64)
    ends = torch.tensor([0, 100, n], dtype=torch.int32, device=DEV)
    ref = attention(q, k, v, spans=key_spans(b, n, n, documents=ends))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attention(q, k, v, spans=key_spans(b, n, n, documents=ends))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ref)
    static, static_ends = torch.zeros_like(q), torch.zeros_like(ends)
    row, cache = q[:, :, :1].contiguous(), torch.randn(b, h, 5000, 64, device=DEV).to(torch.bfloat16)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = attention(static, k, v, spans=key_spans(b, n, n, documents=static_ends)), attention(row, cache, cache)
        graphs.append((graph, out))
    static.copy_(q)
    static_ends.copy_(ends)
    for _ in range(2):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out[0], ref) and torch.equal(out[1], attention(row, cache, cache))
    assert _native.device_status(clear=True) == 0
