"""What attention and its plans refuse before they look for a device, and their C entries' checks of arguments."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from peco_b200 import _native
from peco_b200.attention import KeySpans, attention, attention_backward, key_spans

Q = torch.zeros(2, 4, 6, 64, dtype=torch.bfloat16)
K = torch.zeros(2, 2, 9, 64, dtype=torch.bfloat16)
LSE = torch.zeros(2, 4, 6)
ROWS = KeySpans(torch.zeros(2, 6, 4, dtype=torch.int32), torch.zeros(2, 1, 4, dtype=torch.int32), 6, 9)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


@pytest.mark.parametrize("call,error", [
    (lambda: attention(Q[0], K, K), ValueError),
    (lambda: attention(Q.float(), K, K), TypeError),
    (lambda: attention(Q, K.half(), K), TypeError),
    (lambda: attention(Q, K[:1], K[:1]), ValueError),
    (lambda: attention(Q, K, K[:, :, :8]), ValueError),
    (lambda: attention(Q[:, :3], K, K), ValueError),
    (lambda: attention(Q, K[:, :0], K[:, :0]), ValueError),
    (lambda: attention(Q[..., :60], K[..., :60], K[..., :60]), ValueError),
    (lambda: attention(torch.zeros(1, 1, 2, 136).half(), torch.zeros(1, 1, 2, 136).half(), torch.zeros(1, 1, 2, 136).half()), ValueError),
    (lambda: attention(Q, K, K, scale=0.0), ValueError),
    (lambda: attention(Q, K, K, scale=-1.0), ValueError),
    (lambda: attention(Q, K, K, scale=float("nan")), ValueError),
    (lambda: attention(Q, K, K, softcap=0.0), ValueError),
    (lambda: attention(Q, K, K, softcap=float("inf")), ValueError),
    (lambda: attention(Q, K, K, slopes=torch.zeros(3)), ValueError),
    (lambda: attention(Q, K, K, slopes=torch.zeros(4).double()), ValueError),
    (lambda: attention(Q, K, K, slopes=torch.zeros(4, requires_grad=True)), RuntimeError),
    (lambda: attention(Q, K, K, spans=(ROWS.rows, ROWS.tiles)), TypeError),
    (lambda: attention(Q, K, K, spans=KeySpans(ROWS.rows, ROWS.tiles, 6, 8)), ValueError),
    (lambda: attention(Q, K, K, spans=KeySpans(ROWS.rows, ROWS.tiles, 5, 9)), ValueError),
    (lambda: attention(Q, K, K, spans=KeySpans(ROWS.rows[..., :3], ROWS.tiles, 6, 9)), ValueError),
    (lambda: attention(Q, K, K, spans=KeySpans(ROWS.rows, ROWS.tiles[:, :0], 6, 9)), ValueError),
    (lambda: attention(Q, K, K, spans=KeySpans(ROWS.rows.long(), ROWS.tiles, 6, 9)), ValueError),
    (lambda: attention(Q, K, K, spans=KeySpans(ROWS.rows.flip(2).transpose(1, 2).contiguous().transpose(1, 2), ROWS.tiles, 6, 9)), ValueError),
    (lambda: attention(torch.cat((Q, Q[:1])), torch.cat((K, K[:1])), torch.cat((K, K[:1])), spans=ROWS), ValueError),
    (lambda: attention(Q, K, K), RuntimeError),  # no CUDA device
    (lambda: attention_backward(Q[:, :, :5], Q, K, K, Q, LSE), ValueError),
    (lambda: attention_backward(Q.half(), Q, K, K, Q, LSE), TypeError),
    (lambda: attention_backward(Q, Q, K, K, Q[..., :32], LSE), ValueError),
    (lambda: attention_backward(Q, Q, K, K, Q, LSE[:, :, :5]), ValueError),
    (lambda: attention_backward(Q, Q, K, K, Q, LSE.double()), ValueError),
    (lambda: key_spans(0, 6, 9, device="cuda"), ValueError),
    (lambda: key_spans(65536, 6, 9, device="cuda"), ValueError),
    (lambda: key_spans(1, -1, 9, device="cuda"), ValueError),
    (lambda: key_spans(1, 6, 9, documents=[0, 6]), TypeError),
    (lambda: key_spans(1, 6, 9, documents=torch.zeros(2)), TypeError),
    (lambda: key_spans(1, 6, 9, documents=ints(0)), ValueError),
    (lambda: key_spans(3, 6, 9, documents=torch.zeros(2, 3, dtype=torch.int32)), ValueError),
    (lambda: key_spans(1, 6, 9, documents=ints(0, 6), key_documents=ints(0, 5, 9)), ValueError),
    (lambda: key_spans(1, 6, 9, key_documents=ints(0, 9)), ValueError),
    (lambda: key_spans(1, 6, 9, documents=ints(0, 6), lengths=ints(9)), ValueError),
    (lambda: key_spans(2, 6, 9, lengths=ints(9)), ValueError),
    (lambda: key_spans(1, 6, 9, lengths=torch.ones(1)), TypeError),
    (lambda: key_spans(1, 6, 9, prefix=3, device="cuda"), ValueError),
    (lambda: key_spans(1, 6, 9, causal=True, prefix=3, window=2, device="cuda"), ValueError),
    (lambda: key_spans(1, 6, 9, window=0, device="cuda"), ValueError),
    (lambda: key_spans(2, 6, 9, causal=True, prefix=ints(1, 2, 3)), ValueError),
    (lambda: key_spans(1, 6, 9, causal=True, prefix=torch.ones(1)), TypeError),
    (lambda: key_spans(1, 6, 9, documents=ints(0, 6)), RuntimeError),
    (lambda: key_spans(1, 6, 9, causal=True, device="cpu"), RuntimeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_needs_must_name_inputs():
    for needs in (["out"], ["q", "lse"]):
        with pytest.raises(ValueError, match="needs"):
            attention_backward(Q, Q, K, K, Q, LSE, needs=needs)


def test_tangents_are_refused():
    calls = [lambda d: attention(d(Q), K, K), lambda d: attention(Q, d(K), K), lambda d: attention(Q, K, d(K)),
             lambda d: attention_backward(d(Q), Q, K, K, Q, LSE), lambda d: attention_backward(Q, Q, K, K, d(Q), LSE)]
    with forward_ad.dual_level():
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))


def test_entries_check_their_arguments():
    lib = _native.load()
    at = 0x10000  # never read: every call is refused

    def spans(q=at, k=at, documents=1, lengths=0, window=0, batch=1, queries=6, keys=9, rows=at, tiles=at):
        return lib.peco_key_spans(q, 0, k, 0, documents, lengths, 0, 0, 0, 0, 1, window, batch, queries, keys, rows, tiles, 0)

    assert spans(batch=0) == 0 and spans(queries=0) == 0
    for bad in (dict(q=0), dict(k=0), dict(lengths=at), dict(window=-1), dict(batch=-1), dict(batch=65536), dict(queries=-1),
                dict(keys=-1), dict(documents=-1), dict(rows=0), dict(tiles=0), dict(rows=at + 8), dict(tiles=at + 4)):
        assert spans(**bad) == 1, bad

    def strides(n, **over):
        s = [4 * 6 * 64, 6 * 64, 64] * n
        for i, v in over.items():
            s[int(i[1:])] = v
        return (ctypes.c_longlong * (3 * n))(*s)

    def forward(q=at, k=at, v=at, st=None, rows=0, tiles=0, scale=1.0, cap=0.0, out=at, lse=at, batch=2, heads=4, kv=2, sq=6,
                sk=9, d=64, dtype=1, ws=0, n=0):
        return lib.peco_span_attention(q, k, v, st or strides(4), rows, tiles, 0, 0, scale, cap, out, lse, batch, heads, kv, sq,
                                       sk, d, dtype, ws, n, 0)

    assert forward(batch=0) == 0 and forward(sq=0) == 0
    for bad in (dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(lse=0), dict(rows=at), dict(tiles=at), dict(scale=0.0),
                dict(scale=float("nan")), dict(cap=-1.0), dict(heads=3), dict(kv=0), dict(d=60), dict(d=136), dict(sq=-1), dict(sk=-1),
                dict(q=at + 8), dict(st=strides(4, s2=60)), dict(st=strides(4, s4=-8)), dict(st=strides(4, s9=4))):
        assert forward(**bad) == 1, bad
    assert forward(dtype=2) == 20001
    assert lib.peco_span_attention_workspace(2, 4, 2, 6, 9, 64) == 0
    need = lib.peco_span_attention_workspace(1, 4, 2, 6, 9000, 64)
    assert need > 0 and lib.peco_span_attention_workspace(1, 4, 3, 6, 9, 64) == -1
    for bad in (dict(), dict(ws=at, n=need - 1), dict(ws=at + 8, n=need)):
        assert forward(batch=1, sk=9000, **bad) == 20005

    def backward(grad=at, q=at, k=at, v=at, out=at, lse=at, st=None, rows=0, scale=1.0, dq=at, dk=at, dv=at, heads=4, kv=2, sq=6,
                 sk=9, d=64, dtype=1, ws=at, n=1 << 20):
        return lib.peco_span_attention_backward(grad, q, k, v, out, lse, st or strides(8), rows, 0, 0, 0, scale, 0.0, dq, dk, dv, 2,
                                                heads, kv, sq, sk, d, dtype, ws, n, 0)

    assert backward(dq=0, dk=0, dv=0) == 0 and backward(sq=0, sk=0) == 0
    for bad in (dict(grad=0), dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(lse=0), dict(rows=at), dict(scale=-1.0),
                dict(heads=5), dict(d=4), dict(st=strides(8, s15=4)), dict(st=strides(8, s22=0))):
        assert backward(**bad) == 1, bad
    assert backward(dtype=2) == 20001
    need = lib.peco_span_attention_backward_workspace(2, 4, 2, 6, 9, 64, 0)
    assert need == 8 * 2 * 4 * 128
    for bad in (dict(ws=0), dict(n=need - 1), dict(ws=at + 8)):
        assert backward(**bad) == 20005
