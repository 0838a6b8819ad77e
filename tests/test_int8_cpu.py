"""What the 8-bit linear layers refuse before they look for a device, and their C entries' checks of arguments."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from peco_b200 import _native
from peco_b200.int8 import QuantizedRows, linear_int8, quantize_rows

X = torch.zeros(2, 4, 16, dtype=torch.bfloat16)
W = QuantizedRows(torch.zeros(8, 16, dtype=torch.int8), torch.zeros(8))
Q = QuantizedRows(torch.zeros(2, 4, 16, dtype=torch.int8), torch.zeros(2, 4))


@pytest.mark.parametrize("call,error", [
    (lambda: quantize_rows(X.float()), TypeError),
    (lambda: quantize_rows(X, X.half()), TypeError),
    (lambda: quantize_rows(X, X[:1]), ValueError),
    (lambda: quantize_rows(X[..., :0]), ValueError),
    (lambda: quantize_rows(torch.zeros((), dtype=torch.bfloat16)), ValueError),
    (lambda: quantize_rows(torch.zeros(1, 131072, dtype=torch.bfloat16)), ValueError),
    (lambda: linear_int8(X, torch.zeros(8, 16)), TypeError),
    (lambda: linear_int8(X, QuantizedRows(W.values, W.scales.half())), TypeError),
    (lambda: linear_int8(X, QuantizedRows(W.values.float(), W.scales)), TypeError),
    (lambda: linear_int8(X, QuantizedRows(W.values, W.scales[:7])), ValueError),
    (lambda: linear_int8(X, QuantizedRows(W.values[:, :15], W.scales)), ValueError),
    (lambda: linear_int8(X, QuantizedRows(W.values[:0], W.scales[:0])), ValueError),
    (lambda: linear_int8(X, W, dtype=torch.float16), TypeError),
    (lambda: linear_int8(Q, W), TypeError),
    (lambda: linear_int8(Q, W, dtype=torch.float32), TypeError),
    (lambda: linear_int8(Q, W, x2=X, dtype=torch.bfloat16), ValueError),
    (lambda: linear_int8(X, W, activation="relu"), ValueError),
    (lambda: linear_int8(X, W, torch.zeros(8)), TypeError),
    (lambda: linear_int8(X, W, torch.zeros(7, dtype=torch.bfloat16)), ValueError),
    (lambda: linear_int8(X, W, gate=torch.zeros(3, 8, dtype=torch.bfloat16)), ValueError),
    (lambda: linear_int8(X, W, residual=torch.zeros(2, 4, 16, dtype=torch.bfloat16)), ValueError),
    (lambda: quantize_rows(X), RuntimeError),                 # no CUDA device
    (lambda: linear_int8(X, W), RuntimeError),
    (lambda: linear_int8(Q, W, dtype=torch.bfloat16), RuntimeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_gradients_and_tangents_are_refused():
    x = X.clone().requires_grad_()
    for call in (lambda t: quantize_rows(t), lambda t: linear_int8(t, W), lambda t: linear_int8(X, W, residual=t[..., :8])):
        with pytest.raises(RuntimeError, match="no gradient"):
            call(x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call(x)
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(X, torch.ones_like(X)))


def test_entries_check_their_arguments():
    lib = _native.load()
    at = 0x10000  # never read: every call is refused

    def linear(x=at, values=0, v_stride=0, rs=0, w=at, w_stride=16, cs=at, out=at, out_stride=8, k=16, k2=0, x_stride=16,
               n=8, act=0, dtype=1, ws=at, bytes_=1 << 20, rows=4):
        return lib.peco_linear_int8(x, x_stride, 0, 0, values, v_stride, rs, w, w_stride, cs, 0, 0, 0, 0, 0, out,
                                    out_stride, 1, rows, k, k2, n, act, dtype, ws, bytes_, 0)

    assert linear(rows=0) == 0
    for bad in (dict(x=0), dict(w=0), dict(cs=0), dict(out=0), dict(k=0), dict(k=131072), dict(n=0), dict(act=4),
                dict(act=-1), dict(w_stride=15), dict(out_stride=7), dict(x_stride=15), dict(k2=16),
                dict(values=at, v_stride=16), dict(values=at, v_stride=15, rs=at), dict(rows=-1)):
        assert linear(**bad) == 1, bad
    assert linear(dtype=2) == 20001
    for bad in (dict(ws=0), dict(bytes_=10), dict(ws=at + 8)):
        assert linear(**bad) == 20005
    assert linear(values=at + 1, v_stride=16, rs=at, ws=0) == 20005  # rows to be copied, and no room
    assert lib.peco_linear_int8_workspace(0, at, 16, at, 16, 1, 4, 16, 0, 8) == 0
    assert lib.peco_linear_int8_workspace(1, 0, 0, at, 16, 1, 4, 16, 0, 8) == 512
    assert lib.peco_linear_int8_workspace(0, at, 17, at + 1, 16, 1, 4, 16, 0, 8) == 512
    assert lib.peco_linear_int8_workspace(0, at, 16, at, 16, 1, 4, 131072, 0, 8) == -1

    def rows(x=at, x_stride=16, x2=0, values=at, v_stride=16, scales=at, n=4, k=16, k2=0, dtype=1):
        return lib.peco_quantize_rows(x, x_stride, x2, 16, values, v_stride, scales, n, k, k2, dtype, 0)

    assert rows(n=0) == 0
    for bad in (dict(x=0), dict(values=0), dict(scales=0), dict(k=0), dict(k2=8), dict(x_stride=15), dict(v_stride=15),
                dict(n=-1)):
        assert rows(**bad) == 1, bad
    assert rows(dtype=2) == 20001
