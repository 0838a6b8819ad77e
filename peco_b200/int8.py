"""Linear layers of a transformer block in 8-bit integers, over libpeco_b200.so.

``quantize_rows`` rounds rows to 8-bit integers with one scale a row (for a
weight [N, K]: one an output channel); ``linear_int8`` computes

    out = residual + gate * act(sx sw (X W^T) + bias)

from 16-bit rows, which it quantises itself, or from quantised ones.  The
integer products run on the tcgen05 tensor cores at twice the 16-bit rate and
are exact; scales, bias, activation, gate and residual are applied in fp32 and
each output element is rounded once.  Inference only.

CUDA tensors only; work is enqueued on the current stream.
"""

from __future__ import annotations

import weakref
from typing import NamedTuple

import torch

from . import _native
from .linear import ACTIVATIONS, _gate_rows, _rows, _weight_rows, is_plain_linear

MAX_FEATURES = 131071  # 128 * 128 * K stays below 2^31
_SIXTEEN_BITS = (torch.float16, torch.bfloat16)


class QuantizedRows(NamedTuple):
    """Rows in 8-bit integers: row i stands for ``values[i] * scales[i]``."""

    values: torch.Tensor  # int8 [..., K]
    scales: torch.Tensor  # float32 [...]


def _no_gradient(what, *inputs):
    _native.refuse_tangents(what, *inputs)
    if torch.is_grad_enabled() and _native.wants_grad(*inputs):
        raise RuntimeError(f"{what} has no gradient; use torch.no_grad() or detached tensors")


def _joined(x, x2):
    """Checked feature counts of the rows [x | x2]."""
    if x.dtype not in _SIXTEEN_BITS or x2 is not None and x2.dtype is not x.dtype:
        raise TypeError("rows must be float16 or bfloat16 tensors of one dtype")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("Expected x [..., K]")
    if x2 is not None and (x2.dim() != x.dim() or x2.shape[:-1] != x.shape[:-1] or x2.shape[-1] < 1):
        raise ValueError("x2 must be [..., K2] with the leading shape of x")
    k, k2 = x.shape[-1], 0 if x2 is None else x2.shape[-1]
    if k + k2 > MAX_FEATURES:
        raise ValueError(f"rows of at most {MAX_FEATURES} features")
    return k, k2


def quantize_rows(x, x2=None) -> QuantizedRows:
    """Rows x [..., K] (and x2 [..., K2] beside them) in 8-bit integers.

    scale = max |x| / 127 over the whole row, values = 127 x / max |x| rounded
    to the nearest integer, ties to even, as of the exact quotient.  A row of
    zeros has scale 0; a row that holds an infinity or a NaN has scale NaN (and
    values 0), which makes every result computed from it NaN.  The values' rows
    are padded to multiples of 16 bytes, as ``linear_int8`` reads them in place.
    """
    _no_gradient("quantize_rows", x, x2)
    k, k2 = _joined(x, x2)
    _native.require_cuda(*(t for t in (x, x2) if t is not None))
    lead = x.shape[:-1]
    ld = -(-(k + k2) // 16) * 16
    values = torch.empty((*lead, ld), dtype=torch.int8, device=x.device)
    scales = torch.empty(lead, dtype=torch.float32, device=x.device)
    rows = scales.numel()
    if rows:
        x, x_step = _rows(x, k)
        x2, x2_step = _rows(x2, k2) if k2 else (None, 0)
        _native.enqueue(x.device, "peco_quantize_rows", _native.load().peco_quantize_rows,
                        (x.data_ptr(), x_step, _native.address(x2), x2_step, values.data_ptr(), ld, scales.data_ptr(),
                         rows, k, k2, _native.DTYPE_CODE[x.dtype]), (x, x2))
    return QuantizedRows(values[..., :k + k2], scales)


def _quantized(rows, what):
    if not isinstance(rows, tuple) or len(rows) != 2:
        raise TypeError(f"{what} must be QuantizedRows(values, scales)")
    values, scales = rows
    if not isinstance(values, torch.Tensor) or not isinstance(scales, torch.Tensor):
        raise TypeError(f"{what} must be QuantizedRows(values, scales)")
    if values.dtype is not torch.int8 or scales.dtype is not torch.float32:
        raise TypeError(f"{what} must have int8 values and float32 scales")
    shape = values.shape
    if not shape or shape[-1] < 1 or scales.shape != shape[:-1]:
        raise ValueError(f"{what} must have values [..., K] and scales [...] of one leading shape")
    return values, scales


def linear_int8(x, weight, bias=None, *, activation=None, gate=None, residual=None, x2=None, dtype=None):
    """residual + gate * act(scale_x scale_w ([x | x2] W^T) + bias) with 8-bit products.

    x [..., K] and the optional x2 [..., K2] in float16 or bfloat16, quantised
    here with one scale a row over both; or x as ``quantize_rows`` gives it
    (rows that several layers read are quantised once), with ``dtype`` the type
    of the result.  weight: ``QuantizedRows`` with values [N, K + K2] and a
    scale for each output channel, as ``quantize_rows(W)`` gives it.  bias [N],
    activation, gate and residual as in ``linear_act``, in the result's type.
    Row strides are free; 8-bit rows that do not start on 16-byte boundaries are
    copied first.  No gradient.
    """
    w_values, w_scales = _quantized(weight, "weight")
    given = isinstance(x, tuple)
    if given:
        values, scales = _quantized(x, "x")
        if x2 is not None:
            raise ValueError("x2 goes with 16-bit rows; quantize_rows(x, x2) quantises both together")
        if dtype not in _SIXTEEN_BITS:
            raise TypeError("quantised rows need dtype=torch.float16 or torch.bfloat16 for the result")
        if values.shape[-1] > MAX_FEATURES:
            raise ValueError(f"rows of at most {MAX_FEATURES} features")
        first, lead, k, k2 = values, values.shape[:-1], values.shape[-1], 0
    else:
        values = scales = None
        k, k2 = _joined(x, x2)
        if dtype is not None and dtype is not x.dtype:
            raise TypeError("the result of 16-bit rows has their dtype")
        first, lead, dtype = x, x.shape[:-1], x.dtype
    operands = (None if given else x, x2, values, scales, w_values, w_scales, bias, gate, residual)
    _no_gradient("linear_int8", *operands)
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(a for a in ACTIVATIONS if a)} or None, got {activation!r}")
    if w_values.dim() != 2 or w_values.shape[1] != k + k2 or w_values.shape[0] < 1:
        raise ValueError(f"weight values must be [N, {k + k2}] for these inputs, got {list(w_values.shape)}")
    n = w_values.shape[0]
    samples = 1
    if bias is not None:
        if bias.dtype is not dtype:
            raise TypeError("bias must have the result's dtype")
        if bias.shape != (n,):
            raise ValueError(f"bias must be [{n}]")
    if gate is not None:
        if gate.dtype is not dtype:
            raise TypeError("gate must have the result's dtype")
        if gate.shape != (n,):
            samples = lead[0] if len(lead) >= 2 else 1
            if tuple(gate.shape) not in ((samples, n), (samples, 1, n)):
                raise ValueError(f"gate must be [{n}] or one row for each of the {samples} samples, got {list(gate.shape)}")
    if residual is not None:
        if residual.dtype is not dtype:
            raise TypeError("residual must have the result's dtype")
        if residual.shape != (*lead, n):
            raise ValueError(f"residual must have the output's shape {[*lead, n]}")
    device = first.device
    if device.type != "cuda":
        _native.require_cuda(first)
    for t in operands:
        if t is not None and t.device != device:
            _native.require_cuda(first, t)
    out = torch.empty((*lead, n), dtype=dtype, device=device)
    rows = out.numel() // n
    if rows == 0:
        return out
    xp = x2p = vp = x_step = x2_step = v_step = bp = gp = g_step = rp = r_step = sp = 0
    if given:
        values, v_step = _rows(values, k)
        scales = scales.contiguous()
        vp, sp = values.data_ptr(), scales.data_ptr()
    else:
        x, x_step = _rows(x, k)
        xp = x.data_ptr()
        if k2:
            x2, x2_step = _rows(x2, k2)
            x2p = x2.data_ptr()
    w_values, w_step = _weight_rows(w_values)
    w_scales = w_scales.contiguous()
    if bias is not None:
        bias = bias.contiguous()
        bp = bias.data_ptr()
    if gate is not None:
        gate, g_step = _gate_rows(gate, n, samples)
        gp = gate.data_ptr()
    if residual is not None:
        residual, r_step = _rows(residual, n)
        rp = residual.data_ptr()
    lib = _native.load()
    wp, per, need, ws = w_values.data_ptr(), rows // samples, 0, 0
    # (quantised rows and weights on 16 bytes need no workspace)
    if not given or _off_16_bytes(vp | wp, v_step | w_step):
        need = int(lib.peco_linear_int8_workspace(0 if given else 1, vp, v_step, wp, w_step, samples, per, k, k2, n))
        space = torch.empty(need, dtype=torch.uint8, device=device)
        ws = space.data_ptr()
    _native.enqueue(device, "peco_linear_int8", lib.peco_linear_int8,
                    (xp, x_step, x2p, x2_step, vp, v_step, sp, wp, w_step, w_scales.data_ptr(), bp, gp, g_step, rp, r_step,
                     out.data_ptr(), n, samples, per, k, k2, n, act, _native.DTYPE_CODE[dtype], ws, need),
                    (None if given else x, x2, values, scales, w_values, w_scales, bias, gate, residual))
    return out


def _off_16_bytes(pointers: int, strides: int) -> bool:
    """Whether some rows of bytes may not start on 16 bytes."""
    return bool((pointers | strides) & 15)


class LayerInt8(NamedTuple):
    """A layer's weight in 8-bit integers, the parameter it was taken from, its storage, and its address and version then."""

    weight: QuantizedRows
    source: torch.Tensor
    place: object  # weak reference to the parameter's storage (whose address may be another's later); None: stale
    state: tuple

    def fresh(self) -> bool:
        return self.place is not None and self.place() is self.source.untyped_storage() and \
            self.state == _state(self.source)

    def __reduce__(self):  # a copied or stored layer's weight lies elsewhere and counts its versions anew
        return _layer_int8, (self.weight, self.source, self.fresh())


def _state(weight):
    return weight.data_ptr(), None if weight.is_inference() else weight._version  # (tensors of inference mode have none)


def _layer_int8(weight, source, fresh=True):
    return LayerInt8(weight, source, weakref.ref(source.untyped_storage()) if fresh else None, _state(source))


@torch.no_grad()
def quantize_layer(layer) -> bool:
    """Keep ``layer``'s weight in 8-bit integers beside it (``layer.int8``), where it is a plain linear layer on a CUDA
    device in 16 bits; whether it is.  The 16-bit weight stays the layer's parameter.  A layer whose weight is changed,
    replaced or moved afterwards raises until it is quantised again.  Values written in place through ``weight.data`` (as
    some ways of merging adapters do) leave no trace: quantise again after them."""
    if not is_plain_linear(layer) or layer.weight.dtype not in _SIXTEEN_BITS or not layer.weight.is_cuda or \
            not isinstance(getattr(layer, "int8", None), (LayerInt8, type(None))):  # (an attribute of somebody else's)
        return False
    layer.int8 = _layer_int8(quantize_rows(layer.weight), layer.weight)
    return True


def int8_weight(layer):
    """The 8-bit weight that ``quantize_layer`` keeps with ``layer``, or None."""
    kept = getattr(layer, "int8", None)
    if not isinstance(kept, LayerInt8) or not is_plain_linear(layer):
        return None
    if kept.source is not layer.weight or not kept.fresh():
        raise RuntimeError("the layer's weight changed or moved after it was quantised; quantise it again")
    return kept.weight
