"""Linear layers of a transformer block with their epilogue, over libpeco_b200.so.

``linear_act``:  out = residual + gate * act([x | x2] W^T + bias), one kernel
launch for what a block otherwise runs as a concatenation, a matrix product, an
activation, a product with the adaLN gate and a residual sum.  The products run
on the tcgen05 tensor cores with fp32 sums and each output element is rounded
once; float16 and bfloat16.  Differentiable: under autograd the pre-activation
is saved (rounded to the operands' type) when a gradient needs it, and
``linear_act_backward`` computes the gradients with the same product kernel.

CUDA tensors only; work is enqueued on the current stream.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _native

ACTIVATIONS = {None: 0, "none": 0, "gelu_tanh": 1, "gelu": 2, "silu": 3}


class LinearGrads(NamedTuple):
    """Gradients of ``linear_act``; None where the input is absent or was not asked for."""

    x: Optional[torch.Tensor]
    x2: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]


def _flat(t: torch.Tensor) -> torch.Tensor:
    """[rows, features] view with adjacent features and one stride between rows
    (a copy where the layout has no such view)."""
    t = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    if t.stride(1) != 1 and t.shape[1] > 1 or t.stride(0) < t.shape[1] and t.shape[0] > 1:
        t = t.contiguous()
    return t


def _stride(t: Optional[torch.Tensor]) -> int:
    if t is None:
        return 0
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _check(x, weight, bias, gate, residual, x2, activation):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("x and weight must be torch tensors")
    dtype, device = x.dtype, x.device
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError("linear_act takes float16 or bfloat16 tensors of one dtype")
    for t in (weight, bias, gate, residual, x2):
        if t is not None and t.dtype is not dtype:
            raise TypeError("linear_act takes float16 or bfloat16 tensors of one dtype")
    if x.dim() < 1 or weight.dim() != 2:
        raise ValueError("Expected x [..., K] and weight [N, K + K2]")
    shape = x.shape
    n, wide = weight.shape
    k, k2 = shape[-1], 0
    if x2 is not None:
        k2 = x2.shape[-1]
        if x2.shape[:-1] != shape[:-1]:
            raise ValueError("x and x2 must have the same leading shape")
        if k2 < 1:
            raise ValueError("x2 must have at least one feature")
    if k < 1 or n < 1 or wide != k + k2:
        raise ValueError(f"weight must be [N, {k + k2}] for these inputs, got {list(weight.shape)}")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias must be [{n}]")
    samples = 1
    if gate is not None and gate.shape != (n,):
        samples = shape[0] if len(shape) >= 3 else 1
        if tuple(gate.shape) not in ((samples, n), (samples, 1, n)):
            raise ValueError(f"gate must be [{n}] or one row for each of the {samples} samples, got {list(gate.shape)}")
    if residual is not None and residual.shape != (*shape[:-1], n):
        raise ValueError(f"residual must have the output's shape {[*shape[:-1], n]}")
    if device.type != "cuda":
        _native.require_cuda(x)
    for t in (weight, bias, gate, residual, x2):
        if t is not None and t.device != device:
            _native.require_cuda(x, t)
    return k, k2, n, samples


def _gate_rows(gate, n):
    """The gate as [samples, N] with adjacent columns."""
    if gate is None:
        return None
    gate = gate.reshape(-1, n) if gate.dim() != 2 else gate
    return gate if gate.stride(1) == 1 or n == 1 else gate.contiguous()


def _forward(x, weight, bias, gate, residual, x2, activation, out, want_preact):
    k, k2, n, samples = _check(x, weight, bias, gate, residual, x2, activation)
    shape = (*x.shape[:-1], n)
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
    elif out.shape != shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError(f"out must be a {x.dtype} tensor of shape {list(shape)} on {x.device}")
    rows = out.numel() // n
    preact = torch.empty((rows, n), dtype=x.dtype, device=x.device) if want_preact else None
    if rows == 0:
        return out, preact
    try:
        out_rows = out.view(-1, n) if out.dim() != 2 else out
    except RuntimeError:
        out_rows = None
    if out_rows is None or out_rows.stride(1) != 1 and n > 1 or out_rows.stride(0) < n and rows > 1:
        raise ValueError("out must have adjacent columns and one stride between rows")
    xf, x2f, res = _flat(x), None if x2 is None else _flat(x2), None if residual is None else _flat(residual)
    w = weight if weight.stride(1) == 1 and weight.stride(0) >= weight.shape[1] else weight.contiguous()
    gates = _gate_rows(gate, n)
    bias = None if bias is None else bias.contiguous()
    lib = _native.load()
    dev, addr = x.device, _native.address
    operands = (addr(xf), _stride(xf), addr(x2f), _stride(x2f), addr(w), _stride(w))
    sizes = (samples, rows // samples, k, k2, n)
    need, ws = 0, None
    if (operands[0] | operands[2] | operands[4]) & 15 or (operands[1] | operands[3] | operands[5] | (k if k2 else 0)) & 7:
        # some operand may not start every row on 16 bytes
        need = int(lib.peco_linear_forward_workspace(*operands, *sizes))
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    _native.enqueue(dev, "peco_linear_forward", lib.peco_linear_forward,
                    (*operands, addr(bias), addr(gates), gates.stride(0) if samples > 1 else 0, addr(res), _stride(res),
                     out_rows.data_ptr(), _stride(out_rows), addr(preact), *sizes, ACTIVATIONS[activation],
                     _native.DTYPE_CODE[x.dtype], addr(ws), max(need, 0)), (xf, x2f, w, bias, gates, res, out))
    return out, preact


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate, residual, x2, activation):
        acts = ACTIVATIONS.get(activation, 0) != 0
        need = ctx.needs_input_grad
        through = need[0] or need[1] or need[2] or need[5]
        out, preact = _forward(x, weight, bias, gate, residual, x2, activation, None, need[3] or acts and through)
        ctx.activation, ctx.has_bias = activation, bias is not None
        ctx.save_for_backward(x, weight, gate, x2, preact)
        return out

    @staticmethod
    def backward(ctx, grad):
        x, weight, gate, x2, preact = ctx.saved_tensors
        need = ctx.needs_input_grad
        names = [n for n, i in (("x", 0), ("weight", 1), ("bias", 2), ("gate", 3), ("x2", 5)) if need[i]]
        g = LinearGrads(*[None] * 5)
        if names:
            g = linear_act_backward(grad, x, weight, preact=preact, activation=ctx.activation, gate=gate, x2=x2,
                                    bias=ctx.has_bias, needs=names)
        return g.x, g.weight, g.bias, g.gate, grad if need[4] else None, g.x2, None


def linear_act(x, weight, bias=None, *, activation=None, gate=None, residual=None, x2=None, out=None):
    """residual + gate * act([x | x2] W^T + bias).

    x [..., K] and the optional x2 [..., K2] (two inputs side by side, in place
    of their concatenation); weight [N, K + K2]; bias [N]; ``activation`` None,
    "gelu_tanh", "gelu" or "silu"; gate [N], or [B, N] / [B, 1, N] with one row
    for each sample of x [B, ..., K]; residual [..., N].  Row strides are free;
    operands whose rows do not start on 16-byte boundaries are copied first
    (keep odd-width weights in padded rows to avoid that).  ``out`` (not under
    autograd) receives the result and may be ``residual``.
    """
    inputs = (x, weight, bias, gate, residual, x2)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in inputs):
        if out is not None:
            raise RuntimeError("linear_act(out=...) does not record gradients; use torch.no_grad()")
        return _LinearAct.apply(x, weight, bias, gate, residual, x2, activation)
    return _forward(*inputs, activation, out, False)[0]


def linear_act_backward(grad, x, weight, *, preact=None, activation=None, gate=None, x2=None, bias=False, needs=None):
    """Gradients of ``linear_act`` for ``grad`` = d out (that of the residual is
    ``grad`` itself).

    ``preact`` [..., N], the saved pre-activation, is needed where the
    activation is not None or the gate's gradient is asked for.  ``bias``: the
    layer has one.  ``needs``: names of the gradients to compute (default: all
    of x, x2, weight, bias, gate that are there).
    """
    k, k2, n, samples = _check(x, weight, None, gate, grad, x2, activation)
    there = [name for name, t in (("x", x), ("x2", x2), ("weight", weight), ("bias", bias or None), ("gate", gate))
             if t is not None]
    needs = there if needs is None else list(needs)
    if any(name not in there for name in needs):
        raise ValueError(f"needs must name gradients among {there}, got {needs}")
    shapes = {"x": x.shape, "x2": None if x2 is None else x2.shape, "weight": weight.shape, "bias": (n,),
              "gate": None if gate is None else gate.shape}
    rows = grad.numel() // n
    if rows == 0:
        return LinearGrads(**{f: torch.zeros(shapes[f], dtype=x.dtype, device=x.device) if f in needs else None
                              for f in LinearGrads._fields})
    act = ACTIVATIONS[activation]
    if act or "gate" in needs:
        if preact is None:
            raise ValueError("this gradient needs the saved pre-activation (preact)")
        if preact.numel() != rows * n or preact.shape[-1] != n or preact.dtype != x.dtype:
            raise ValueError("preact must be the output-shaped pre-activation of the same dtype")
        _native.require_cuda(x, preact)
        preact = preact.reshape(rows, n).contiguous()
    else:
        preact = None
    outs = {f: torch.empty(shapes[f], dtype=x.dtype, device=x.device) if f in needs else None
            for f in LinearGrads._fields}
    g, xf, x2f, gates = _flat(grad), _flat(x), None if x2 is None else _flat(x2), _gate_rows(gate, n)
    w = weight if weight.stride(1) == 1 and weight.stride(0) >= weight.shape[1] else weight.contiguous()
    lib = _native.load()
    dev, addr = x.device, _native.address
    operands = (addr(xf), _stride(xf), addr(x2f), _stride(x2f), addr(w), _stride(w))
    sizes = (samples, rows // samples, k, k2, n, act)
    need = int(lib.peco_linear_backward_workspace(addr(g), _stride(g), *operands, *sizes, int(gate is not None)))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
    _native.enqueue(dev, "peco_linear_backward", lib.peco_linear_backward,
                    (addr(g), _stride(g), addr(preact), *operands, addr(gates), gates.stride(0) if samples > 1 else 0,
                     *(addr(outs[f]) for f in ("x", "x2", "weight", "bias", "gate")), *sizes,
                     _native.DTYPE_CODE[x.dtype], addr(ws), max(need, 0)), (g, preact, xf, x2f, w, gates))
    return LinearGrads(**outs)
