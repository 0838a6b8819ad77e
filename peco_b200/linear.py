"""Linear layers of a transformer block with their epilogue, over libpeco_b200.so.

``linear_act``:  out = residual + gate * act([x | x2] W^T + bias), one kernel
launch for what a block otherwise runs as a concatenation, a matrix product, an
activation, a product with the adaLN gate and a residual sum.  The products run
on the tcgen05 tensor cores with fp32 sums and each output element is rounded
once; float16 and bfloat16.  Differentiable: under autograd the pre-activation
is saved (rounded to the operands' type) when a gradient needs it, and
``linear_act_backward`` computes the gradients with the same product kernel: for
its products grad * gate * act' is rounded to the operands' type, in float16 to
that type's range too (as unfused float16 layers do; scale the loss for it).

CUDA tensors only; work is enqueued on the current stream.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

_module = torch.nn.modules.module  # holds the hooks of all modules

ACTIVATIONS = {None: 0, "none": 0, "gelu_tanh": 1, "gelu": 2, "silu": 3}


class LinearGrads(NamedTuple):
    """Gradients of ``linear_act``; None where the input is absent or was not asked for."""

    x: Optional[torch.Tensor]
    x2: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    bias: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]


def _rows(t: torch.Tensor, width: int):
    """(tensor, elements between rows) of [..., width] rows with adjacent columns
    and one stride between rows; a copy where the layout has no such view."""
    if t.is_contiguous():
        return t, width
    f = t.reshape(-1, width) if t.dim() != 2 else t
    rows, step = f.shape[0], f.stride(0)
    if f.stride(1) != 1 and width > 1 or step < width and rows > 1:
        return f.contiguous(), width
    return f, max(step, width)


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


def _gate_rows(gate, n, samples):
    """(gate as rows of adjacent columns, elements between samples)."""
    if gate.is_contiguous():
        return gate, n if samples > 1 else 0
    gate = gate.reshape(-1, n)
    if gate.stride(1) != 1 and n > 1:
        gate = gate.contiguous()
    return gate, gate.stride(0) if samples > 1 else 0


def _weight_rows(weight):
    """(weight, elements between rows); rows may be padded."""
    step, inner = weight.stride()
    k = weight.shape[1]
    if (inner == 1 or k == 1) and step >= k:
        return weight, step
    return weight.contiguous(), k


def _check_out(out, operands):
    """Refuse an ``out`` (address in elements, rows, step, width) that shares memory with an operand, which other
    parts of the product may read after its first results are written; the residual's own rows alone may be it."""
    for name, t, rows, step, width in operands:
        if t is None:
            continue
        other = (t.data_ptr() // 2, rows, step, width)
        same_rows = other[0] == out[0] and (step == out[2] or rows == 1)
        if not (name == "residual" and same_rows) and _native.rows_overlap(out, other):
            raise ValueError(f"out shares memory with {name}")


def _misaligned(ptrs: int, strides: int) -> bool:
    """Whether some operand may not start every row on 16 bytes."""
    return bool(ptrs & 15 or strides & 7)


def _forward(x, weight, bias, gate, residual, x2, activation, out, want_preact):
    k, k2, n, samples = _check(x, weight, bias, gate, residual, x2, activation)
    shape = (*x.shape[:-1], n)
    given = out is not None
    if not given:
        out = out_rows = x.new_empty(shape)
        out_step = n
    else:
        if out.shape != shape or out.dtype != x.dtype or out.device != x.device:
            raise ValueError(f"out must be a {x.dtype} tensor of shape {list(shape)} on {x.device}")
        try:
            out_rows, out_step = out.view(-1, n) if out.numel() else out, n
        except RuntimeError:
            raise ValueError("out must have one stride between rows") from None
        if out.numel():
            if out_rows.stride(1) != 1 and n > 1 or out_rows.stride(0) < n and out_rows.shape[0] > 1:
                raise ValueError("out must have adjacent columns and rows apart")
            out_step = max(out_rows.stride(0), n)
    rows = out.numel() // n
    preact = x.new_empty((rows, n)) if want_preact else None
    if rows == 0:
        return out, preact
    x, x_step = _rows(x, k)
    weight, w_step = _weight_rows(weight)
    xp, wp, x2p, bp, gp, rp = x.data_ptr(), weight.data_ptr(), 0, 0, 0, 0
    x2_step = g_step = r_step = 0
    if x2 is not None:
        x2, x2_step = _rows(x2, k2)
        x2p = x2.data_ptr()
    if bias is not None:
        bias = bias.contiguous()
        bp = bias.data_ptr()
    if gate is not None:
        gate, g_step = _gate_rows(gate, n, samples)
        gp = gate.data_ptr()
    if residual is not None:
        residual, r_step = _rows(residual, n)
        rp = residual.data_ptr()
    if given:
        _check_out((out_rows.data_ptr() // 2, rows, out_step, n),
                   (("x", x, rows, x_step, k), ("x2", x2, rows, x2_step, k2), ("weight", weight, n, w_step, k + k2),
                    ("bias", bias, 1, n, n), ("gate", gate, samples if g_step else 1, g_step, n),
                    ("residual", residual, rows, r_step, n)))
    lib = _native.load()
    per, need, ws = rows // samples, 0, None
    if _misaligned(xp | wp | x2p, x_step | w_step | x2_step | (k if k2 else 0)):
        need = int(lib.peco_linear_forward_workspace(xp, x_step, x2p, x2_step, wp, w_step, samples, per, k, k2, n))
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need > 0 else None
    _native.enqueue(x.device, "peco_linear_forward", lib.peco_linear_forward,
                    (xp, x_step, x2p, x2_step, wp, w_step, bp, gp, g_step, rp, r_step, out_rows.data_ptr(), out_step,
                     _native.address(preact), samples, per, k, k2, n, ACTIVATIONS[activation],
                     _native.DTYPE_CODE[x.dtype], _native.address(ws), max(need, 0)),
                    (x, weight, bias, gate, residual, x2, out))
    if given:
        _native.wrote(out)
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
    @once_differentiable
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
    autograd) receives the result; it may be ``residual`` and may share no
    memory with the operands otherwise.
    """
    _native.refuse_tangents("linear_act", x, weight, bias, gate, residual, x2)
    if torch.is_grad_enabled() and _native.wants_grad(x, weight, bias, gate, residual, x2, out):
        if out is not None:
            raise RuntimeError("linear_act(out=...) does not record gradients; use torch.no_grad()")
        return _LinearAct.apply(x, weight, bias, gate, residual, x2, activation)
    return _forward(x, weight, bias, gate, residual, x2, activation, out, False)[0]


def linear_act_backward(grad, x, weight, *, preact=None, activation=None, gate=None, x2=None, bias=False, needs=None):
    """Gradients of ``linear_act`` for ``grad`` = d out (that of the residual is
    ``grad`` itself).

    ``preact`` [..., N], the saved pre-activation, is needed where the
    activation is not None or the gate's gradient is asked for.  ``bias``: the
    layer has one.  ``needs``: names of the gradients to compute (default: all
    of x, x2, weight, bias, gate that are there).
    """
    _native.refuse_tangents("linear_act_backward", grad, x, weight, preact, gate, x2)
    k, k2, n, samples = _check(x, weight, None, gate, grad, x2, activation)
    if needs is None:
        want_x, want_x2, want_w, want_b, want_g = True, x2 is not None, True, bool(bias), gate is not None
    else:
        needs = tuple(needs)  # looked through more than once
        want_x, want_x2, want_w, want_b, want_g = (name in needs for name in LinearGrads._fields)
        if len(set(needs) - set(LinearGrads._fields)) or want_x2 and x2 is None or want_b and not bias or \
                want_g and gate is None:
            raise ValueError(f"needs must name gradients of inputs that are there, got {list(needs)}")
    dx = x.new_empty(x.shape) if want_x else None
    dx2 = x.new_empty(x2.shape) if want_x2 else None
    dw = x.new_empty((n, k + k2)) if want_w else None
    db = x.new_empty((n,)) if want_b else None
    dg = x.new_empty(gate.shape) if want_g else None
    rows = grad.numel() // n
    if rows == 0:
        return LinearGrads(*(None if t is None else t.zero_() for t in (dx, dx2, dw, db, dg)))
    act = ACTIVATIONS[activation]
    preact_p = 0
    if act or want_g:
        if preact is None:
            raise ValueError("this gradient needs the saved pre-activation (preact)")
        if preact.numel() != rows * n or preact.shape[-1] != n or preact.dtype != x.dtype:
            raise ValueError("preact must be the output-shaped pre-activation of the same dtype")
        if preact.device != x.device:
            _native.require_cuda(x, preact)
        preact = preact.contiguous()
        preact_p = preact.data_ptr()
    else:
        preact = None
    grad, grad_step = _rows(grad, n)
    x, x_step = _rows(x, k)
    x2p = x2_step = gp = g_step = 0
    if x2 is not None:
        x2, x2_step = _rows(x2, k2)
        x2p = x2.data_ptr()
    if gate is not None:
        gate, g_step = _gate_rows(gate, n, samples)
        gp = gate.data_ptr()
    weight, w_step = _weight_rows(weight)
    lib = _native.load()
    addr = _native.address
    grad_p = grad.data_ptr()
    operands = (x.data_ptr(), x_step, x2p, x2_step, weight.data_ptr(), w_step)
    sizes = (samples, rows // samples, k, k2, n, act)
    need = int(lib.peco_linear_backward_workspace(grad_p, grad_step, *operands, *sizes, 1 if gp else 0))
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need > 0 else None
    _native.enqueue(x.device, "peco_linear_backward", lib.peco_linear_backward,
                    (grad_p, grad_step, preact_p, *operands, gp, g_step, addr(dx), addr(dx2), addr(dw), addr(db),
                     addr(dg), *sizes, _native.DTYPE_CODE[x.dtype], addr(ws), max(need, 0)),
                    (grad, preact, x, x2, weight, gate))
    return LinearGrads(dx, dx2, dw, db, dg)


def without_hooks(module) -> bool:
    """Whether calling ``module`` runs its class's ``forward`` and nothing else."""
    return "forward" not in vars(module) and not (
        module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks
        or _module._global_forward_hooks or _module._global_forward_pre_hooks or _module._global_backward_hooks
        or _module._global_backward_pre_hooks)


def is_plain_linear(layer) -> bool:
    """Whether ``linear_act(x, layer.weight, layer.bias)`` stands for ``layer(x)``:
    an ``nn.Linear`` itself, or a class that says ``plain_linear`` of itself (not of
    its subclasses), with an ordinary weight and no hooks.  Wrapped, adapted,
    quantised and observed layers are to be called."""
    kind = type(layer)
    return (kind is torch.nn.Linear or vars(kind).get("plain_linear") is True) and \
        type(layer.weight) in (torch.nn.Parameter, torch.Tensor) and without_hooks(layer)
