"""Gated residual and norm between the parts of a transformer block, over libpeco_b200.so.

``modulated_norm``: one pass over the rows for what a block otherwise runs as
the branch's own norm, a product with the adaLN gate, the residual sum, a layer
or RMS norm and the shift / scale modulation:

    b = post_norm(branch) * post_weight
    r = residual_scale * x + gate * b
    h = norm(r) * weight * (1 + scale) + shift

Statistics and products are fp32; r and h are each rounded once.  float16 and
bfloat16, up to 16384 features.  Differentiable; nothing beyond the inputs is
saved.  CUDA tensors only; work is enqueued on the current stream.
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

NORMS = {None: 0, "none": 0, "layer": 1, "rms": 2}


class NormGrads(NamedTuple):
    """Gradients of ``modulated_norm``; None where the input is absent."""

    x: Optional[torch.Tensor]
    branch: Optional[torch.Tensor]
    gate: Optional[torch.Tensor]
    scale: Optional[torch.Tensor]
    shift: Optional[torch.Tensor]
    weight: Optional[torch.Tensor]
    post_weight: Optional[torch.Tensor]


def _rows(t, samples, rows, width):
    """(tensor, batch stride, row stride) of rows [samples, rows, width] with adjacent columns."""
    if t is None:
        return None, 0, 0
    if t.is_contiguous():
        return t, rows * width, width
    t = t.reshape(samples, rows, width) if t.dim() != 3 else t
    if t.stride(2) != 1 and width > 1:
        return t.contiguous(), rows * width, width
    return t, t.stride(0), t.stride(1)


def _vec(t, width):
    """(tensor, sample stride) of a vector [C] (stride 0) or [B, C] / [B, 1, C]."""
    if t is None:
        return None, 0
    if t.is_contiguous():
        return t, width if t.dim() > 1 else 0
    if t.stride(-1) != 1 and width > 1:
        t = t.contiguous()
    return t, t.stride(0) if t.dim() > 1 else 0


def _extent(x):
    """(samples, rows) of x: the leading axis of [B, ..., T, C] counts samples, [T, C] and [C] are one."""
    c = x.shape[-1]
    samples = x.shape[0] if x.dim() >= 3 else 1
    return samples, x.numel() // (c * samples) if samples else 0


def _check(x, branch, gate, scale, shift, weight, post_weight, norm, post_norm, eps, post_eps, residual_scale):
    if norm != "layer" and norm != "rms":
        raise ValueError(f'norm must be "layer" or "rms", got {norm!r}')
    post = NORMS.get(post_norm)
    if post is None:
        raise ValueError(f'post_norm must be None, "layer" or "rms", got {post_norm!r}')
    if not isinstance(x, torch.Tensor) or x.dim() < 1:
        raise TypeError("x must be a torch tensor [..., C]")
    dtype, device, shape = x.dtype, x.device, x.shape
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError("modulated_norm takes float16 or bfloat16 tensors of one dtype")
    if device.type != "cuda":
        _native.require_cuda(x)
    c = shape[-1]
    samples = shape[0] if len(shape) >= 3 else 1
    for t in (branch, gate, scale, shift, weight, post_weight):
        if t is not None:
            if t.dtype is not dtype:
                raise TypeError("modulated_norm takes float16 or bfloat16 tensors of one dtype")
            if t.device != device:
                _native.require_cuda(x, t)
    if not 1 <= c <= 16384:
        raise ValueError("modulated_norm takes 1 to 16384 features")
    if branch is None:
        if gate is not None or post or post_weight is not None:
            raise ValueError("gate, post_norm and post_weight need a branch")
    elif branch.shape != shape:
        raise ValueError("branch must have the shape of x")
    if post_weight is not None and not post:
        raise ValueError("post_weight needs a post_norm")
    for t in (gate, scale, shift):
        if t is not None:
            v = t.shape
            if v != (samples, c) and v != (c,) and v != (samples, 1, c):
                raise ValueError(f"gate, scale and shift must be [{c}] or one row for each of the {samples} samples, "
                                 f"got {list(v)}")
    for t in (weight, post_weight):
        if t is not None and t.shape != (c,):
            raise ValueError(f"weight and post_weight must be [{c}]")
    if not eps >= 0 or post_eps is not None and not post_eps >= 0 or not abs(residual_scale) < math.inf:
        raise ValueError("eps and post_eps must be nonnegative and residual_scale finite")


def _forward(x, branch, gate, scale, shift, weight, post_weight, norm, post_norm, eps, post_eps, residual_scale):
    _check(x, branch, gate, scale, shift, weight, post_weight, norm, post_norm, eps, post_eps, residual_scale)
    shape = x.shape
    c = shape[-1]
    normed = torch.empty_like(x, memory_format=torch.contiguous_format)
    residual = None
    samples = shape[0] if len(shape) >= 3 else 1
    size = x.numel()
    if size == 0:
        return (None if branch is None else torch.empty_like(normed)), normed
    rows = size // (c * samples)
    xp = xb = xr = bp = bb = br = gp = gb = sp = sb = tp = tb = wp = pp = rp = 0
    if x.is_contiguous():
        xb, xr = rows * c, c
    else:
        x, xb, xr = _rows(x, samples, rows, c)
    xp = x.data_ptr()
    if branch is not None:
        if branch.is_contiguous():
            bb, br = rows * c, c
        else:
            branch, bb, br = _rows(branch, samples, rows, c)
        bp = branch.data_ptr()
        residual = torch.empty_like(normed)
        rp = residual.data_ptr()
    if gate is not None:
        gate, gb = _vec(gate, c)
        gp = gate.data_ptr()
    if scale is not None:
        scale, sb = _vec(scale, c)
        sp = scale.data_ptr()
    if shift is not None:
        shift, tb = _vec(shift, c)
        tp = shift.data_ptr()
    if weight is not None:
        weight = weight.contiguous()
        wp = weight.data_ptr()
    if post_weight is not None:
        post_weight = post_weight.contiguous()
        pp = post_weight.data_ptr()
    _native.enqueue(x.device, "peco_gated_norm", _native.load().peco_gated_norm,
                    (xp, xb, xr, bp, bb, br, gp, gb, sp, sb, tp, tb, wp, pp, rp, normed.data_ptr(), samples, rows, c,
                     NORMS[norm], NORMS[post_norm], eps, eps if post_eps is None else post_eps, residual_scale,
                     _native.DTYPE_CODE[x.dtype]), (x, branch, gate, scale, shift, weight, post_weight))
    return residual, normed


class _ModulatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, gate, scale, shift, weight, post_weight, options):
        residual, normed = _forward(x, branch, gate, scale, shift, weight, post_weight, **options)
        ctx.options = options
        ctx.save_for_backward(x, branch, gate, scale, shift, weight, post_weight)
        ctx.set_materialize_grads(False)
        return normed if residual is None else (residual, normed)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        x = ctx.saved_tensors[0]
        dr, dh = grads if len(grads) == 2 else (None, grads[0])
        if dr is None and dh is None:
            return (None,) * 8
        if dh is None:
            dh = torch.zeros_like(x)
        names = [n for n, need in zip(NormGrads._fields, ctx.needs_input_grad) if need]
        g = modulated_norm_backward(dh, dr, *ctx.saved_tensors[:2],
                                    **dict(zip(NormGrads._fields[2:], ctx.saved_tensors[2:])), **ctx.options, needs=names)
        return (*g, None)


def modulated_norm(x, branch=None, *, gate=None, scale=None, shift=None, weight=None, post_weight=None, norm="layer",
                   post_norm=None, eps=1e-6, post_eps=None, residual_scale=1.0):
    """(r, h) of the module's formulas when there is a branch, h alone without one.

    x, branch [B, T, C] (or [T, C], one sample; any row and batch strides);
    gate, scale, shift [C] (one vector for all rows) or [B, C] / [B, 1, C];
    weight, post_weight [C].  ``norm`` / ``post_norm``: "layer" (mean and
    variance) or "rms"; ``post_eps`` defaults to ``eps``.  Absent parts drop out
    of the formulas.
    """
    _native.refuse_tangents("modulated_norm", x, branch, gate, scale, shift, weight, post_weight)
    if torch.is_grad_enabled() and _native.wants_grad(x, branch, gate, scale, shift, weight, post_weight):
        options = dict(norm=norm, post_norm=post_norm, eps=eps, post_eps=post_eps, residual_scale=residual_scale)
        return _ModulatedNorm.apply(x, branch, gate, scale, shift, weight, post_weight, options)
    residual, normed = _forward(x, branch, gate, scale, shift, weight, post_weight, norm, post_norm, eps, post_eps,
                                residual_scale)
    return normed if residual is None else (residual, normed)


def modulated_norm_backward(grad_normed, grad_residual, x, branch=None, *, gate=None, scale=None, shift=None,
                            weight=None, post_weight=None, norm="layer", post_norm=None, eps=1e-6, post_eps=None,
                            residual_scale=1.0, needs=None):
    """Gradients of ``modulated_norm`` for ``grad_normed`` = d h and
    ``grad_residual`` = d r (None: zero).  ``needs``: names of the gradients to
    compute (default: those of all inputs that are there)."""
    _native.refuse_tangents("modulated_norm_backward", grad_normed, grad_residual, x, branch, gate, scale, shift, weight,
                            post_weight)
    _check(x, branch, gate, scale, shift, weight, post_weight, norm, post_norm, eps, post_eps, residual_scale)
    if grad_normed is None:
        raise ValueError("grad_normed is required")
    shape, dtype, device = x.shape, x.dtype, x.device
    for t in (grad_normed, grad_residual):
        if t is not None:
            if t.shape != shape or t.dtype is not dtype:
                raise ValueError("grad_normed and grad_residual must have the shape and dtype of x")
            if t.device != device:
                _native.require_cuda(x, t)
    if grad_residual is not None and branch is None:
        raise ValueError("grad_residual needs a branch")
    inputs = (x, branch, gate, scale, shift, weight, post_weight)
    if needs is None:
        grads = [None if t is None else x.new_empty(t.shape) for t in inputs]
    else:
        needs = tuple(needs)  # looked through more than once
        if any(n not in NormGrads._fields or inputs[NormGrads._fields.index(n)] is None for n in needs):
            raise ValueError("needs names a gradient whose input is absent")
        grads = [x.new_empty(t.shape) if n in needs else None for n, t in zip(NormGrads._fields, inputs)]
    samples, rows = _extent(x)
    if samples * rows == 0:
        return NormGrads(*(None if g is None else g.zero_() for g in grads))
    c = shape[-1]
    gh, ghb, ghr = _rows(grad_normed, samples, rows, c)
    gr, grb, grr = _rows(grad_residual, samples, rows, c)
    x, xb, xr = _rows(x, samples, rows, c)
    branch, bb, br = _rows(branch, samples, rows, c)
    # a vector without a sample axis sums its gradient over the samples
    shared = (1 if gate is not None and gate.dim() == 1 else 0) | (2 if scale is not None and scale.dim() == 1 else 0) | \
        (4 if shift is not None and shift.dim() == 1 else 0)
    gate, gb = _vec(gate, c)
    scale, sb = _vec(scale, c)
    if weight is not None:
        weight = weight.contiguous()
    if post_weight is not None:
        post_weight = post_weight.contiguous()
    lib = _native.load()
    need, ws = 0, None
    if any(g is not None for g in grads[2:]):
        need = int(lib.peco_gated_norm_backward_workspace(samples, rows, c))
        ws = torch.empty(need, dtype=torch.uint8, device=device)
    addr = _native.address
    _native.enqueue(device, "peco_gated_norm_backward", lib.peco_gated_norm_backward,
                    (gh.data_ptr(), ghb, ghr, addr(gr), grb, grr, x.data_ptr(), xb, xr, addr(branch), bb, br, addr(gate),
                     gb, addr(scale), sb, addr(weight), addr(post_weight), addr(grads[0]), addr(grads[1]),
                     addr(grads[2]), addr(grads[3]), addr(grads[4]), shared, addr(grads[5]), addr(grads[6]), samples,
                     rows, c, NORMS[norm], NORMS[post_norm], eps, eps if post_eps is None else post_eps, residual_scale,
                     _native.DTYPE_CODE[dtype], addr(ws), need),
                    (gh, gr, x, branch, gate, scale, weight, post_weight))
    return NormGrads(*grads)
