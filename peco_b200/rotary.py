"""Rotary embedding by positions on several axes, over libpeco_b200.so.

A video token has a position on each of several axes (time, height, width);
the head dimension is cut into one section per axis and each section's pairs
turn by its axis's position.  ``rotate`` turns Q and K of an attention call in
one launch, without tables: the angles come from the token grid, or from
explicit positions, in 64 bits.  float16, bfloat16 and float32, any strides.
Differentiable (the gradient is the inverse turn).  CUDA tensors only; work is
enqueued on the current stream.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

_Strides = ctypes.c_longlong * 6
_Ints = [ctypes.c_int * i for i in range(5)]
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


@functools.lru_cache(maxsize=256)
def _sections(axes, d):
    """The checked section sizes as a C array."""
    sizes = tuple(int(a) for a in axes)
    if not 1 <= len(sizes) <= 4 or any(a < 0 or a % 2 for a in sizes) or sum(sizes) > d:
        raise ValueError("axes must be one to four even section sizes that fit the head dimension")
    return _Ints[len(sizes)](*sizes)


@functools.lru_cache(maxsize=256)
def _grid(grid, n_axes):
    """(the token grid as a C array, its number of tokens)."""
    sizes = tuple(int(s) for s in grid)
    if len(sizes) != n_axes or any(s < 0 for s in sizes):
        raise ValueError("grid must have one size per axis")
    return _Ints[n_axes](*sizes), math.prod(sizes)


def _run(q, k, axes, theta, grid, positions, interleaved, inverse, inplace):
    if not isinstance(q, torch.Tensor) or q.dim() != 4:
        raise ValueError("Expected q [B, H, N, D]")
    b, _, n, d = q.shape
    dtype, device = q.dtype, q.device
    code = _native.DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError("rotate takes float16, bfloat16 or float32 tensors")
    if k is not None:
        if k.dim() != 4 or (k.shape[0], k.shape[2], k.shape[3]) != (b, n, d):
            raise ValueError("q and k must agree in batch, tokens and head dimension")
        if k.dtype is not dtype:
            raise TypeError("q and k must have one dtype")
    if d % 2 or not 2 <= d <= 256:
        raise ValueError("the head dimension must be even and at most 256")
    sections = _sections(axes, d)
    a = len(sections)
    if not (theta > 0 and math.isfinite(theta)):
        raise ValueError("theta must be positive")
    if (grid is None) == (positions is None):
        raise ValueError("give either grid or positions")
    pos_p = pos_sb = pos_sn = pos_type = 0
    grid_c = None
    if grid is not None:
        grid_c, turned = _grid(grid, a)
    else:
        if positions.dtype not in _POSITION_TYPES:
            raise TypeError("positions must be int32, int64 or float32")
        if positions.dim() not in (2, 3) or positions.shape[-1] != a or \
                positions.dim() == 3 and positions.shape[0] not in (1, b):
            raise ValueError("positions must be [tokens, axes] or [B, tokens, axes]")
        turned = positions.shape[-2]
    if turned > n:
        raise ValueError(f"{turned} positions for {n} tokens")
    if device.type != "cuda":
        _native.require_cuda(q)
    for t in (k, positions):
        if t is not None and t.device != device:
            _native.require_cuda(q, t)
    if positions is not None:
        if positions.stride(-1) != 1 and a > 1:
            positions = positions.contiguous()
        pos_type, pos_sn = _POSITION_TYPES[positions.dtype], positions.stride(-2)
        pos_sb = positions.stride(0) if positions.dim() == 3 and positions.shape[0] > 1 else 0
        pos_p = positions.data_ptr()
        if turned == 0:
            pos_p, grid_c = 0, _grid((0,) * a, a)[0]
    q, q_out, q_args = _source(q, d, inplace)
    k_out, k_args = None, (0, 0, 0, None)
    if k is not None:
        k, k_out, k_args = _source(k, d, inplace)
        if inplace and _share_memory(q, k):
            raise ValueError("inplace would turn elements twice: q and k share memory")
    _native.enqueue(device, "peco_rotary", _native.load().peco_rotary,
                    (*q_args, *k_args, b, n, turned, d, sections, a, theta, grid_c, pos_p, pos_sb, pos_sn, pos_type,
                     1 if interleaved else 0, 1 if inverse else 0, code), (q, k, positions))
    if inplace:
        _native.wrote(q_out, *(() if k is None else (k_out,)))
    return q_out, k_out


def _share_memory(q, k) -> bool:
    """Whether q and k [B, H, N, D] (adjacent dimensions, no expanded axes) have an element in common."""
    if not q.numel() or not k.numel():
        return False
    (b, hq, n, d), hk, size = q.shape, k.shape[1], q.element_size()
    pq, pk, width = q.data_ptr(), k.data_ptr(), d * size
    (qb, qh, qn), (kb, kh, kn) = ([t.stride(i) * size for i in range(3)] for t in (q, k))
    if pq >= pk + (b - 1) * kb + (hk - 1) * kh + (n - 1) * kn + width or \
            pk >= pq + (b - 1) * qb + (hq - 1) * qh + (n - 1) * qn + width:
        return False
    if (b == 1 or qb == kb) and (hq == 1 or hk == 1 or qh == kh) and (n == 1 or qn == kn):
        # parts of one buffer: only the difference of two rows' batches and heads counts
        qs = (pq, n, qn, width)
        if hq > 1 and hk > 1 or hq == hk:
            places = {i * qb + j * qh for i in range(1 - b, b) for j in range(1 - hq, hk)}
        elif hq == 1:
            places = {i * qb + j * kh for i in range(1 - b, b) for j in range(hk)}
        else:
            places = {i * qb - j * qh for i in range(1 - b, b) for j in range(hq)}
        return any(_native.rows_overlap((pk + at, n, kn, width), qs) for at in places)
    return any(_native.rows_overlap((pq + i * qb + j * qh, n, qn, width), (pk + x * kb + y * kh, n, kn, width))
               for i in range(b) for j in range(hq) for x in range(b) for y in range(hk))


def _source(t, d, inplace):
    """(readable tensor, its output, the call's arguments for the two)."""
    st = t.stride()
    if st[3] != 1 and d > 1:
        if inplace:
            raise ValueError("inplace needs adjacent head dimensions and no expanded axes")
        t = t.contiguous()
        st = t.stride()
    if inplace:
        if any(s == 0 for s, m in zip(st, t.shape) if m > 1):
            raise ValueError("inplace needs adjacent head dimensions and no expanded axes")
        out, so = t, st
    else:
        out = torch.empty_like(t)  # keeps a dense layout (token-major views stay so)
        so = out.stride()
        if so[3] != 1:
            out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
            so = out.stride()
    return t, out, (t.data_ptr(), out.data_ptr(), t.shape[1], _Strides(st[0], st[1], st[2], so[0], so[1], so[2]))


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, options):
        ctx.options = options
        ctx.save_for_backward(positions)  # a change of them before the backward is an error
        ctx.set_materialize_grads(False)
        q, k = _run(q, k, positions=positions, **options, inplace=False)
        return q if k is None else (q, k)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        back = dict(ctx.options, inverse=not ctx.options["inverse"], positions=ctx.saved_tensors[0])
        gq, gk = (*grads, None)[:2]
        if gq is None and gk is None:
            return (None,) * 4
        if gq is None:
            gk, _ = _run(gk, None, **back, inplace=False)
        else:
            gq, gk = _run(gq, gk, **back, inplace=False)
        return gq, gk, None, None


def rotate(q, k=None, *, axes, theta=256.0, grid=None, positions=None, interleaved=True, inverse=False,
           inplace=False):
    """q [B, H, N, D] (and k [B, Hk, N, D], H and Hk free) turned by their tokens' positions.

    ``axes``: dimensions of each axis's section, in order, e.g. (16, 56, 56);
    dimensions after them are copied.  ``grid``: sizes of a row-major token
    grid that the first prod(grid) rows walk; or ``positions`` [N', axes] /
    [B, N', axes] (int32, int64 or float32; no gradient) of the first N' rows.  Later rows
    (the text) are copied.  ``interleaved``: pairs (2i, 2i+1), else one from
    each half of the rotated dimensions.  Angles are position * theta^(-2j/d).
    ``inverse``: the opposite turn.  ``inplace`` (not under autograd)
    overwrites q and k, which share no memory then.  Returns q, or (q, k).
    """
    _native.refuse_tangents("rotate", q, k, positions)
    if isinstance(positions, torch.Tensor) and positions.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("rotate has no gradient of positions; detach them")
    # fixed here: the backward turns by the same sections and grid
    options = dict(axes=tuple(axes), theta=theta, grid=None if grid is None else tuple(grid), interleaved=interleaved,
                   inverse=inverse)
    if torch.is_grad_enabled() and isinstance(q, torch.Tensor) and _native.wants_grad(q, k):
        if inplace:
            raise RuntimeError("rotate(inplace=True) does not record gradients; use torch.no_grad()")
        return _Rotate.apply(q, k, positions, options)
    q, k = _run(q, k, positions=positions, **options, inplace=inplace)
    return q if k is None else (q, k)


@dataclass(frozen=True)
class AxialPositions:
    """Rotary positions of a call's video rows, in place of (cos, sin) tables:
    the arguments of ``rotate`` that describe them.  The attention processor
    takes one as ``image_rotary_emb``."""

    axes: tuple
    theta: float = 256.0
    grid: Optional[tuple] = None
    positions: Optional[torch.Tensor] = None
    interleaved: bool = True

    @property
    def rows(self) -> int:
        """How many rows have positions."""
        return math.prod(self.grid) if self.grid is not None else self.positions.shape[-2]

    def checked(self, rows: int) -> "AxialPositions":
        """These positions, which have to be of exactly ``rows`` rows."""
        if self.rows != rows:
            raise ValueError(f"rotary positions of {self.rows} rows for {rows} video rows")
        return self

    def rotate(self, q, k=None, **options):
        return rotate(q, k, axes=self.axes, theta=self.theta, grid=self.grid, positions=self.positions,
                      interleaved=self.interleaved, **options)
