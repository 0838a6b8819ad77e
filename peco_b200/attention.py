"""Exact attention under masks of key spans, over libpeco_b200.so.

Each query row sees one interval of keys, which covers the documents of a packed
sequence, a causal order with a prefix that every row sees, windows, and
samples of unequal lengths (``key_spans``).  Scores can be capped by a tanh and
get a bias that depends on the distance:

    z_ij = cap tanh(scale q_i.k_j / cap) - slope_h |pos_i - j|
    out_i = sum_j softmax_j(z_ij) v_j      over the keys that row i sees

Products run on the tcgen05 tensor cores with fp32 sums, softmax statistics in
fp32; float16 and bfloat16; keys may be shared by groups of query heads.  A row
that sees no key is 0.  Differentiable.  CUDA tensors only; work is enqueued on
the current stream.
"""

from __future__ import annotations

import functools
import struct
from dataclasses import dataclass
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

_strides = struct.Struct("=12q").pack  # (quicker to make than an array of ctypes)
_grad_strides = struct.Struct("=24q").pack
_SIXTEEN_BITS = (torch.float16, torch.bfloat16)
_LEAST, _MOST = 1e-30, 1e30  # scale and cap reach the kernels in fp32, their quotient too


class AttentionGrads(NamedTuple):
    """Gradients of ``attention``; None where not asked for."""

    q: Optional[torch.Tensor]
    k: Optional[torch.Tensor]
    v: Optional[torch.Tensor]


@dataclass(frozen=True)
class KeySpans:
    """The keys that each query row sees, as ``key_spans`` lays them out."""

    rows: torch.Tensor   # int32 [B or 1, queries, 4]: first key, key behind the last, the row's position among the keys;
                         # of the first rows also the tiles of 128 rows, those that see most keys first
    tiles: torch.Tensor  # int32 [B or 1, tiles of 128 rows, 4]
    queries: int
    keys: int


def _int32(t):
    """Counts as contiguous int32; larger ones held to its range."""
    return t.contiguous() if t.dtype is torch.int32 else t.clamp(-1, 2 ** 31 - 1).to(torch.int32)


def _ends(ends, batch, what):
    """Document ends as int32 [1 or batch, n + 1] rows."""
    if not isinstance(ends, torch.Tensor) or ends.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what} must be an int32 or int64 tensor")
    if ends.dim() not in (1, 2) or ends.shape[-1] < 2 or ends.dim() == 2 and ends.shape[0] not in (1, batch):
        raise ValueError(f"{what} must be [n + 1] or one such row for each of the {batch} samples")
    ends = _int32(ends)
    return ends, ends.shape[1] if ends.dim() == 2 and ends.shape[0] > 1 else 0


def key_spans(batch, queries, keys, *, documents=None, key_documents=None, lengths=None, causal=False, prefix=None,
              window=None, device=None) -> KeySpans:
    """Spans of keys for ``queries`` rows and ``keys`` keys of ``batch`` samples (1: the same for all samples of a call).

    ``documents``: ends of a packed sequence's documents, int [n + 1] or
    [batch, n + 1], ascending from the first row: document i holds rows
    [documents[i], documents[i + 1]) and, with ``key_documents`` (default: the
    same), those keys; its rows see its keys only.  Rows outside all documents
    see nothing.  ``lengths``: int [batch], each sample's number of keys, instead
    of documents.  The last row of a document (or sample) stands at its last key.
    ``causal``: a row sees the keys up to its own position, and the first
    ``prefix`` keys of its document wherever it stands (an int, or an int tensor
    [n], [batch, 1] or [batch, n]).  ``window``: a row sees the keys less
    than ``window`` away from its position (not with a prefix).

    Offsets are read on the device and held to the sequence there; nothing is
    synchronised.  A plan serves every layer that has the same mask.
    """
    batch, queries, keys = int(batch), int(queries), int(keys)
    if batch < 1 or batch > 65535 or queries < 0 or keys < 0:
        raise ValueError("Expected a batch of 1 to 65535 and nonnegative lengths")
    if lengths is not None and documents is not None:
        raise ValueError("lengths and documents exclude each other")
    if key_documents is not None and documents is None:
        raise ValueError("key_documents goes with documents")
    if prefix is not None and not causal:
        raise ValueError("a prefix goes with a causal order")
    if window is not None and (int(window) < 1 or prefix is not None):
        raise ValueError("window must be positive and has no prefix")
    tensors, n = [], 0
    q_ends = k_ends = None
    q_stride = k_stride = 0
    if documents is not None:
        q_ends, q_stride = _ends(documents, batch, "documents")
        k_ends, k_stride = (q_ends, q_stride) if key_documents is None else _ends(key_documents, batch, "key_documents")
        n = q_ends.shape[-1] - 1
        if k_ends.shape[-1] != n + 1:
            raise ValueError("documents and key_documents must have as many documents")
        tensors += [q_ends, k_ends]
    elif lengths is not None:
        if not isinstance(lengths, torch.Tensor) or lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError("lengths must be an int32 or int64 tensor")
        if lengths.shape != (batch,):
            raise ValueError(f"lengths must be [{batch}]")
        lengths = _int32(lengths)
        tensors.append(lengths)
    prefix_rows, prefix_all, prefix_batch, prefix_doc = None, 0, 0, 0
    if isinstance(prefix, torch.Tensor):
        if prefix.dtype not in (torch.int32, torch.int64):
            raise TypeError("prefix must be an int or an int32 or int64 tensor")
        shape = tuple(prefix.shape)
        if shape not in ((max(n, 1),), (batch, 1), (batch, max(n, 1))):
            raise ValueError(f"prefix must be one number, [{max(n, 1)}], [{batch}, 1] or [{batch}, {max(n, 1)}]")
        prefix_rows = _int32(prefix)
        prefix_batch, prefix_doc = (shape[1] if len(shape) == 2 else 0), 1 if shape[-1] > 1 else 0
        tensors.append(prefix_rows)
    elif prefix is not None:
        prefix_all = min(max(int(prefix), 0), 2 ** 31 - 1)
    if device is None:
        device = tensors[0].device if tensors else torch.device("cuda", torch.cuda.current_device())
    elif not isinstance(device, torch.device) or device.type == "cuda" and device.index is None:
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
    if device.type != "cuda":
        raise RuntimeError("peco_b200 runs on CUDA devices only; got " + str(device))
    for t in tensors:
        if t.device != device:
            raise ValueError("all tensors must be on the same CUDA device")
    rows = torch.empty((batch, queries, 4), dtype=torch.int32, device=device)
    tiles = torch.empty((batch, -(-queries // 128), 4), dtype=torch.int32, device=device)
    address = _native.address
    _native.enqueue(device, "peco_key_spans", _native.load().peco_key_spans,
                    (address(q_ends), q_stride, address(k_ends), k_stride, n, address(lengths), address(prefix_rows),
                     prefix_batch, prefix_doc, prefix_all, 1 if causal else 0,
                     min(int(window), 2 ** 31 - 1) if window is not None else 0, batch, queries, keys, rows.data_ptr(),
                     tiles.data_ptr()), tensors)
    return KeySpans(rows, tiles, queries, keys)


def _check(q, k, v, spans, scale, softcap, slopes):
    """Checked (batch, heads, key heads, queries, keys, dims), scale and cap."""
    if not (isinstance(q, torch.Tensor) and isinstance(k, torch.Tensor) and isinstance(v, torch.Tensor)
            and q.dim() == 4 and k.dim() == 4):
        raise ValueError("Expected q [B, H, N, D] and k, v [B, KV, M, D]")
    dtype = q.dtype
    if dtype not in _SIXTEEN_BITS or k.dtype is not dtype or v.dtype is not dtype:
        raise TypeError("attention takes float16 or bfloat16 tensors of one dtype")
    b, h, n, d = q.shape
    shape = k.shape
    kv, m = shape[1], shape[2]
    if shape[0] != b or shape[3] != d or v.shape != shape:
        raise ValueError("k and v must be [B, KV, M, D] with the batch and head dimension of q")
    if kv < 1 or h < 1 or h % kv:
        raise ValueError("the query heads must be a multiple of the key heads")
    if d < 8 or d > 128 or d % 8:
        raise ValueError("the head dimension must be a multiple of 8 up to 128")
    if n > 0x7ffffe00 or m > 0x7ffffe00:
        raise ValueError("too many rows")
    scale = d ** -0.5 if scale is None else float(scale)
    if not (_LEAST <= scale <= _MOST):
        raise ValueError("scale must be positive, from 1e-30 to 1e30")
    cap = 0.0
    if softcap is not None:
        cap = float(softcap)
        if not (_LEAST <= cap <= _MOST and scale / cap <= _MOST):
            raise ValueError("softcap must be positive, from 1e-30 to 1e30 (scale / softcap at most 1e30)")
    if slopes is not None:
        if not isinstance(slopes, torch.Tensor) or slopes.dtype is not torch.float32 or slopes.shape != (h,):
            raise ValueError(f"slopes must be a float32 tensor [{h}]")
    if spans is not None:
        if not isinstance(spans, KeySpans):
            raise TypeError("spans must come from key_spans")
        if spans.queries != n or spans.keys != m or spans.rows.shape[0] not in (1, b):
            raise ValueError(f"spans are for {spans.rows.shape[0]} samples of {spans.queries} rows and {spans.keys} keys, "
                             f"the call has {b} of {n} and {m}")
        samples = spans.rows.shape[0]
        if spans.rows.shape != (samples, n, 4) or spans.tiles.shape != (samples, -(-n // 128), 4) or \
                spans.rows.dtype is not torch.int32 or spans.tiles.dtype is not torch.int32 or \
                not spans.rows.is_contiguous() or not spans.tiles.is_contiguous() or \
                (spans.rows.data_ptr() | spans.tiles.data_ptr()) & 15:
            raise ValueError("spans must be as key_spans lays them out")
    return (b, h, kv, n, m, d), scale, cap


def _refuse_slopes_gradient(slopes):
    """Where grad mode is still the caller's: a Function's forward runs without."""
    if isinstance(slopes, torch.Tensor) and slopes.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("attention has no gradient of slopes")


def _on_one_device(q, *others):
    """The inputs' CUDA device."""
    device = q.device
    if device.type != "cuda":
        _native.require_cuda(q)
    for t in others:
        if t is not None and t.device != device:
            _native.require_cuda(q, t)
    return device


def _in_place(t) -> bool:
    """Whether the kernels can read and write ``t`` as it lies: dims adjacent, every row, head and sample on 16 bytes."""
    if t.data_ptr() & 15:
        return False
    if t.is_contiguous():
        return True
    steps = t.stride()
    return steps[3] == 1 and all(n <= 1 or 0 < s < 1 << 38 and s % 8 == 0 for n, s in zip(t.shape[:3], steps[:3]))


def _readable(t):
    """``t``, or a copy of a layout that the kernels can read."""
    return t if _in_place(t) else t.clone(memory_format=torch.contiguous_format)


def _mask_args(spans, b):
    if spans is None:
        return 0, 0, 0
    return spans.rows.data_ptr(), spans.tiles.data_ptr(), 1 if spans.rows.shape[0] == b and b > 1 else 0


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes) -> int:
    return int(_native.load().peco_span_attention_workspace(*sizes))


def _forward(q, k, v, spans, scale, softcap, slopes):
    (b, h, kv, n, m, d), scale, cap = _check(q, k, v, spans, scale, softcap, slopes)
    mask = (None, None) if spans is None else (spans.rows, spans.tiles)
    device = _on_one_device(q, k, v, slopes, *mask)
    out = torch.empty_like(q)
    lse = torch.empty((b, h, n), dtype=torch.float32, device=device)
    if b == 0 or n == 0:
        return out, lse
    q, k, v, whole = _readable(q), _readable(k), _readable(v), out
    if not _in_place(out):
        whole = torch.empty(q.shape, dtype=q.dtype, device=device)
    if slopes is not None:
        slopes = slopes.contiguous()
    lib = _native.load()
    need = _workspace_bytes(b, h, kv, n, m, d)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    strides = _strides(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *whole.stride()[:3])
    rows, tiles, batched = _mask_args(spans, b)
    _native.enqueue(device, "peco_span_attention", lib.peco_span_attention,
                    (q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, rows, tiles, batched, _native.address(slopes), scale,
                     cap, whole.data_ptr(), lse.data_ptr(), b, h, kv, n, m, d, _native.DTYPE_CODE[q.dtype],
                     _native.address(ws), max(need, 0)), (q, k, v, slopes, *mask))
    return out.copy_(whole) if whole is not out else out, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, spans, scale, softcap, slopes):
        out, lse = _forward(q, k, v, spans, scale, softcap, slopes)
        ctx.sizes, ctx.scores = (spans.queries, spans.keys) if spans is not None else None, (scale, softcap)
        mask = (spans.rows, spans.tiles) if spans is not None else (None, None)
        ctx.save_for_backward(q, k, v, out, lse, slopes, *mask)  # (changing any of them meanwhile is an error)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _):
        q, k, v, out, lse, slopes, rows, tiles = ctx.saved_tensors
        spans = KeySpans(rows, tiles, *ctx.sizes) if ctx.sizes is not None else None
        scale, softcap = ctx.scores
        names = [n for n, need in zip("qkv", ctx.needs_input_grad) if need]
        g = attention_backward(grad, q, k, v, out, lse, spans=spans, scale=scale, softcap=softcap, slopes=slopes, needs=names)
        return g.q, g.k, g.v, None, None, None, None


def attention(q, k, v, *, spans=None, scale=None, softcap=None, slopes=None, return_lse=False):
    """Attention of q [B, H, N, D] over k, v [B, KV, M, D] (H a multiple of KV: each key head serves H / KV query heads).

    ``spans``: what ``key_spans(B or 1, N, M, ...)`` gives; None: every row sees
    every key, and the last row stands at the last key.  ``scale`` defaults to
    D^-0.5.  ``softcap``: scores are softcap * tanh(score / softcap); it, ``scale`` and
    scale / softcap stay inside fp32 (1e-30 to 1e30).  ``slopes`` float32 [H]:
    slope * |position - j| is taken from the score of key j (no gradient of
    slopes: such a call is refused).
    ``return_lse``: also the logarithm of each row's sum of exponentials, float32
    [B, H, N] (no gradient flows through it), -inf where a row sees nothing.

    Scores are fp32 with its rounding, 2^-23 of their size, which is the relative
    error of a probability.  Past 2^26 (uncapped) a row may be infinite or NaN.

    D is a multiple of 8 up to 128.  Strides are free where D is adjacent and
    rows, heads and samples start on 16 bytes; other layouts are copied first.
    The result has the layout of q.  Keys and values that a row's mask leaves
    out do not reach its result, whatever they hold.
    """
    _native.refuse_tangents("attention", q, k, v, slopes)
    _refuse_slopes_gradient(slopes)
    if torch.is_grad_enabled() and _native.wants_grad(q, k, v):
        out, lse = _Attention.apply(q, k, v, spans, scale, softcap, slopes)
    else:
        out, lse = _forward(q, k, v, spans, scale, softcap, slopes)
    return (out, lse) if return_lse else out


def attention_backward(grad, q, k, v, out, lse, *, spans=None, scale=None, softcap=None, slopes=None, needs=None):
    """Gradients of ``attention`` for ``grad`` = d out, with the call's results ``out`` and ``lse``.

    ``needs``: names of the gradients to compute (default: q, k and v).  The
    probabilities and their gradients are rounded to the operands' type for the
    products (in float16 to that type's range too: scale the loss for it); sums
    run in a fixed order.  A row that sees one key has no gradient of its score
    (q's and k's are exact zeros); rows of up to eight keys take grad.out from
    their probabilities, others from ``out`` as it is rounded.  Probabilities
    come from ``lse``, whose rounding is 2^-23 of its size: scores past some 2^16
    leave little of them.  Rows that see no key, and keys that no row sees, get
    zeros and may hold anything; a NaN in a row or key that is seen reaches
    the gradients of its tile.
    """
    _native.refuse_tangents("attention_backward", grad, q, k, v, out, slopes)
    _refuse_slopes_gradient(slopes)
    sizes, scale, cap = _check(q, k, v, spans, scale, softcap, slopes)
    b, h, kv, n, m, d = sizes
    for name, t in (("grad", grad), ("out", out)):
        if not isinstance(t, torch.Tensor) or t.shape != q.shape:
            raise ValueError(f"{name} must have the shape of q")
        if t.dtype is not q.dtype:
            raise TypeError(f"{name} must have the dtype of q")
    if not isinstance(lse, torch.Tensor) or lse.dtype is not torch.float32 or lse.shape != (b, h, n):
        raise ValueError(f"lse must be a float32 tensor {[b, h, n]}")
    needs = ("q", "k", "v") if needs is None else tuple(needs)
    if set(needs) - {"q", "k", "v"}:
        raise ValueError(f"needs must name gradients of q, k and v, got {list(needs)}")
    mask = (None, None) if spans is None else (spans.rows, spans.tiles)
    device = _on_one_device(q, k, v, grad, out, lse, slopes, *mask)
    given = {"q": q, "k": k, "v": v}
    made = {name: torch.empty_like(t) for name, t in given.items() if name in needs}
    if not made:
        return AttentionGrads(None, None, None)
    # results whose layout TMA could not read are made elsewhere and copied
    whole = {name: t if t.numel() == 0 or _in_place(t) else torch.empty(t.shape, dtype=t.dtype, device=device)
             for name, t in made.items()}
    if b and (n or m):
        grad, q, k, v, out = (t if t.numel() == 0 else _readable(t) for t in (grad, q, k, v, out))
        lse = lse.contiguous()
        if slopes is not None:
            slopes = slopes.contiguous()
        lib = _native.load()
        need = int(lib.peco_span_attention_backward_workspace(b, h, kv, n, m, d, 0 if spans is None else 1))
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
        to = [whole.get(name) for name in "qkv"]
        strides = _grad_strides(*(s for t in (grad, q, k, v, out, *to) for s in (t.stride()[:3] if t is not None else (0, 0, 0))))
        rows, tiles, batched = _mask_args(spans, b)
        _native.enqueue(device, "peco_span_attention_backward", lib.peco_span_attention_backward,
                        (grad.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), strides,
                         rows, tiles, batched, _native.address(slopes), scale, cap, *(_native.address(t) for t in to), b, h,
                         kv, n, m, d, _native.DTYPE_CODE[q.dtype], _native.address(ws), max(need, 0)),
                        (grad, q, k, v, out, lse, slopes, *mask))
    for name, t in made.items():
        if whole[name] is not t:
            t.copy_(whole[name])
    return AttentionGrads(*(made.get(name) for name in "qkv"))
