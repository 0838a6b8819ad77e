"""Attention over key spans by its definition in 64 bits, for the tests of the operators."""

import torch


def visible(batch, queries, keys, *, documents=None, key_documents=None, lengths=None, causal=False, prefix=0, window=None):
    """(mask [B, N, M], position [B, N]) from the words of the mask, a document at a time (host lists)."""
    seen = torch.zeros(batch, queries, keys, dtype=torch.bool)
    pos = torch.zeros(batch, queries, dtype=torch.int64)
    j = torch.arange(keys)
    for b in range(batch):
        if documents is not None:
            qe = documents[b] if isinstance(documents[0], (list, tuple)) else documents
            ke = qe if key_documents is None else key_documents[b] if isinstance(key_documents[0], (list, tuple)) else key_documents
            parts = [(qe[i], qe[i + 1], ke[i], ke[i + 1]) for i in range(len(qe) - 1)]
        else:
            parts = [(0, queries, 0, keys if lengths is None else lengths[b])]
        for n, (q0, q1, k0, k1) in enumerate(parts):
            early = prefix if isinstance(prefix, int) else prefix[b][n] if isinstance(prefix[0], (list, tuple)) else prefix[n]
            for i in range(q0, q1):
                at = k0 + (i - q0) + (k1 - k0) - (q1 - q0)
                pos[b, i] = at
                ok = (j >= k0) & (j < k1)
                if causal:
                    ok &= (j <= at) | (j < k0 + early)
                if window is not None:
                    ok &= (j - at).abs() < window
                seen[b, i] = ok
    return seen, pos


def scores(q, k, seen, pos, scale=None, softcap=None, slopes=None):
    """(z, tanh of the capped scores or None), masked keys at -inf; in the inputs' 64 bits, differentiable."""
    group = q.shape[1] // k.shape[1]
    raw = q @ k.repeat_interleave(group, 1).transpose(-1, -2) * (q.shape[-1] ** -0.5 if scale is None else scale)
    z = raw if softcap is None else softcap * torch.tanh(raw / softcap)
    if slopes is not None:
        apart = (pos[..., None] - torch.arange(k.shape[2], device=pos.device)).abs()
        z = z - slopes.to(z)[:, None, None] * apart[:, None]
    return torch.where(seen[:, None], z, -torch.inf)


def attend(q, k, v, seen, pos, **args):
    """(out, lse, probabilities) in 64 bits; rows without a visible key 0 and -inf."""
    z = scores(q, k, seen, pos, **args)
    lse = torch.logsumexp(z, -1, keepdim=True)
    p = torch.where(seen[:, None], torch.exp(z - torch.where(lse.isinf(), 0.0, lse)), 0.0)
    group = q.shape[1] // k.shape[1]
    return p @ v.repeat_interleave(group, 1), lse[..., 0], p


def score_size(q, k, seen, pos, scale=None, softcap=None, slopes=None):
    """Per row, the largest sum of magnitudes that its scores are made of (for rounding bounds)."""
    group = q.shape[1] // k.shape[1]
    size = q.abs() @ k.abs().repeat_interleave(group, 1).transpose(-1, -2) * (q.shape[-1] ** -0.5 if scale is None else scale)
    if slopes is not None:
        apart = (pos[..., None] - torch.arange(k.shape[2], device=pos.device)).abs()
        size = size + slopes.to(size)[:, None, None] * apart[:, None]
    size = torch.where(seen[:, None], size, 0.0).amax(-1, keepdim=True)
    return size if softcap is None else size + softcap
