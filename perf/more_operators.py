"""Cases of the 8-bit linear layers and of attention under masks, and their plain forms.

Three operators that a video transformer's block runs where the sparse call does not:

* ``int8``: out = residual + gate * act(sx sw (X W^T) + bias) with X the rows [x | x2] in 8-bit integers (one scale a
  row, taken from the row), W 8-bit weights with one scale a channel;
* ``attention``: softmax(mask(cap(scale q k^T) - slope |i - j|)) v, each query row seeing one interval of keys
  (documents of a packed sequence, a causal order with a prefix that all see, a window, lengths);
* ``attention_backward``: the gradients of q, k and v.

``listed`` gives the cases, ``draw`` more of the same ranges, ``prepare`` a case's inputs, ``run`` one pass (the plain
form in elementary torch operations, or the package's operators when ``own`` is set), ``exact`` the definition in 64
bits and ``work`` the bytes and operations no form can avoid.
"""

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the modulation vector of a dual-stream block from one row: the weight's read is all there is
        _int8("int8 modulation row", rows=1, k=3072, n=18432),
        # text stream's first MLP layer: few rows
        _int8("int8 text mlp", rows=256, k=3072, n=12288, act="gelu_tanh"),
        # Q, K and V of the video rows: the rows are quantised once for three layers
        _int8("int8 video qkv", rows=6750, k=3072, n=3072, layers=3),
        # video stream's first MLP layer at the 480-line call's token count
        _int8("int8 video mlp", rows=6750, k=3072, n=12288, act="gelu_tanh"),
        # single-stream block's output: attention rows and MLP hidden side by side, gate and residual
        _int8("int8 joined projection", rows=7006, k=3072, k2=12288, n=3072, gate=True, residual=True),
        # rows, features and outputs that no vector width divides, a gate per sample
        _int8("int8 odd fp16", batch=3, rows=333, k=1001, n=1999, act="gelu", gate=True, residual=True, dtype="fp16"),
        # a dense step of the 480-line call: video and valid text see each other, the padding only itself
        _attention("attention dense step", heads=24, kv=24, rows=7006, keys=7006, docs=2),
        # clips of unequal lengths packed in one sequence, generated in order after a prompt that all rows see; rows
        # behind the last clip see nothing; four query heads to a key head
        _attention("attention packed clips", heads=8, kv=2, rows=9999, keys=9999, docs=4, tail=77, causal=True, prefix=200,
                   d=64, dtype="fp16"),
        # text rows with capped scores and a bias by distance: latency counts
        _attention("attention text capped", batch=2, heads=12, kv=12, rows=256, keys=256, cap=30.0, slopes=True, d=64),
        # one new row of each of four clips over its cache of unequal length
        _attention("attention one row", batch=4, heads=24, kv=4, rows=1, keys=16384, lengths=True, causal=True),
        # training a dense step
        _attention("attention dense step backward", heads=24, kv=24, rows=7006, keys=7006, docs=2, backward=True),
        # training on packed clips, every part of the scores' definition, shared key heads
        _attention("attention packed clips backward", heads=6, kv=2, rows=4001, keys=4001, docs=5, tail=33, causal=True,
                   prefix=64, cap=20.0, slopes=True, dtype="fp16", d=80, backward=True),
    ]


def _int8(name, rows, k, n, batch=1, k2=0, act="none", gate=False, residual=False, layers=1, dtype="bf16"):
    return {"name": name, "op": "int8", "batch": batch, "rows": rows, "k": k, "k2": k2, "n": n, "act": act, "gate": gate,
            "residual": residual, "layers": layers, "dtype": dtype}


def _attention(name, heads, kv, rows, keys, batch=1, docs=0, tail=0, lengths=False, causal=False, prefix=0, window=0,
               cap=0.0, slopes=False, d=128, dtype="bf16", backward=False, token_major=False):
    return {"name": name, "op": "attention", "batch": batch, "heads": heads, "kv": kv, "rows": rows, "keys": keys, "d": d,
            "docs": docs, "tail": tail, "lengths": lengths, "causal": causal, "prefix": prefix, "window": window, "cap": cap,
            "slopes": slopes, "dtype": dtype, "backward": backward, "token_major": token_major}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if rng.random() < 0.4:
        batch = rng.choice((1, 1, 2, 3))
        rows, k, n = _log(rng, 1, 8192 // batch), _log(rng, 64, 4096), _log(rng, 64, 12288)
        layers = rng.choice((1, 1, 1, 3))
        k2 = rng.choice((0, 0, _log(rng, 64, 8192))) if layers == 1 else 0
        n = n if layers == 1 else max(64, n // 3)
        if rng.random() < 0.6:  # most layers' widths are multiples of a vector; the rest stay odd
            k, n, k2 = k // 16 * 16, n // 8 * 8, k2 // 16 * 16
        rows = max(1, min(rows, int(3.2e11 / (batch * (k + k2) * n * layers))))
        c = _int8("", rows, k, n, batch, k2, rng.choice(("none", "gelu_tanh", "gelu", "silu")), rng.random() < 0.5,
                  rng.random() < 0.5, layers, dtype)
    else:
        batch, kv = rng.choice((1, 1, 2, 4)), rng.choice((1, 2, 4, 6))
        heads = kv * rng.choice((1, 1, 2, 4))
        backward = rng.random() < 0.4
        most = int(math.sqrt(1.0e9 / (batch * heads)))  # the plain form holds every score
        form = rng.choice(("self", "self", "cross", "one"))
        rows = 1 if form == "one" and not backward else _log(rng, 1, min(most, 9000))
        keys = rows if form == "self" else _log(rng, 1, min(16384, int(1.0e9 / (batch * heads * rows))))
        docs = rng.choice((0, 1, 3, 8)) if form == "self" and rows >= 64 else 0
        causal = rng.random() < 0.5
        c = _attention("", heads, kv, rows, keys, batch, docs, rng.choice((0, 5, 40)) if docs else 0,
                       lengths=not docs and rng.random() < 0.5, causal=causal,
                       prefix=rng.choice((0, 0, 1, 77)) if causal else 0,
                       cap=rng.choice((0.0, 0.0, 15.0, 50.0)), slopes=rng.random() < 0.4,
                       d=rng.choice((64, 128, 128, 40, 80, 96)), dtype=dtype, backward=backward,
                       token_major=rng.random() < 0.5)
        if not c["prefix"] and rng.random() < 0.3:
            c["window"] = _log(rng, 1, 2000)
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dt)

    return {"case": dict(case), **(_int8_inputs if case["op"] == "int8" else _attention_inputs)(case, g, normal)}


def _int8_inputs(c, g, normal):
    b, m, k, n = c["batch"], c["rows"], c["k"] + c["k2"], c["n"]

    def rows(width):  # activations: some channels are much larger than the rest
        spread = torch.exp(0.7 * torch.randn(width, generator=g, device="cuda"))
        return (torch.randn(b, m, width, generator=g, device="cuda") * spread).to(_DT[c["dtype"]])

    s = {"x": rows(c["k"]), "x2": rows(c["k2"]) if c["k2"] else None,
         "gate": normal(b, 3 * n, std=0.5).unflatten(1, (3, n))[:, 2] if c["gate"] else None,
         "residual": normal(b, m, n) if c["residual"] else None, "layers": []}
    for _ in range(c["layers"]):  # weights as a checkpoint in 8 bits holds them
        values = torch.randn(n, k, generator=g, device="cuda").mul_(35).round_().clamp_(-127, 127).to(torch.int8)
        scales = torch.rand(n, generator=g, device="cuda").add_(0.5).mul_(k ** -0.5 / 55)
        s["layers"].append((values, scales, normal(n, std=0.1)))
    return s


def _cuts(c):
    """Ends of the documents: unequal, the same for every seed (they are part of the case's size)."""
    rng, total, n = random.Random(c["rows"] * 31 + c["docs"]), c["rows"] - c["tail"], c["docs"]
    share = [rng.uniform(0.3, 1.7) for _ in range(n)] if n != 2 else [0.979, 0.021]
    ends, at = [0], 0.0
    for w in share:
        at += w
        ends.append(int(total * at / sum(share)))
    return ends


def _lengths(c):
    rng = random.Random(c["keys"] * 17 + c["batch"])
    return [max(1, int(c["keys"] * rng.uniform(0.4, 1.0))) for _ in range(c["batch"])]


def _attention_inputs(c, g, normal):
    b, d = c["batch"], c["d"]

    def heads(n, rows):
        if c["token_major"]:
            return normal(b, rows, n, d).transpose(1, 2)
        return normal(b, n, rows, d)

    s = {"q": heads(c["heads"], c["rows"]), "k": heads(c["kv"], c["keys"]), "v": heads(c["kv"], c["keys"]),
         "documents": torch.tensor(_cuts(c), dtype=torch.int32, device="cuda") if c["docs"] else None,
         "lengths": torch.tensor(_lengths(c), dtype=torch.int32, device="cuda") if c["lengths"] else None,
         # geometric slopes from 1/2 down
         "slopes": 0.5 ** (1 + 7 * torch.arange(c["heads"], device="cuda") / c["heads"]) if c["slopes"] else None}
    if c["backward"]:
        s["grad"] = heads(c["heads"], c["rows"])
        out, s["lse"], _, _ = _scores_and_output(c, s)
        s["out"] = out.to(_DT[c["dtype"]])
    return s


# ---- one pass ----------------------------------------------------------------

def run(state):
    c = state["case"]
    if c["op"] == "int8":
        return (_own_int8 if own else _plain_int8)(c, state)
    if c["backward"]:
        return (_own_backward if own else _plain_backward)(c, state)
    return (_own_attention if own else _plain_attention)(c, state)


def _own_int8(c, s):
    from peco_b200 import int8
    args = dict(activation=None if c["act"] == "none" else c["act"], gate=s["gate"], residual=s["residual"])
    if c["layers"] == 1:
        values, scales, bias = s["layers"][0]
        return [int8.linear_int8(s["x"], int8.QuantizedRows(values, scales), bias, x2=s["x2"], **args)]
    rows = int8.quantize_rows(s["x"])
    return [int8.linear_int8(rows, int8.QuantizedRows(values, scales), bias, dtype=s["x"].dtype, **args)
            for values, scales, bias in s["layers"]]


def _own_args(c, s):
    from peco_b200 import attention
    spans = None
    if c["docs"] or c["lengths"] or c["causal"] or c["window"]:
        spans = attention.key_spans(c["batch"], c["rows"], c["keys"], documents=s["documents"], lengths=s["lengths"],
                                    causal=c["causal"], prefix=c["prefix"] or None, window=c["window"] or None,
                                    device=s["q"].device)
    return dict(spans=spans, softcap=c["cap"] or None, slopes=s["slopes"])


def _own_attention(c, s):
    from peco_b200 import attention
    out, lse = attention.attention(s["q"], s["k"], s["v"], return_lse=True, **_own_args(c, s))
    return {"out": out, "lse": lse}


def _own_backward(c, s):
    from peco_b200 import attention
    g = attention.attention_backward(s["grad"], s["q"], s["k"], s["v"], s["out"], s["lse"], **_own_args(c, s))
    return {"q": g.q, "k": g.k, "v": g.v}


def _activate(z, act):
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_int8(c, s):
    dt = s["x"].dtype
    x = s["x"] if s["x2"] is None else torch.cat((s["x"], s["x2"]), -1)
    top = x.abs().amax(-1, keepdim=True)
    # in 64 bits: whether a value lies on the border between two integers
    q = torch.round(x.double() * 127 / top.double().clamp_min(1e-300)).float()
    step = top.float() / 127
    outs = []
    for values, scales, bias in s["layers"]:
        y = _activate(q @ values.float().t() * step * scales + bias.float(), c["act"])
        if s["gate"] is not None:
            y = y * s["gate"].float()[:, None]
        if s["residual"] is not None:
            y = y + s["residual"].float()
        outs.append(y.to(dt))
    return outs


def _intervals(c, s):
    """(first key, key behind the last, position among the keys) of every query row, [batch, rows, 1] each."""
    b, n, keys = c["batch"], c["rows"], c["keys"]
    i = torch.arange(n, device="cuda")
    if c["docs"]:
        ends = s["documents"].long()
        doc = (torch.searchsorted(ends, i, right=True) - 1).clamp(0, c["docs"] - 1)
        lo, hi, pos = ends[doc], ends[doc + 1], i
        hi = torch.where(i < ends[-1], hi, lo)
        lo, hi, pos = (t.expand(b, n) for t in (lo, hi, pos))
    else:
        hi = s["lengths"].long()[:, None].expand(b, n) if c["lengths"] else torch.full((b, n), keys, device="cuda")
        lo, pos = torch.zeros_like(hi), i + hi - n
    if c["causal"]:
        seen = pos + 1
        if c["prefix"]:
            seen = torch.maximum(seen, lo + c["prefix"])
        hi = torch.minimum(hi, seen)
    if c["window"]:
        lo, hi = torch.maximum(lo, pos - c["window"] + 1), torch.minimum(hi, pos + c["window"])
    return lo[..., None], hi[..., None], pos[..., None]


def _scores_and_output(c, s):
    b, h, kv, n, d = c["batch"], c["heads"], c["kv"], c["rows"], c["d"]
    group = h // kv
    q = s["q"].float().reshape(b, kv, group * n, d)
    k, v = s["k"].float(), s["v"].float()
    z = (q @ k.transpose(-1, -2)).view(b, h, n, c["keys"]) * d ** -0.5
    slope = None
    if c["cap"]:
        t = torch.tanh(z / c["cap"])
        z, slope = c["cap"] * t, 1 - t * t
    lo, hi, pos = _intervals(c, s)
    j = torch.arange(c["keys"], device="cuda")
    if c["slopes"]:
        z = z - s["slopes"].float()[:, None, None] * (pos - j).abs().float()[:, None]
    z = z.masked_fill(((j < lo) | (j >= hi))[:, None], -math.inf)
    top = z.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, 1.0)
    out = (p.view(b, kv, group * n, -1) @ v).view(b, h, n, d)
    lse = torch.where(total > 0, top + torch.log(total), -math.inf)[..., 0]
    return out, lse, p, slope


def _plain_attention(c, s):
    out, lse, _, _ = _scores_and_output(c, s)
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _plain_backward(c, s):
    b, h, kv, n, d = c["batch"], c["heads"], c["kv"], c["rows"], c["d"]
    dt, joined = s["q"].dtype, (b, kv, h // kv * n)
    out, _, p, slope = _scores_and_output(c, s)
    g = s["grad"].float()
    dp = (g.reshape(*joined, d) @ s["v"].float().transpose(-1, -2)).view_as(p)
    dz = p * (dp - (g * out).sum(-1, keepdim=True))
    if slope is not None:
        dz = dz * slope
    dz = (dz * d ** -0.5).view(*joined, -1)
    dq = (dz @ s["k"].float()).view(b, h, n, d)
    dk = dz.transpose(-1, -2) @ s["q"].float().reshape(*joined, d)
    dv = p.view(*joined, -1).transpose(-1, -2) @ g.reshape(*joined, d)
    return {"q": dq.to(dt), "k": dk.to(dt), "v": dv.to(dt)}


# ---- the definition in 64 bits -------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_int8(case, s) if case["op"] == "int8" else _exact_attention(case, s)


def _exact_int8(c, s):
    fn = torch.nn.functional
    act = {"none": lambda z: z, "gelu_tanh": lambda z: fn.gelu(z, approximate="tanh"), "gelu": fn.gelu, "silu": fn.silu}[c["act"]]
    rows = [t.double() for t in (s["x"], s["x2"]) if t is not None]
    top = torch.stack([r.abs().amax(-1) for r in rows]).amax(0).unsqueeze(-1)
    steps, parts = [], []
    for r in rows:  # |r| 127 / top, to the nearest integer by comparing what is left over with a half; ties to even
        size = r.abs() * 127
        whole = torch.floor(size / top)
        rest = 2 * (size - whole * top)
        up = (rest > top) | ((rest == top) & (torch.remainder(whole, 2) == 1))
        parts.append(torch.where(top > 0, torch.copysign(whole + up, r), 0.0))
    steps = top / 127
    outs = []
    for values, scales, bias in s["layers"]:
        w = values.double()
        z = parts[0] @ w[:, :c["k"]].t()
        if len(parts) > 1:
            z = z + parts[1] @ w[:, c["k"]:].t()
        y = act(torch.addcmul(bias.double(), z, steps * scales.double()))
        y = y if s["gate"] is None else s["gate"].double().unsqueeze(1) * y
        outs.append(y if s["residual"] is None else y + s["residual"].double())
    return outs


def _exact_attention(c, s):
    """One head after another, the mask from its words: a document's rows, the order, the prefix, the window."""
    b, h, kv, n, keys, d = (c[x] for x in ("batch", "heads", "kv", "rows", "keys", "d"))
    i, j = torch.arange(n, device="cuda").unsqueeze(1), torch.arange(keys, device="cuda").unsqueeze(0)
    got = {"out": [], "lse": [], "q": [], "k": [], "v": []}
    for x in range(b):
        if c["docs"]:
            ends = s["documents"].tolist()
            seen = torch.zeros(n, keys, dtype=torch.bool, device="cuda")
            early = torch.zeros_like(seen)
            for a, e in zip(ends, ends[1:]):
                seen[a:e, a:e] = True
                early[a:e, a:a + c["prefix"]] = True
            apart = i - j
        else:
            length = int(s["lengths"][x]) if c["lengths"] else keys
            seen = (j < length).expand(n, keys)
            early = j < c["prefix"]
            apart = i + (length - n) - j
        if c["causal"]:
            seen = seen & ((apart >= 0) | early)
        if c["window"]:
            seen = seen & (apart.abs() < c["window"])
        per = {"k": [], "v": []}
        for y in range(h):
            q, k, v = (t.double() for t in (s["q"][x, y], s["k"][x, y // (h // kv)], s["v"][x, y // (h // kv)]))
            z = (q @ k.t()) / math.sqrt(d)
            capped = c["cap"] * torch.tanh(z / c["cap"]) if c["cap"] else z
            raw = capped
            if c["slopes"]:
                raw = raw - s["slopes"][y].double() * apart.abs()
            raw = torch.where(seen, raw, -math.inf)
            lse = torch.logsumexp(raw, 1, keepdim=True)
            p = torch.where(seen, torch.exp(raw - lse), 0.0)
            out = p @ v
            if not c["backward"]:
                got["out"].append(out)
                got["lse"].append(lse[:, 0])
                continue
            g = s["grad"][x, y].double()
            dz = p * (g @ v.t() - (g * out).sum(1, keepdim=True))
            if c["cap"]:
                dz = dz * (1 - torch.square(capped / c["cap"]))
            got["q"].append(dz @ k / math.sqrt(d))
            per["k"].append(dz.t() @ q / math.sqrt(d))
            per["v"].append(p.t() @ g)
        if c["backward"]:
            for name in ("k", "v"):
                got[name].append(torch.stack(per[name]).view(kv, h // kv, keys, d).sum(1))
    if c["backward"]:
        return {"q": torch.stack(got["q"]).view(b, h, n, d), "k": torch.stack(got["k"]), "v": torch.stack(got["v"])}
    return {"out": torch.stack(got["out"]).view(b, h, n, d), "lse": torch.stack(got["lse"]).view(b, h, n)}


# ---- what no form can avoid ------------------------------------------------------

def _seen(c):
    """Pairs of query row and key that see each other, in one head of every sample."""
    total = 0
    if c["docs"]:
        ends = _cuts(c)
        spans = [(e - a, e - a) for a, e in zip(ends, ends[1:])] * c["batch"]
    else:
        spans = [(c["rows"], n) for n in (_lengths(c) if c["lengths"] else [c["keys"]] * c["batch"])]
    for n, keys in spans:
        for i in range(n):
            pos, lo, hi = i + keys - n, 0, keys
            if c["causal"]:
                hi = min(hi, max(pos + 1, c["prefix"]))
            if c["window"]:
                lo, hi = max(lo, pos - c["window"] + 1), min(hi, pos + c["window"])
            total += max(0, hi - lo)
    return total


def work(case):
    c = case
    if c["op"] == "int8":
        m, k, n, layers = c["batch"] * c["rows"], c["k"] + c["k2"], c["n"], c["layers"]
        size = 2 * m * k + layers * (n * k + 6 * n + 2 * m * n + (2 * m * n if c["residual"] else 0)) + \
            (2 * c["batch"] * n if c["gate"] else 0)
        return {"bytes": size, "flops": 2 * m * n * k * layers}
    b, h, kv, n, keys, d = (c[x] for x in ("batch", "heads", "kv", "rows", "keys", "d"))
    kept = sum(_lengths(c)) if c["lengths"] else b * keys
    pairs = _seen(c) * h
    q, k = b * h * n * d, kept * kv * d
    if c["backward"]:
        return {"bytes": 2 * (4 * q + 4 * k) + 4 * b * h * n, "flops": 10 * d * pairs}
    return {"bytes": 2 * (2 * q + 2 * k) + 4 * b * h * n, "flops": 4 * d * pairs}
