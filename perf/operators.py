"""Cases of the transformer-block operators around the PECO attention call, and their plain forms.

Three operators of one video-transformer block, each with its gradient:

* ``linear``: out = residual + gate * act([x | x2] W^T + bias);
* ``norm``: r = residual_scale * x + gate * post_norm(branch), h = norm(r) * weight * (1 + scale) + shift;
* ``rotary``: rotation of Q and K by positions on several axes (time, height, width).

``listed`` gives the cases, ``draw`` more of the same ranges, ``prepare`` a
case's inputs, ``run`` one pass (the plain form in elementary fp32 torch
operations, or the package's operators when ``own`` is set), ``exact`` the
definition in 64 bits and ``work`` the bytes and operations no form can avoid.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # the modulation vector of a dual-stream block: one row (batch of one prompt) against six hidden
        # sizes of outputs; the weight's read is all there is
        _linear("linear modulation row", batch=1, rows=1, k=3072, k2=0, n=18432, act="none", bias=True),
        # text stream's first MLP layer: few rows, wide weight
        _linear("linear text mlp", batch=1, rows=256, k=3072, k2=0, n=12288, act="gelu_tanh", bias=True),
        # video stream's first MLP layer at the 480-line call's token count
        _linear("linear video mlp", batch=1, rows=6750, k=3072, k2=0, n=12288, act="gelu_tanh", bias=True),
        # single-stream block's output projection: attention rows and MLP hidden side by side, gate and residual
        _linear("linear joined projection", batch=1, rows=7006, k=3072, k2=12288, n=3072, act="none", bias=True,
                gate=True, residual=True),
        # odd everything: rows, features and outputs that no vector width divides, a gate per sample
        _linear("linear odd fp16", batch=3, rows=333, k=1001, k2=0, n=1999, act="gelu", bias=True, gate=True,
                residual=True, dtype="fp16"),
        # training the video MLP's first layer: gradients of the rows, the weight and the bias
        _linear("linear video mlp backward", batch=1, rows=6750, k=3072, k2=0, n=12288, act="gelu_tanh", bias=True,
                backward=True),
        # text rows before a block: layer norm and modulation alone; latency counts
        _norm("norm text rows", batch=1, rows=256, c=3072, norm="layer", modulate=True),
        # between attention and MLP at 544x960x61 frames: gated residual, then norm and modulation
        _norm("norm gated video rows", batch=1, rows=34680, c=3072, norm="layer", modulate=True, branch=True,
              gate=True),
        # odd width, norms on both sides of the block, two samples
        _norm("norm odd fp16 sandwich", batch=2, rows=777, c=1001, norm="rms", weight=True, modulate=True,
              branch=True, gate=True, post="rms", residual_scale=0.5, dtype="fp16"),
        # gradients of the gated residual norm at the 480-line call's sequence
        _norm("norm gated backward", batch=1, rows=7006, c=3072, norm="layer", modulate=True, branch=True, gate=True,
              backward=True),
        # Q and K of the long video: 118800 grid tokens and 256 text rows that stay as they are
        _rotary("rotary long video", batch=1, heads=24, kv=24, t=33, h=45, w=80, text=256, a0=16, a1=56, a2=56),
        # gradient direction, explicit positions, fewer key heads, halves paired, token-major rows, a part of the
        # head left unrotated
        _rotary("rotary positions inverse", batch=2, heads=6, kv=2, t=1, h=30, w=45, text=64, a0=16, a1=20, a2=20,
                d=64, positions=True, split=True, inverse=True, token_major=True, dtype="fp16"),
    ]


def _linear(name, batch, rows, k, k2, n, act, bias=False, gate=False, residual=False, dtype="bf16", backward=False):
    return {"name": name, "op": "linear", "batch": batch, "rows": rows, "k": k, "k2": k2, "n": n, "act": act,
            "bias": bias, "gate": gate, "residual": residual, "dtype": dtype, "backward": backward}


def _norm(name, batch, rows, c, norm, modulate=False, weight=False, branch=False, gate=False, post="none",
          residual_scale=1.0, dtype="bf16", backward=False):
    return {"name": name, "op": "norm", "batch": batch, "rows": rows, "c": c, "norm": norm, "modulate": modulate,
            "weight": weight, "branch": branch, "gate": gate, "post": post, "residual_scale": residual_scale,
            "dtype": dtype, "backward": backward}


def _rotary(name, batch, heads, kv, t, h, w, text, a0, a1, a2, d=128, positions=False, split=False, inverse=False,
            token_major=False, dtype="bf16"):
    return {"name": name, "op": "rotary", "batch": batch, "heads": heads, "kv": kv, "t": t, "h": h, "w": w,
            "text": text, "a0": a0, "a1": a1, "a2": a2, "d": d, "positions": positions, "split": split,
            "inverse": inverse, "token_major": token_major, "dtype": dtype}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "norm", "rotary"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "linear":
        batch = rng.choice((1, 1, 2, 3))
        rows, k, n = _log(rng, 1, 8192 // batch), _log(rng, 64, 4096), _log(rng, 64, 12288)
        k2 = rng.choice((0, 0, _log(rng, 64, 8192)))
        if rng.random() < 0.6:  # most layers' widths are multiples of a vector; the rest stay odd
            k, n, k2 = k // 8 * 8, n // 8 * 8, k2 // 8 * 8
        backward = rng.random() < 0.35
        c = _linear("", batch, rows, k, k2, n, rng.choice(("none", "gelu_tanh", "gelu", "silu")), rng.random() < 0.8,
                    rng.random() < 0.5, rng.random() < 0.5 and not backward, dtype, backward)
    elif op == "norm":
        batch = rng.choice((1, 1, 2, 4))
        c = _log(rng, 64, 6144)
        if rng.random() < 0.6:
            c = c // 8 * 8
        branch = rng.random() < 0.7
        post = rng.choice(("none", "rms", "layer")) if branch else "none"
        c = _norm("", batch, _log(rng, 1, 16384 // batch), c, rng.choice(("layer", "rms")), rng.random() < 0.8,
                  rng.random() < 0.4, branch, branch and rng.random() < 0.8, post, rng.choice((1.0, 1.0, 0.5)), dtype,
                  rng.random() < 0.4)
    else:
        a0, a1, a2, d = rng.choice(((16, 56, 56, 128), (16, 24, 24, 64), (8, 12, 12, 40), (44, 42, 42, 128), (22, 22, 20, 96)))
        kv = rng.choice((1, 2, 4))
        c = _rotary("", rng.choice((1, 1, 2)), kv * rng.choice((1, 2, 5)), kv, _log(rng, 1, 16), _log(rng, 2, 45),
                    _log(rng, 2, 80), rng.choice((0, 7, 64, 256)), a0, a1, a2, d, rng.random() < 0.5,
                    rng.random() < 0.5, rng.random() < 0.4, rng.random() < 0.5, rng.choice((dtype, dtype, "fp32")))
    del c["name"]
    return c


# ---- inputs ------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).add_(mean).to(dt)

    return {"case": dict(case), **{"linear": _linear_inputs, "norm": _norm_inputs, "rotary": _rotary_inputs}[case["op"]](
        case, g, normal)}


def _linear_inputs(c, g, normal):
    b, m, k, k2, n = c["batch"], c["rows"], c["k"], c["k2"], c["n"]
    s = {"x": normal(b, m, k), "x2": normal(b, m, k2) if k2 else None,
         "weight": normal(n, k + k2, std=(k + k2) ** -0.5),
         "bias": normal(n, std=0.1) if c["bias"] else None,
         # one row of a modulation vector, as it is cut from a wider projection
         "gate": normal(b, 3 * n, std=0.5).unflatten(1, (3, n))[:, 2] if c["gate"] else None,
         "residual": normal(b, m, n) if c["residual"] else None}
    if c["backward"]:
        s["grad"] = normal(b, m, n)
        # the saved pre-activation, needed where the gradient depends on it
        s["preact"] = normal(b, m, n) if c["act"] != "none" or c["gate"] else None
    return s


def _norm_inputs(c, g, normal):
    b, t, w = c["batch"], c["rows"], c["c"]
    mod = normal(b, 6 * w, std=0.3).unflatten(1, (6, w))  # shift, scale, gate, ... of one projection
    s = {"x": normal(b, t, w, std=2.0, mean=0.3), "branch": normal(b, t, w) if c["branch"] else None,
         "shift": mod[:, 0] if c["modulate"] else None, "scale": mod[:, 1] if c["modulate"] else None,
         "gate": mod[:, 2] if c["gate"] else None,
         "weight": normal(w, std=0.1, mean=1.0) if c["weight"] else None,
         "post_weight": normal(w, std=0.1, mean=1.0) if c["post"] == "rms" else None}
    if c["backward"]:
        s["grad_h"] = normal(b, t, w)
        s["grad_r"] = normal(b, t, w) if c["branch"] else None
    return s


def _rotary_inputs(c, g, normal):
    b, d = c["batch"], c["d"]
    rows = c["t"] * c["h"] * c["w"] + c["text"]

    def heads(n):
        if c["token_major"]:
            return normal(b, rows, n, d).transpose(1, 2)
        return normal(b, n, rows, d)

    s = {"q": heads(c["heads"]), "k": heads(c["kv"]), "positions": None}
    if c["positions"]:  # every sample's window of a longer clip starts elsewhere
        start = torch.randint(0, 20, (b, 1, 3), generator=g, device="cuda", dtype=torch.int32)
        s["positions"] = start + _grid_positions(c)
    return s


def _grid_positions(c):
    i = torch.arange(c["t"] * c["h"] * c["w"], device="cuda", dtype=torch.int32)
    return torch.stack((i // (c["h"] * c["w"]), i // c["w"] % c["h"], i % c["w"]), -1)


# ---- one pass ----------------------------------------------------------------

def run(state):
    c = state["case"]
    f = {"linear": (_plain_linear, _own_linear), "norm": (_plain_norm, _own_norm),
         "rotary": (_plain_rotary, _own_rotary)}[c["op"]][1 if own else 0]
    return f(c, state)


def _own_linear(c, s):
    from peco_b200 import linear
    act = None if c["act"] == "none" else c["act"]
    if c["backward"]:
        r = linear.linear_act_backward(s["grad"], s["x"], s["weight"], preact=s["preact"], activation=act,
                                       gate=s["gate"], x2=s["x2"], bias=c["bias"])
        return {"x": r.x, "x2": r.x2, "weight": r.weight, "bias": r.bias, "gate": r.gate}
    return {"out": linear.linear_act(s["x"], s["weight"], s["bias"], activation=act, gate=s["gate"],
                                     residual=s["residual"], x2=s["x2"])}


def _own_norm(c, s):
    from peco_b200 import norms
    args = dict(gate=s["gate"], scale=s["scale"], shift=s["shift"], weight=s["weight"], post_weight=s["post_weight"],
                norm=c["norm"], post_norm=None if c["post"] == "none" else c["post"], eps=1e-6,
                residual_scale=c["residual_scale"])
    if c["backward"]:
        r = norms.modulated_norm_backward(s["grad_h"], s["grad_r"], s["x"], s["branch"], **args)
        return {"x": r.x, "branch": r.branch, "gate": r.gate, "scale": r.scale, "shift": r.shift, "weight": r.weight,
                "post_weight": r.post_weight}
    out = norms.modulated_norm(s["x"], s["branch"], **args)
    return {"r": out[0], "h": out[1]} if c["branch"] else {"h": out}


def _own_rotary(c, s):
    from peco_b200 import rotary
    q, k = rotary.rotate(s["q"], s["k"], axes=(c["a0"], c["a1"], c["a2"]), theta=256.0,
                         grid=None if c["positions"] else (c["t"], c["h"], c["w"]), positions=s["positions"],
                         interleaved=not c["split"], inverse=c["inverse"])
    return {"q": q, "k": k}


def _activate(z, act):
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, act):
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_linear(c, s):
    dt = s["x"].dtype
    x = s["x"].float() if s["x2"] is None else torch.cat((s["x"].float(), s["x2"].float()), -1)
    w = s["weight"].float()
    if c["backward"]:
        g = s["grad"].float()
        dz, dgate = g, None
        if s["gate"] is not None:
            dgate = (g * _activate(s["preact"].float(), c["act"])).sum(1).to(dt)
            dz = dz * s["gate"].float()[:, None]
        if c["act"] != "none":
            dz = dz * _slope(s["preact"].float(), c["act"])
        dx = dz @ w
        dw = dz.flatten(0, 1).t() @ x.flatten(0, 1)
        return {"x": dx[..., :c["k"]].to(dt), "x2": dx[..., c["k"]:].to(dt) if c["k2"] else None, "weight": dw.to(dt),
                "bias": dz.sum((0, 1)).to(dt) if c["bias"] else None, "gate": dgate}
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _activate(z, c["act"])
    if s["gate"] is not None:
        y = y * s["gate"].float()[:, None]
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"out": y.to(dt)}


def _normalize(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    return x * inv, inv


def _normalize_slope(g, n, inv, kind):
    d = g - n * (g * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(-1, keepdim=True)
    return d * inv


def _plain_norm(c, s):
    dt = s["x"].dtype
    r = c["residual_scale"] * s["x"].float()
    b = None
    if c["branch"]:
        b, pn, pinv = s["branch"].float(), None, None
        if c["post"] != "none":
            pn, pinv = _normalize(b, c["post"])
            b = pn if s["post_weight"] is None else pn * s["post_weight"].float()
        gb = b if s["gate"] is None else b * s["gate"].float()[:, None]
        r = r + gb
    n, inv = _normalize(r, c["norm"])
    y = n if s["weight"] is None else n * s["weight"].float()
    if not c["backward"]:
        if c["modulate"]:
            y = y * (1 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
        return {"r": r.to(dt), "h": y.to(dt)} if c["branch"] else {"h": y.to(dt)}
    g = s["grad_h"].float()
    grads = dict.fromkeys(("x", "branch", "gate", "scale", "shift", "weight", "post_weight"))
    if c["modulate"]:
        grads["shift"], grads["scale"] = g.sum(1), (g * y).sum(1)
        g = g * (1 + s["scale"].float()[:, None])
    if s["weight"] is not None:
        grads["weight"] = (g * n).sum((0, 1))
        g = g * s["weight"].float()
    dr = _normalize_slope(g, n, inv, c["norm"])
    if c["branch"]:
        dr = dr + s["grad_r"].float()
        db = dr
        if s["gate"] is not None:
            grads["gate"] = (dr * b).sum(1)
            db = dr * s["gate"].float()[:, None]
        if c["post"] != "none":
            if s["post_weight"] is not None:
                grads["post_weight"] = (db * pn).sum((0, 1))
                db = db * s["post_weight"].float()
            db = _normalize_slope(db, pn, pinv, c["post"])
        grads["branch"] = db
    grads["x"] = c["residual_scale"] * dr
    return {k: None if v is None else v.to(dt) for k, v in grads.items()}


def _angles(c, positions):
    freq = torch.cat([256.0 ** (-torch.arange(0, a, 2, device="cuda", dtype=torch.float32) / a)
                      for a in (c["a0"], c["a1"], c["a2"])])
    axis = torch.arange(3, device="cuda").repeat_interleave(torch.tensor([c["a0"], c["a1"], c["a2"]], device="cuda") // 2,
                                                            output_size=freq.numel())
    return (positions.float()[..., axis] * freq).unsqueeze(-3)  # [.., 1, tokens, pairs]


def _plain_rotary(c, s):
    pos = s["positions"] if s["positions"] is not None else _grid_positions(c)
    ang = _angles(c, pos)
    if pos.dim() == 2:
        ang = ang[None]
    cos, sin = torch.cos(ang), torch.sin(ang)
    if c["inverse"]:
        sin = -sin
    n, p = pos.shape[-2], ang.shape[-1]

    def turn(x):
        out = x.float().clone()
        rows = x[:, :, :n, :2 * p].float()
        if c["split"]:
            a, b = rows[..., :p], rows[..., p:]
            out[:, :, :n, :2 * p] = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = rows[..., 0::2], rows[..., 1::2]
            out[:, :, :n, :2 * p] = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return out.to(x.dtype)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


# ---- the definition in 64 bits -------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"linear": _exact_linear, "norm": _exact_norm, "rotary": _exact_rotary}[case["op"]](case, s)


def _leaf(t):
    return None if t is None else t.double().detach().requires_grad_()


def _through(names, tensors, outputs, grads):
    """Gradients of ``outputs`` against the named tensors that are there, by differentiation."""
    there = [(n, t) for n, t in zip(names, tensors) if t is not None]
    got = torch.autograd.grad(outputs, [t for _, t in there], grads)
    return {**dict.fromkeys(names), **dict(zip([n for n, _ in there], got))}


def _exact_linear(c, s):
    fn = torch.nn.functional
    act = {"none": lambda z: z, "gelu_tanh": lambda z: fn.gelu(z, approximate="tanh"), "gelu": fn.gelu,
           "silu": fn.silu}[c["act"]]
    x, x2, w, gate = (_leaf(s[k]) for k in ("x", "x2", "weight", "gate"))
    if not c["backward"]:
        with torch.no_grad():
            y = x @ w[:, :c["k"]].t()
            if x2 is not None:
                y += x2 @ w[:, c["k"]:].t()
            y = act(y if s["bias"] is None else y + s["bias"].double())
            y = y if gate is None else gate.unsqueeze(1) * y
            return {"out": y if s["residual"] is None else s["residual"].double() + y}
    g = s["grad"].double()
    z = (s["preact"] if s["preact"] is not None else s["grad"]).double().requires_grad_()
    y = act(z) if gate is None else gate.unsqueeze(1) * act(z)
    first = _through(("z", "gate"), (z, gate), [y], [g])
    with torch.no_grad():
        dz = first["z"].reshape(-1, c["n"])
        dx = (dz @ w).reshape(c["batch"], c["rows"], -1)
        rows = x if x2 is None else torch.cat((x, x2), 2)
        return {"x": dx[..., :c["k"]], "x2": None if x2 is None else dx[..., c["k"]:],
                "weight": torch.mm(dz.t(), rows.reshape(dz.shape[0], -1)),
                "bias": dz.sum(0) if c["bias"] else None, "gate": first["gate"]}


def _exact_norm(c, s):
    names = ("x", "branch", "gate", "scale", "shift", "weight", "post_weight")
    x, branch, gate, scale, shift, weight, post_weight = leaves = [_leaf(s[k]) for k in names]

    def norm(v, kind, gain):
        mean = v.mean(2, keepdim=True) if kind == "layer" else 0.0
        out = (v - mean) * torch.rsqrt(torch.square(v - mean).mean(2, keepdim=True) + 1e-6)
        return out if gain is None else gain * out

    r = c["residual_scale"] * x
    if branch is not None:
        y = branch if c["post"] == "none" else norm(branch, c["post"], post_weight)
        r = r + (y if gate is None else gate.unsqueeze(1) * y)
    h = norm(r, c["norm"], weight)
    if scale is not None:
        h = torch.addcmul(shift.unsqueeze(1), h, 1 + scale.unsqueeze(1))
    if not c["backward"]:
        return {"h": h.detach()} if branch is None else {"r": r.detach(), "h": h.detach()}
    if branch is None:
        return _through(names, leaves, [h], [s["grad_h"].double()])
    return _through(names, leaves, [h, r], [s["grad_h"].double(), s["grad_r"].double()])


def _exact_rotary(c, s):
    pos = s["positions"]
    if pos is None:  # row-major walk of the grid
        pos = torch.cartesian_prod(*(torch.arange(c[n], device="cuda") for n in "thw")).reshape(1, -1, 3)
    ang = torch.cat([pos[..., i:i + 1].double() / 256.0 ** (torch.arange(a // 2, device="cuda").double() * 2 / a)
                     for i, a in enumerate((c["a0"], c["a1"], c["a2"]))], -1).unsqueeze(1)
    turn = torch.polar(torch.ones_like(ang), -ang if c["inverse"] else ang)
    n, p = pos.shape[1], ang.shape[-1]

    def rotated(x):
        out = x.double()
        rows = out[:, :, :n, :2 * p]
        if c["split"]:
            z = torch.complex(rows[..., :p], rows[..., p:]) * turn
            rows = torch.cat((z.real, z.imag), 3)
        else:
            z = torch.complex(rows[..., ::2], rows[..., 1::2]) * turn
            rows = torch.view_as_real(z).flatten(3)
        out[:, :, :n, :2 * p] = rows
        return out

    return {"q": rotated(s["q"]), "k": rotated(s["k"])}


# ---- what no form can avoid ------------------------------------------------------

def work(case):
    c, e = case, _SIZE[case["dtype"]]
    if c["op"] == "linear":
        m, k, n = c["batch"] * c["rows"], c["k"] + c["k2"], c["n"]
        vec = (n if c["bias"] else 0) + (c["batch"] * n if c["gate"] else 0)
        if c["backward"]:
            saved = 1 if c["act"] != "none" or c["gate"] else 0
            gates = 2 * c["batch"] * n if c["gate"] else 0
            return {"bytes": e * (2 * m * k + 2 * n * k + (1 + saved) * m * n + (n if c["bias"] else 0) + gates),
                    "flops": 4 * m * k * n}
        return {"bytes": e * (m * k + n * k + (2 if c["residual"] else 1) * m * n + vec), "flops": 2 * m * k * n}
    if c["op"] == "norm":
        b, rows = c["batch"], c["batch"] * c["rows"]
        vec = b * ((2 if c["modulate"] else 0) + (1 if c["gate"] else 0)) + (1 if c["weight"] else 0) + (1 if c["post"] == "rms" else 0)
        if c["backward"]:
            return {"bytes": e * c["c"] * (rows * (6 if c["branch"] else 3) + 2 * vec), "flops": 30 * rows * c["c"]}
        return {"bytes": e * c["c"] * (rows * (4 if c["branch"] else 2) + vec), "flops": 12 * rows * c["c"]}
    grid = c["t"] * c["h"] * c["w"]
    heads = c["batch"] * (c["heads"] + c["kv"])
    return {"bytes": 2 * e * heads * (grid + c["text"]) * c["d"] + (12 * c["batch"] * grid if c["positions"] else 0),
            "flops": 3 * heads * grid * (c["a0"] + c["a1"] + c["a2"])}
