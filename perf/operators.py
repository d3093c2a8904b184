"""What is measured of the operators of attention blocks (trace_amd.layers): attention and its backward pass, rotary
positions, and the norms around a block fused with its gate and residual scale.

The sizes are those of a denoiser that attends along the 52-step horizon of every trajectory of the default sampling
call (256 agents x 20 samples, both halves of classifier-free guidance: 10240 rows), of agents attending to each
other, and generic long and single-token ones.  `own` is False: elementary torch operations in 32 bits.  `own` is
True: the calls a user makes of the library.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------------------------- cases ----

def _attention(name, back, dtype, B, Lq, Lk, Hq, Hk, D, causal=False, lengths=False, mask=False, packed=False):
    return {"name": name, "op": "attention", "backward": back, "dtype": dtype, "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq,
            "Hk": Hk, "D": D, "causal": causal, "lengths": lengths, "mask": mask, "packed": packed}


def _rotary(name, back, dtype, B, L, Hq, Hk, D, rot, interleaved, factor, start):
    return {"name": name, "op": "rotary", "backward": back, "dtype": dtype, "B": B, "L": L, "Hq": Hq, "Hk": Hk, "D": D,
            "rot": rot, "interleaved": interleaved, "factor": factor, "start": start}


def _norm(name, back, dtype, stream, groups, rows, C, kind, post, per_cond, alpha):
    return {"name": name, "op": "norm", "backward": back, "dtype": dtype, "stream": stream, "groups": groups,
            "rows": rows, "C": C, "kind": kind, "post": post, "per_cond": per_cond, "alpha": alpha}


def listed():
    return [
        # every denoiser row of a sampling call attends along its horizon; q, k, v are windows of one projection
        _attention("time axis forward f32", False, "f32", 10240, 52, 52, 4, 4, 64, packed=True),
        # the same under clean guidance, which differentiates the denoiser at every reverse step
        _attention("time axis backward f32", True, "f32", 10240, 52, 52, 4, 4, 64, packed=True),
        # agents of a scene attend to each other at each of 52 steps x 20 samples; absent agents are masked, and some
        # scenes are empty
        _attention("scene forward f16", False, "f16", 1040, 256, 256, 4, 4, 32, mask=True),
        # a prompt of 8192 tokens, four query heads to a key head
        _attention("long causal forward bf16", False, "bf16", 1, 8192, 8192, 16, 4, 128, causal=True),
        # a training step over two sequences of an odd length
        _attention("long causal backward bf16", True, "bf16", 2, 4001, 4001, 16, 4, 128, causal=True),
        # one new token for each of eight sequences, against a cache that each has filled to its own length
        _attention("token step bf16", False, "bf16", 8, 1, 8192, 32, 8, 128, lengths=True),
        # the smallest call: one token of one sequence on a short cache
        _attention("small step f32", False, "f32", 1, 1, 52, 4, 4, 64),
        # positions past the trained length, the slow pairs stretched
        _rotary("rotary long bf16", False, "bf16", 2, 8192, 32, 8, 128, 128, False, 8.0, 100000),
        # the gradient of rotated queries and keys along the horizon, half of each head rotated
        _rotary("rotary time axis backward f32", True, "f32", 10240, 52, 4, 4, 64, 32, True, 1.0, 0),
        # between two wide blocks: norm of the block's output, gate, residual, norm for the next block
        _norm("norm wide forward bf16", False, "bf16", "bf16", 1, 8192, 4096, "rms", True, False, 1.0),
        # its gradient between two blocks of a conditioned denoiser: gate, scale and shift of each trajectory
        _norm("norm time axis backward f32", True, "f32", "f32", 10240, 52, 256, "layer", False, True, 1.0),
        # the smallest call: one trajectory
        _norm("norm small forward f32", False, "f32", "f32", 1, 52, 256, "layer", False, True, 0.5),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype, back = rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5
    op = rng.choice(["attention", "attention", "attention", "rotary", "norm", "norm"])
    if op == "attention":
        group = rng.choice([1, 1, 2, 4])
        Hk = rng.choice([1, 2, 4])
        D = rng.choice([16, 20, 32, 40, 64, 72, 80, 96, 128])
        kind = rng.choice(["rows", "scene", "long", "step"])
        if kind == "rows":
            L = _log(rng, 1, 128)
            B = max(1, min(_log(rng, 16, 10240), 10240 * 52 * 4 * 64 // (L * Hk * group * D)))
            c = _attention("", back, dtype, B, L, L, Hk * group, Hk, D, causal=rng.random() < 0.3, packed=rng.random() < 0.5)
        elif kind == "scene":
            Lq, Lk = _log(rng, 2, 300), _log(rng, 2, 300)
            B = max(1, min(_log(rng, 1, 1040), 1040 * 256 * 256 * 4 // (max(Lq, Lk) ** 2 * Hk * group)))
            c = _attention("", back, dtype, B, Lq, Lk, Hk * group, Hk, D, mask=True)
        elif kind == "long":
            L = _log(rng, 129, 4001)
            c = _attention("", back, dtype, rng.choice([1, 2]), L, L, Hk * group, Hk, D, causal=rng.random() < 0.7,
                           lengths=rng.random() < 0.3)
        else:
            c = _attention("", False, dtype, _log(rng, 1, 16), rng.choice([1, 1, 1, 2, 5]), _log(rng, 20, 8192),
                           Hk * group, Hk, D, causal=rng.random() < 0.5, lengths=rng.random() < 0.7)
    elif op == "rotary":
        L, D = _log(rng, 1, 8192), rng.choice([16, 24, 64, 80, 128])
        Hk = rng.choice([1, 2, 4, 8])
        Hq = Hk * rng.choice([1, 2, 4])
        B = max(1, min(_log(rng, 1, 10240), 2 * 8192 * 40 * 128 // (L * (Hq + Hk) * D)))
        c = _rotary("", back, dtype, B, L, Hq, Hk, D, rng.choice([D, D, D // 2 // 2 * 2]), rng.random() < 0.5,
                    rng.choice([1.0, 4.0, 8.0]), rng.choice([0, 0, 1000, 100000, 1000000]))
    else:
        C = rng.choice([_log(rng, 8, 8192), rng.choice([64, 128, 256, 1024, 2048])])
        rows = _log(rng, 1, 8192)
        G = max(1, min(rng.choice([1, _log(rng, 1, 10240)]), 8192 * 4096 // (rows * C)))
        c = _norm("", back, dtype, rng.choice([dtype, "f32"]), G, rows, C, rng.choice(["rms", "layer"]),
                  rng.random() < 0.5, rng.random() < 0.5, rng.choice([1.0, 0.5]))
    del c["name"]
    return c


# --------------------------------------------------------------------------------------------- inputs ----

def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, dtype=dt, mean=0.0, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    s = dict(case)
    if case["op"] == "attention":
        B, Lq, Lk, Hq, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
        if case["packed"]:                                    # windows of one projection's output
            qkv = normal(B, Lq, Hq + 2 * Hk, D)
            s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
        else:
            s["q"], s["k"], s["v"] = normal(B, Lq, Hq, D), normal(B, Lk, Hk, D), normal(B, Lk, Hk, D)
        s["key_lengths"] = s["key_mask"] = s["query_start"] = None
        if case["lengths"]:
            n = _lengths(case).cuda()
            s["key_lengths"] = n[torch.randperm(B, generator=g, device="cuda")].contiguous()
            if case["causal"] and Lq < Lk:                    # the new tokens are the last of the cache
                s["query_start"] = s["key_lengths"] - Lq
        if case["mask"]:
            present = torch.rand(B, 1, generator=g, device="cuda") * 1.2 - 0.1
            s["key_mask"] = torch.rand(B, Lk, generator=g, device="cuda") < present
        s["scale"] = D ** -0.5
        if case["backward"]:
            s["dout"] = normal(B, Lq, Hq, D)
            s["out"], s["lse"] = _attention_forward(s)
    elif case["op"] == "rotary":
        B, L, Hq, Hk, D = (case[k] for k in ("B", "L", "Hq", "Hk", "D"))
        s["q"], s["k"] = normal(B, L, Hq, D), normal(B, L, Hk, D)
        s["positions"] = torch.arange(L, device="cuda") + case["start"] + torch.randint(
            0, 1 + case["start"] // 2, (B, 1), generator=g, device="cuda")
        half = torch.arange(case["rot"] // 2, device="cuda", dtype=torch.float64)
        f = 10000.0 ** (-2 * half / case["rot"])
        # pairs that turn less than once in 4096 positions are stretched by the factor, those that turn 32 times stay
        ramp = ((4096 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        s["freqs"] = f * ramp + f / case["factor"] * (1 - ramp)
        s["scale"] = 1 + 0.1 * math.log(case["factor"])
    else:
        G, rows, C = case["groups"], case["rows"], case["C"]
        R, n = G * rows, G if case["per_cond"] else 1
        st = _TYPES[case["stream"]]
        s["x"], s["y"] = normal(R, C, dtype=st, std=2.0, mean=0.1), normal(R, C)
        s["gate"] = normal(G, C, dtype=torch.float32, std=0.5)
        s["weight"] = normal(n, C, dtype=torch.float32, mean=1.0, std=0.2)
        s["bias"] = normal(n, C, dtype=torch.float32, std=0.2) if case["kind"] == "layer" else None
        s["post_weight"] = normal(C, dtype=torch.float32, mean=1.0, std=0.2) if case["post"] else None
        if case["backward"]:
            s["dh"], s["dz"] = normal(R, C, dtype=st), normal(R, C)
    return s


def _lengths(case):
    """The lengths a batch has, in some order: evenly spread over the upper half of the cache, one of them all of it;
    a batch of eight and more holds an empty one."""
    B, Lk = case["B"], case["Lk"]
    n = torch.linspace(Lk / 2, Lk, B).round().int() if B > 1 else torch.tensor([Lk], dtype=torch.int32)
    if B > 8:
        n[0] = 0
    return n


# ---------------------------------------------------------------------------------------- plain forms ----

def _fold(t, Hk):
    """(B, L, H, D) -> (B Hk, H / Hk * L, D) in 32 bits: the query heads of a key head one after the other."""
    B, L, H, D = t.shape
    return t.float().reshape(B, L, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B * Hk, H // Hk * L, D)


def _unfold(t, B, Hk, L):
    D = t.shape[-1]
    return t.reshape(B, Hk, -1, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, -1, D)


def _visible(s, dtype=torch.float32):
    """(B or 1, Lq, Lk) truth values: key j is seen by query i; None where all are."""
    Lq, Lk = s["Lq"], s["Lk"]
    j = torch.arange(Lk, device="cuda")
    see = None
    if s["key_lengths"] is not None:
        see = (j < s["key_lengths"][:, None])[:, None, :]
    if s["key_mask"] is not None:
        see = s["key_mask"][:, None, :] if see is None else see & s["key_mask"][:, None, :]
    if s["causal"]:
        i = torch.arange(Lq, device="cuda")[:, None]
        first = Lk - Lq if s["query_start"] is None else s["query_start"][:, None, None]
        c = j <= i + first
        c = c if c.dim() == 3 else c[None]
        see = c if see is None else see & c
    return see


def _scores(s):
    B, Lq, Lk, Hk = s["B"], s["Lq"], s["Lk"], s["Hk"]
    x = torch.matmul(_fold(s["q"], Hk), _fold(s["k"], Hk).transpose(1, 2)) * s["scale"]
    see = _visible(s)
    if see is not None:
        x = x.view(B, Hk, -1, Lq, Lk).masked_fill(~see[:, None, None], -math.inf).view(B * Hk, -1, Lk)
    return x


def _attention_forward(s):
    B, Lq, Hk = s["B"], s["Lq"], s["Hk"]
    x = _scores(s)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _fold(s["v"], Hk)) / torch.where(total == 0, 1.0, total)
    return _unfold(out, B, Hk, Lq).to(s["q"].dtype), (top + torch.log(total)).view(B, -1, Lq)


def _attention_backward(s):
    B, Lq, Lk, Hk, t = s["B"], s["Lq"], s["Lk"], s["Hk"], s["q"].dtype
    q, k, v, do = _fold(s["q"], Hk), _fold(s["k"], Hk), _fold(s["v"], Hk), _fold(s["dout"], Hk)
    lse = s["lse"].reshape(B * Hk, -1, 1)
    p = torch.exp(_scores(s) - torch.where(lse == -math.inf, 0.0, lse))
    delta = (do * _fold(s["out"], Hk)).sum(-1, keepdim=True)
    ds = p * (torch.matmul(do, v.transpose(1, 2)) - delta) * s["scale"]
    return (_unfold(torch.matmul(ds, k), B, Hk, Lq).to(t),
            _unfold(torch.matmul(ds.transpose(1, 2), q), B, Hk, Lk).to(t),
            _unfold(torch.matmul(p.transpose(1, 2), do), B, Hk, Lk).to(t))


def _rotate(x, angle, case, scale):
    x, rot = x.float(), case["rot"]
    c, n = (torch.cos(angle) * scale).float()[:, :, None], (torch.sin(angle) * scale).float()[:, :, None]
    if case["backward"]:
        n = -n
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        r = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([r, x[..., rot:]], -1)


def _spread(t, rows):
    """A table of (n, C) over the rows of its groups."""
    return t if t is None or t.shape[0] == 1 else t.repeat_interleave(rows, 0)


def _normed(t, kind):
    """(t - mean) / sqrt(var + eps), or t / sqrt(mean t^2 + eps), and the factor."""
    t = t - t.mean(-1, keepdim=True) if kind == "layer" else t
    r = torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)
    return t * r, r


def _normed_backward(d, n, r, kind):
    g = d - n * (d * n).mean(-1, keepdim=True)
    return r * (g - d.mean(-1, keepdim=True) if kind == "layer" else g)


def _norm_parts(s):
    x, y, gate = s["x"].float(), s["y"].float(), _spread(s["gate"], s["rows"])
    ny, ry = _normed(y, s["kind"]) if s["post"] else (y, None)
    u = ny * s["post_weight"] if s["post"] else y
    h = s["alpha"] * x + gate * u
    return gate, ny, ry, u, h, *_normed(h, s["kind"])


def _norm_forward(s):
    gate, ny, ry, u, h, n, r = _norm_parts(s)
    z = n * _spread(s["weight"], s["rows"])
    if s["bias"] is not None:
        z = z + _spread(s["bias"], s["rows"])
    return {"h": h.to(s["x"].dtype), "z": z.to(s["y"].dtype)}


def _norm_backward(s):
    gate, ny, ry, u, h, n, r = _norm_parts(s)
    dz, G, C = s["dz"].float(), s["groups"], s["C"]
    d = s["dh"].float() + _normed_backward(dz * _spread(s["weight"], s["rows"]), n, r, s["kind"])
    du = d * gate
    m = G if s["per_cond"] else 1
    got = {"dx": (s["alpha"] * d).to(s["x"].dtype), "dgate": (d * u).view(G, -1, C).sum(1),
           "dweight": (dz * n).view(m, -1, C).sum(1)}
    if s["bias"] is not None:
        got["dbias"] = dz.view(m, -1, C).sum(1)
    if s["post"]:
        got["dpost_weight"] = (du * ny).sum(0)
        du = _normed_backward(du * s["post_weight"], ny, ry, s["kind"])
    return {**got, "dy": du.to(s["y"].dtype)}


# ------------------------------------------------------------------------------------------ the calls ----

def run(state):
    s = state
    if own:
        from trace_amd import layers
        if s["op"] == "attention":
            masks = {"causal": s["causal"], "query_start": s["query_start"], "key_lengths": s["key_lengths"],
                     "key_mask": s["key_mask"], "scale": s["scale"]}
            if s["backward"]:
                return layers.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], **masks)
            return layers.attention(s["q"], s["k"], s["v"], **masks)
        if s["op"] == "rotary":
            return layers.rotary(s["q"], s["positions"], s["freqs"], k=s["k"], interleaved=s["interleaved"],
                                 scale=s["scale"], inverse=s["backward"])
        about = {"gate": s["gate"], "post_weight": s["post_weight"], "weight": s["weight"], "bias": s["bias"],
                 "kind": s["kind"], "residual_scale": s["alpha"], "eps": 1e-6, "rows_per_cond": s["rows"]}
        if s["backward"]:
            got = layers.residual_norm_backward(s["dh"], s["dz"], s["x"], s["y"], **about)
            return {k: v for k, v in got.items() if v is not None}
        h, z = layers.residual_norm(s["x"], s["y"], **about)
        return {"h": h, "z": z}
    if s["op"] == "attention":
        return _attention_backward(s) if s["backward"] else _attention_forward(s)
    if s["op"] == "rotary":
        angle = s["positions"].double()[..., None] * s["freqs"]
        return tuple(_rotate(s[t], angle, s, s["scale"]).to(s[t].dtype) for t in ("q", "k"))
    return _norm_backward(s) if s["backward"] else _norm_forward(s)


# ------------------------------------------------------------------------------------------- the work ----

def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "attention":
        B, Lq, Lk, Hq, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
        keys = int(_lengths(case).sum()) if case["lengths"] else B * Lk
        pairs = keys * Lq * (0.5 if case["mask"] else 1.0)           # half of the agents are there
        if case["causal"] and Lq > 1:
            pairs *= 0.5 if Lq == Lk else 1 - Lq / (2 * Lk)
        if case["backward"]:
            # in: q, out, dout, lse, k, v; out: dq, dk, dv; five products of 2 D operations a pair
            return {"bytes": e * D * (4 * B * Lq * Hq + 2 * keys * Hk + 2 * B * Lk * Hk) + 4 * B * Hq * Lq,
                    "flops": 10 * pairs * Hq * D}
        return {"bytes": e * D * (2 * B * Lq * Hq + 2 * keys * Hk) + 4 * B * Hq * Lq, "flops": 4 * pairs * Hq * D}
    if case["op"] == "rotary":
        n = case["B"] * case["L"]
        return {"bytes": 2 * n * (case["Hq"] + case["Hk"]) * case["D"] * e + 8 * n,
                "flops": 3 * n * (case["Hq"] + case["Hk"]) * case["rot"]}
    R, C, st = case["groups"] * case["rows"], case["C"], _BYTES[case["stream"]]
    tables = 4 * C * (case["groups"] + (2 if case["kind"] == "layer" else 1) * (case["groups"] if case["per_cond"] else 1)
                      + (1 if case["post"] else 0))
    if case["backward"]:                                             # in: x, y, dh, dz; out: dx, dy; tables both ways
        return {"bytes": R * C * (3 * st + 3 * e) + 2 * tables, "flops": 40 * R * C}
    return {"bytes": R * C * (2 * st + 2 * e) + tables, "flops": 15 * R * C}


# ----------------------------------------------------------------------------- the definition, 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    back = case["backward"]

    def leaf(t):
        return None if t is None else t.detach().double().requires_grad_(back)

    if case["op"] == "attention":
        q, k, v = leaf(s["q"]), leaf(s["k"]), leaf(s["v"])
        share = case["Hq"] // case["Hk"]
        kk, vv = (t.repeat_interleave(share, 2).permute(0, 2, 1, 3).contiguous() for t in (k, v))
        x = torch.matmul(q.permute(0, 2, 1, 3).contiguous(), kk.transpose(2, 3).contiguous()) * s["scale"]
        see = _visible(s)
        see = torch.ones(1, 1, 1, dtype=torch.bool, device="cuda") if see is None else see
        x = torch.where(see[:, None], x, -1e300)
        top = x.detach().amax(-1, keepdim=True)
        w = torch.exp(x - top) * see[:, None]
        total = w.sum(-1, keepdim=True)
        out = torch.matmul(w / torch.where(total == 0, 1.0, total), vv).permute(0, 2, 1, 3)
        if back:
            return torch.autograd.grad(out, (q, k, v), s["dout"].double())
        lse = torch.where(total == 0, -math.inf, top + torch.log(total))
        return out, lse[..., 0]
    if case["op"] == "rotary":
        turn = torch.polar(torch.full((), s["scale"], dtype=torch.float64, device="cuda"),
                           s["positions"].double()[..., None] * s["freqs"])[:, :, None]
        turn, rot, found = turn.conj() if back else turn, case["rot"], []
        for t in ("q", "k"):
            x = s[t].double()
            h = x[..., :rot]
            pairs = h.unflatten(-1, (-1, 2)) if case["interleaved"] else h.unflatten(-1, (2, -1)).transpose(-1, -2)
            r = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
            found.append(torch.cat([(r if case["interleaved"] else r.transpose(-1, -2)).flatten(-2), x[..., rot:]], -1))
        return tuple(found)
    x, y, gate, w, b, p = (leaf(s[t]) for t in ("x", "y", "gate", "weight", "bias", "post_weight"))
    G, C = case["groups"], case["C"]

    def norm(t):
        if case["kind"] == "layer":
            return (t - t.mean(-1, keepdim=True)) / torch.sqrt(t.var(-1, unbiased=False, keepdim=True) + 1e-6)
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6)

    u = norm(y) * p if case["post"] else y
    h = (case["alpha"] * x).view(G, -1, C) + gate[:, None] * u.view(G, -1, C)
    z = norm(h) * w[:, None]
    z = z if b is None else z + b[:, None]
    h, z = h.reshape(-1, C), z.reshape(-1, C)
    if not back:
        return {"h": h.detach(), "z": z.detach()}
    names = [n for n, t in (("dx", x), ("dy", y), ("dgate", gate), ("dweight", w), ("dbias", b), ("dpost_weight", p))
             if t is not None]
    leaves = [t for t in (x, y, gate, w, b, p) if t is not None]
    return dict(zip(names, torch.autograd.grad((h, z), leaves, (s["dh"].double(), s["dz"].double()))))
