"""Attention and its gradients in 64 bits, as functions of the very tensors that a call gets (out and lse among them), with bounds that
leave one rounding to the type, that of the result: what is in between is held in 32 bits, or in two operands of 16.

u = eps / 2 is half a step of the type, f = 2^-24.  A value taken as the sum of two 16-bit operands is off by w = 4 u^2 of itself at the
most: the first rounding leaves a rest of 2 u (towards zero; u to nearest), of which the second loses as much again.  fp16's second
operand has an end: its numbers are 2^-24 apart there, and rounding towards zero loses up to all of that (to nearest: half, 2^-25; that
is what a result's own rounding loses).  The rest as in tests/test_gpu_layers.py: D products in a score, n f for a sum of n terms, exp2
of a score that is off by e is off by the factor e."""
import math

import torch

F = 2.0 ** -24
SLACK = 1.05                                              # second order


def half_step(t):
    return torch.finfo(t).eps / 2


def two(t):
    return 0.0 if t == torch.float32 else 4 * half_step(t) ** 2


def tiny(t):
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -134


def end(t):
    return 2.0 ** -24 if t == torch.float16 else 2.0 ** -134


def visible(B, Lq, Lk, device, causal=False, query_start=None, key_lengths=None, key_mask=None, **_):
    see = torch.ones(B, Lq, Lk, dtype=torch.bool, device=device)
    j = torch.arange(Lk, device=device)
    if key_lengths is not None:
        see &= (j < key_lengths[:, None])[:, None]
    if key_mask is not None:
        see &= key_mask[:, None]
    if causal:
        first = (Lk - Lq) if query_start is None else query_start.long()[:, None, None]
        see &= j <= torch.arange(Lq, device=device)[:, None] + first
    return see[:, None]


def _heads(x, n):
    return x.double().repeat_interleave(n, 2).permute(0, 2, 1, 3).contiguous()


def _T(x):
    return x.transpose(2, 3).contiguous()


def _scores(q, k, scale, see, base):
    """Scores, and the bound of a score less `base` (a row's maximum or lse), as the kernels form it."""
    D = q.shape[-1]
    S = scale * q @ _T(k)
    Sabs = scale * q.abs() @ _T(k.abs())
    base = S.masked_fill(~see, -math.inf).amax(-1, keepdim=True) if base is None else base
    base = torch.where(base == -math.inf, 0.0, base)
    e = torch.where(see, ((D + 4) * Sabs + 4 * (base.abs() + Sabs) + 4) * F, 0.0) + 2 * F
    return S, base, e


def forward64(q, k, v, scale=None, **masks):
    t, (B, Lq, Hq, D), (Lk, Hk) = q.dtype, q.shape, k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    see = visible(B, Lq, Lk, q.device, **masks)
    Q, K, V = _heads(q, 1), _heads(k, Hq // Hk), _heads(v, Hq // Hk)
    S, top, e = _scores(Q, K, scale, see, None)
    E = torch.exp(S - top) * see
    total = E.sum(-1, keepdim=True)
    some = torch.where(total == 0, 1.0, total)
    out = E / some @ V
    # a probability: its exponential and its operands; the sum: those of its terms
    e_E = ((e + two(t)) * E + end(t) * see) / some
    e_total = ((e + Lk * F) * E).sum(-1, keepdim=True) / some
    err = SLACK * (e_E @ V.abs() + (e_total + (Lk + 4) * F) * (E / some @ V.abs())) + tiny(t)
    return {"out": (out.permute(0, 2, 1, 3), (half_step(t) * (out.abs() + err) + err).permute(0, 2, 1, 3))}


def backward64(dout, q, k, v, out, lse, scale=None, **masks):
    t, (B, Lq, Hq, D), (Lk, Hk) = q.dtype, q.shape, k.shape[1:3]
    u, G = half_step(t), Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    sees = (lse != -math.inf)[..., None]                   # (B, Hq, Lq, 1)
    see = visible(B, Lq, Lk, q.device, **masks) & sees
    Q, dO = torch.where(sees, _heads(q, 1), 0.0), torch.where(sees, _heads(dout, 1), 0.0)
    K, V = _heads(k, G), _heads(v, G)
    S, base, e = _scores(Q, K, scale, see, lse.double()[..., None])
    P = torch.exp(S - base) * see
    O = torch.where(sees, _heads(out, 1), 0.0)
    delta, e_delta = (dO * O).sum(-1, keepdim=True), D * F * (dO * O).abs().sum(-1, keepdim=True)
    dP, e_dP = dO @ _T(V), D * F * dO.abs() @ _T(V.abs())
    dS = P * (dP - delta)
    # fp16 takes 16 P, and 16 dS or, where that would leave its range, dS times a power of two that brings the largest of those that share
    # it to at least 2^14; the second operand's end is that of fp16 over that factor.  A head's (dq) or a sequence's (dk, and all of a short
    # one) share no more than theirs
    e_P = SLACK * (e + two(t) + 2 * F) * P + end(t) / 16 * see
    e_dS = SLACK * (P * (e_dP + e_delta) + (e + two(t) + 4 * F) * dS.abs())
    def ends(d):
        return end(t) * see * (torch.clamp(dS.abs().amax(d, keepdim=True) * 2.0 ** -14, min=2.0 ** -4) if t == torch.float16 else 1.0)

    fold = lambda x: x.view(B, Hk, G, Lk, D).sum(2)
    n = Lq * G
    rows, columns = e_dS + ends((1, 2, 3) if Lq <= 64 and Lk <= 64 else (2, 3)), e_dS + ends((1, 2, 3))
    found = {}
    for name, val, err in (
            ("dq", scale * dS @ K, scale * (rows @ K.abs() + 2 * Lk * F * dS.abs() @ K.abs())),
            ("dk", scale * fold(_T(dS) @ Q), scale * (fold(_T(columns) @ Q.abs()) + 2 * n * F * fold(_T(dS.abs()) @ Q.abs()))),
            ("dv", fold(_T(P) @ dO), fold(_T(e_P) @ dO.abs()) + 2 * n * F * fold(_T(P) @ dO.abs()))):
        err = err + 2 * F * val.abs()
        found[name] = (val.permute(0, 2, 1, 3), (u * (val.abs() + err) + err + tiny(t)).permute(0, 2, 1, 3))
    return found
