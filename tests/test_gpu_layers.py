"""Attention-block operators (trace_amd/layers.py) on the GPU against plain implementations in 64 bits.

Tolerances are bounds, elementwise, to first order: u = eps / 2 is half a step of the type (one rounding), f = 2^-24 half a step of
fp32.  A sum of n terms in fp32, in any order, is off by at most n f times the sum of the terms' magnitudes; a rounded operand
adds u times the magnitudes it enters with; exp2 of a score that is off by e is off by the factor e (exp2 itself 2 f)."""
import math

import pytest
import torch

from trace_amd import layers

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the spacing of the smallest numbers: what rounding to the type loses where relative precision ends."""
    return 2.0 ** -25 if t == torch.float16 else 2.0 ** -134


def near(got, want, bound, what):
    """|got - want| <= bound everywhere; equal where want is not finite."""
    got = got.double()
    assert got.shape == want.shape, what
    fin = torch.isfinite(want)
    assert torch.equal(fin, torch.isfinite(got)) and torch.equal(got[~fin], want[~fin]), what
    over = ((got - want).abs() - bound)[fin]
    if over.numel():
        assert float(over.max()) <= 0, "%s: over its bound by %.3e (bound there %.3e)" % (
            what, float(over.max()), float(bound.expand_as(want)[fin][over.argmax()]))


# ------------------------------------------------------------------------------------------ attention ----

def visible(B, Lq, Lk, causal=False, query_start=None, key_lengths=None, key_mask=None, **_):
    see = torch.ones(B, Lq, Lk, dtype=torch.bool, device=DEV)
    j = torch.arange(Lk, device=DEV)
    if key_lengths is not None:
        see &= (j < key_lengths[:, None])[:, None]
    if key_mask is not None:
        see &= key_mask[:, None]
    if causal:
        first = (Lk - Lq) if query_start is None else query_start.long()[:, None, None]
        see &= j <= torch.arange(Lq, device=DEV)[:, None] + first
    return see


def attention64(q, k, v, dout=None, scale=None, **masks):
    """The formulas in 64 bits; results and their bounds as {name: (value, bound)}."""
    t, (B, Lq, Hq, D), (Lk, Hk) = q.dtype, q.shape, k.shape[1:3]
    u, G = half_step(t), Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    see = visible(B, Lq, Lk, **masks)[:, None]
    heads = lambda x, n: x.double().repeat_interleave(n, 2).permute(0, 2, 1, 3).contiguous()
    none_sees = ~see.any(2).view(B, Lk, 1, 1)                                        # such keys may hold anything
    Q, K, V = heads(q, 1), heads(k.masked_fill(none_sees, 0), G), heads(v.masked_fill(none_sees, 0), G)
    S = torch.where(see, scale * Q @ K.transpose(2, 3).contiguous(), -math.inf)
    top = S.amax(-1, keepdim=True) if Lk else torch.full((B, Hq, Lq, 1), -math.inf, device=DEV, dtype=torch.float64)
    top0 = torch.where(top == -math.inf, 0.0, top)
    E = torch.exp(S - top0)
    total = E.sum(-1, keepdim=True)
    P = E / torch.where(total == 0, 1.0, total)
    out = P @ V
    lse = torch.where(total == 0, -math.inf, top + torch.log(total))
    # a score: D products, its scaling, and what the subtraction of the maximum (lse) rounds
    Sabs = scale * Q.abs() @ K.abs().transpose(2, 3).contiguous()
    eS = torch.where(see, ((D + 4) * Sabs + 4 * (top0.abs() + Sabs) + 4) * F, 0.0) + 2 * F
    eR = eS.amax(-1, keepdim=True) if Lk else torch.zeros_like(top)                 # of a row: also its maximum and sum
    slack = 1.05                                                                    # second order
    A = P @ V.abs()
    Vmax = V.abs().amax((2, 3), keepdim=True) if Lk else torch.zeros(1, device=DEV)
    found = {"out": (out, u * out.abs() + slack * (u + 2 * eR + 3 * Lk * F) * A + tiny(t) * (1 + Lk * Vmax)),
             "lse": (lse, slack * (eR + (Lk + 4) * F) + 4 * F * torch.where(lse.isfinite(), lse.abs(), 0.0))}
    found["out"] = tuple(x.permute(0, 2, 1, 3) for x in found["out"])
    found["lse"] = tuple(x[..., 0] for x in found["lse"])
    if dout is None:
        return found
    row_sees = see.any(-1, keepdim=True)
    dO = torch.where(row_sees, heads(dout, 1), 0.0)
    Q = torch.where(row_sees, Q, 0.0)
    dP = torch.where(see, dO @ V.transpose(2, 3).contiguous(), 0.0)
    delta = (dO * out).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    # dP: D products; delta: D products of a rounded out (its own error: found["out"]); P: eS and the error of lse
    e_out = found["out"][1].permute(0, 2, 1, 3)
    e_delta = (dO.abs() * e_out).sum(-1, keepdim=True) + D * F * (dO.abs() * out.abs()).sum(-1, keepdim=True)
    e_dP = D * F * torch.where(see, dO.abs() @ V.abs().transpose(2, 3).contiguous(), 0.0)
    eP = eS + eR + (Lk + 8) * F + 4 * F * torch.where(lse.isfinite(), lse.abs(), 0.0)
    e_dS = slack * (P * (e_dP + e_delta) + (eP + u + 4 * F) * dS.abs()) + tiny(t) * see
    e_P = slack * (eP + u) * P + tiny(t) * see
    fold = lambda x: x.view(B, Hk, G, Lk, D).sum(2)
    T = lambda x: x.transpose(2, 3).contiguous()
    n = Lq * G
    for name, val, err in (
            ("dq", scale * dS @ K, scale * (e_dS @ K.abs() + Lk * F * dS.abs() @ K.abs())),
            ("dk", scale * fold(T(dS) @ Q), scale * (fold(T(e_dS) @ Q.abs()) + n * F * fold(T(dS.abs()) @ Q.abs()))),
            ("dv", fold(T(P) @ dO), fold(T(e_P) @ dO.abs()) + n * F * fold(T(P) @ dO.abs()))):
        found[name] = (val.permute(0, 2, 1, 3), (err + u * val.abs() + 2 * F * val.abs() + tiny(t)).permute(0, 2, 1, 3))
    return found


def compare(q, k, v, seed=5, scale=None, dout=None, **masks):
    if dout is None:
        g = torch.Generator(DEV).manual_seed(seed)
        dout = torch.randn(q.shape, generator=g, device=DEV).to(q.dtype)
    out, lse = layers.attention(q, k, v, scale=scale, **masks)
    dq, dk, dv = layers.attention_backward(dout, q, k, v, out, lse, scale=scale, **masks)
    want = attention64(q, k, v, dout, scale, **masks)
    for name, got in (("out", out), ("lse", lse), ("dq", dq), ("dk", dk), ("dv", dv)):
        near(got, *want[name], what=name)
    return out, lse, dq, dk, dv


def inputs(dtype, B, Lq, Lk, Hq, Hk, D, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    return r(B, Lq, Hq, D), r(B, Lk, Hk, D), r(B, Lk, Hk, D)


SIZES = [  # B, Lq, Lk, Hq, Hk, D
    (1, 1, 1, 1, 1, 1), (2, 52, 52, 4, 4, 64), (3, 33, 65, 4, 2, 32), (1, 129, 63, 6, 3, 40), (2, 7, 200, 8, 1, 128),
    (1, 300, 300, 2, 1, 80), (2, 64, 1, 3, 3, 17), (5, 1, 77, 8, 2, 64), (1, 257, 513, 2, 2, 128), (1, 130, 96, 4, 4, 20)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_attention_and_gradient(dtype, causal, size):
    compare(*inputs(dtype, *size), causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [16, 64, 128])
def test_attention_lengths_masks_and_empty_rows(dtype, D):
    B, Lq, Lk = 5, 70, 150
    q, k, v = inputs(dtype, B, Lq, Lk, 4, 2, D)
    g = torch.Generator(DEV).manual_seed(9)
    mask = torch.rand(B, Lk, generator=g, device=DEV) < 0.6
    mask[1] = False                                      # a sequence without keys
    mask[2, :64] = False                                 # a tile without keys
    lengths = torch.tensor([150, 150, 97, 0, 1], dtype=torch.int32, device=DEV)
    start = torch.tensor([80, 0, -20, 5, -3], dtype=torch.int32, device=DEV)
    for masks in (dict(key_mask=mask), dict(key_lengths=lengths), dict(key_lengths=lengths, key_mask=mask),
                  dict(causal=True, query_start=start), dict(causal=True, query_start=start, key_lengths=lengths,
                                                             key_mask=mask)):
        out, lse = compare(q, k, v, **masks)[:2]
        empty = ~visible(B, Lq, Lk, **masks).any(-1)
        assert bool(empty.any()) and bool((out[empty] == 0).all())
        assert bool((lse.transpose(1, 2)[empty] == -math.inf).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_ignores_what_masked_places_hold(dtype, bad):
    B, Lq, Lk, D = 2, 40, 100, 64
    q, k, v = inputs(dtype, B, Lq, Lk, 4, 2, D)
    dout = inputs(dtype, B, Lq, 1, 4, 4, D, seed=3)[0]
    lengths = torch.tensor([70, 0], dtype=torch.int32, device=DEV)
    mask = torch.ones(B, Lk, dtype=torch.bool, device=DEV)
    mask[0, 10:20] = False
    masks = dict(key_lengths=lengths, key_mask=mask)
    want = compare(q, k, v, dout=dout, **masks)
    for t in (k, v):
        t[0, 10:20] = bad
        t[0, 70:] = bad
        t[1] = bad
    q[1] = bad                                           # queries that see nothing
    dout[1] = bad
    got = compare(q, k, v, dout=dout, **masks)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_attention_passes_nan_on_where_it_is_seen():
    q, k, v = inputs(torch.bfloat16, 1, 40, 70, 2, 2, 32)
    v[0, 66, 1, 5] = math.nan
    out, lse = layers.attention(q, k, v)
    assert bool(torch.isnan(out[0, :, 1, 5]).all()) and int(torch.isnan(out).sum()) == 40 and bool(lse.isfinite().all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Lq, Lk", [(3, 40), (40, 60), (70, 300), (140, 200)])
def test_attention_ignores_what_lies_past_the_last_query(dtype, Lq, Lk):
    """A cache with room behind the positions that causality lets any query see."""
    q, k, v = inputs(dtype, 2, Lq, Lk, 4, 2, 64)
    start = torch.tensor([Lk - Lq - 9, -2], dtype=torch.int32, device=DEV)
    want = compare(q, k, v, causal=True, query_start=start)
    for b in range(2):
        k[b, max(0, int(start[b]) + Lq):] = math.nan
        v[b, max(0, int(start[b]) + Lq):] = math.inf
    got = compare(q, k, v, causal=True, query_start=start)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(300, 70, 70, 4, 2, 32), (600, 3, 40, 4, 2, 16), (150, 100, 90, 4, 4, 64), (40, 129, 200, 8, 8, 128)])
def test_attention_of_many_heads(dtype, size):
    """Enough workgroups that no kernel's loop is cut into shares."""
    compare(*inputs(dtype, *size), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [30.0, 300.0])
def test_attention_of_peaked_scores(dtype, spread):
    """Scores far apart: one key carries a row, the exponentials of the others vanish; the running maximum grows late."""
    q, k, v = inputs(dtype, 1, 50, 200, 2, 1, 64)
    k = (k.float() * torch.linspace(0, 1, 200, device=DEV)[None, :, None, None]).to(dtype)
    compare(q, k, v, scale=spread / 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_strides(dtype):
    """Windows of one projection, heads before tokens, shared (stride 0) keys, windows off the 16-byte grid: the results are
    those of contiguous copies, bit for bit where the same loads run and within the bounds elsewhere."""
    B, L, H, D = 2, 45, 4, 64
    g = torch.Generator(DEV).manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    packed = r(B, L, 3 * H, D)
    heads_first = r(B, H, L, D).transpose(1, 2)
    off = r(B, L, H, D + 3)[..., 1:D + 1]
    shared = r(B, L, 1, D).expand(B, L, H, D)
    one_token = r(B, 1, H, D).expand(B, L, H, D)
    for q, k, v in ((packed[:, :, :H], packed[:, :, H:2 * H], packed[:, :, 2 * H:]), (heads_first, packed[:, :, :H], heads_first),
                    (packed[:, :, :H], shared, shared), (off, packed[:, ::1, :H], heads_first), (one_token, heads_first, off),
                    (packed[:, ::3, :H], packed[:, ::2, H:2 * H], packed[:, 1::2, 2 * H:].expand(B, 22, H, D)[:, :22])):
        k = k[:, :v.shape[1]]
        dout = r(B, H, q.shape[1], D).transpose(1, 2)
        got = compare(q, k, v, dout=dout, causal=True)
        same = compare(q.contiguous(), k.contiguous(), v.contiguous(), dout=dout.contiguous(), causal=True)
        for a, b in zip(got, same):
            assert torch.equal(a, b)


@pytest.mark.parametrize("backward", [False, True])
def test_attention_offsets_past_32_bits(backward):
    """Five tokens 2^29 + 8 elements apart, in a cache of 4.3 GB: the last one lies past 2^31 elements."""
    far = 2 ** 29 + 8
    room = torch.zeros(4 * far + 2 * 64, dtype=torch.bfloat16, device=DEV)
    k = room.as_strided((1, 5, 1, 64), (0, far, 64, 1))
    v = room.as_strided((1, 5, 1, 64), (0, far, 64, 1), 64)
    q, k0, v0 = inputs(torch.bfloat16, 1, 5, 5, 2, 1, 64)
    k.copy_(k0)
    v.copy_(v0)
    if not backward:
        for n in (1, 5):
            near(layers.attention(q[:, :n], k, v)[0], *attention64(q[:, :n], k0, v0)["out"], what="out")
        return
    out, lse = layers.attention(q, k0, v0)
    want = attention64(q, k0, v0, q)
    for name, got in zip(("dq", "dk", "dv"), layers.attention_backward(q, q, k, v, out, lse)):
        near(got, *want[name], what=name)
    qf = room.as_strided((1, 5, 2, 64), (0, far, 64, 1))
    qf.copy_(q)
    for name, got in zip(("dq", "dk", "dv"), layers.attention_backward(qf, qf, k0, v0, out, lse)):
        near(got, *want[name], what=name)


@pytest.mark.parametrize("Lq, Lk", [(0, 5), (5, 0), (0, 0)])
def test_attention_of_nothing(Lq, Lk):
    q, k, v = inputs(torch.float32, 2, Lq, Lk, 4, 2, 32)
    out, lse = layers.attention(q, k, v)
    assert out.shape == q.shape and bool((out == 0).all()) and bool((lse == -math.inf).all())
    dq, dk, dv = layers.attention_backward(out, q, k, v, out, lse)
    assert bool((dq == 0).all()) and dk.shape == k.shape and bool((dk == 0).all()) and bool((dv == 0).all())
    out, lse = layers.attention(q[:0], k[:0], v[:0])
    assert out.shape[0] == 0 and lse.shape[0] == 0
    assert layers.attention_backward(out, q[:0], k[:0], v[:0], out, lse)[0].shape[0] == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Lq, G, Lk", [(1, 1, 1000), (1, 8, 3000), (4, 4, 2500), (1, 32, 700), (5, 3, 64), (1, 40, 900)])
def test_attention_of_single_tokens_on_a_cache(dtype, Lq, G, Lk):
    B = 3
    q, k, v = inputs(dtype, B, Lq, Lk, 2 * G, 2, 128)
    lengths = torch.tensor([Lk, Lk // 2 + 1, Lq], dtype=torch.int32, device=DEV)
    for masks in (dict(), dict(key_lengths=lengths), dict(causal=True, query_start=lengths - Lq, key_lengths=lengths)):
        out, lse = layers.attention(q, k, v, **masks)
        want = attention64(q, k, v, **masks)
        near(out, *want["out"], what="out")
        near(lse, *want["lse"], what="lse")


def test_attention_gradient_against_differences():
    """<gradient, direction> against central differences of the 64-bit forward, h = 1e-5: their own error is h^2 / 6 times
    a third derivative of order 10 and 2^-53 |loss| / h, below 1e-8 of values of order 10."""
    q, k, v = inputs(torch.float32, 2, 20, 30, 4, 2, 16)
    g = torch.Generator(DEV).manual_seed(1)
    dout = torch.randn(q.shape, generator=g, device=DEV)
    masks = dict(causal=True)
    out, lse = layers.attention(q, k, v, **masks)
    grads = layers.attention_backward(dout, q, k, v, out, lse, **masks)
    bounds = attention64(q, k, v, dout, **masks)
    at = [t.double() for t in (q, k, v)]

    def loss(ts):
        see = visible(2, 20, 30, **masks)[:, None]
        Q, K, V = (t.repeat_interleave(4 // t.shape[2], 2).permute(0, 2, 1, 3).contiguous() for t in ts)
        P = torch.softmax(torch.where(see, Q @ K.transpose(2, 3).contiguous() * 0.25, -1e300), -1)
        return ((P @ V).permute(0, 2, 1, 3) * dout.double()).sum()

    h = 1e-5
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(at[i].shape, generator=g, device=DEV, dtype=torch.float64)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * d, at[i] - h * d
        slope = float((loss(up) - loss(down)) / (2 * h))
        got = float((grads[i].double() * d).sum())
        assert abs(got - slope) <= float((bounds[name][1] * d.abs()).sum()) + 1e-6, name


def test_attention_runs_on_the_current_stream():
    q, k, v = inputs(torch.bfloat16, 2, 100, 400, 4, 2, 64)
    want = layers.attention(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k2, v2 = k + 0, v + 0                             # made on the side stream: a call elsewhere would race with it
        got = layers.attention(q, k2, v2)
        grads = layers.attention_backward(got[0], q, k2, v2, *got)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for a, b in zip(layers.attention_backward(want[0], q, k, v, *want), grads):
        assert torch.equal(a, b)


def test_attention_gives_the_same_bits_again():
    q, k, v = inputs(torch.float16, 3, 200, 700, 8, 2, 64)
    q1 = q[:, :1]
    first = compare(q, k, v, causal=True) + tuple(layers.attention(q1, k, v))
    for _ in range(3):
        again = compare(q, k, v, causal=True) + tuple(layers.attention(q1, k, v))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# --------------------------------------------------------------------------------------------- rotary ----

def rotary64(x, positions, freqs, interleaved, scale, inverse):
    """Value and bound: the angle is right to f 2 pi / 4 after its reduction, sine and cosine to 2 f each, then two products
    and a sum in fp32, and the rounding to the type."""
    rot = 2 * freqs.shape[0]
    w = positions.double().reshape(-1, x.shape[1], 1, 1) * freqs * (-1 if inverse else 1)
    x = x.double()
    h = x[..., :rot]
    a, b = (h[..., 0::2], h[..., 1::2]) if interleaved else (h[..., :rot // 2], h[..., rot // 2:])
    ra, rb = scale * (a * w.cos() - b * w.sin()), scale * (b * w.cos() + a * w.sin())
    e = (abs(scale) * 8 * F * (a.abs() + b.abs())).expand_as(ra)
    join = (lambda s, t: torch.stack([s, t], -1).flatten(-2)) if interleaved else (lambda s, t: torch.cat([s, t], -1))
    return torch.cat([join(ra, rb), x[..., rot:]], -1), torch.cat([join(e, e), torch.zeros_like(x[..., rot:])], -1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 2, 2), (2, 7, 4, 2, 64, 64), (3, 52, 4, 4, 64, 32), (1, 33, 8, 1, 128, 128),
                                  (2, 5, 3, 2, 24, 24), (2, 5, 3, 2, 20, 6), (1, 9, 2, 1, 80, 16), (1, 3, 2, 1, 1024, 1000)])
def test_rotary(dtype, interleaved, inverse, size):
    B, L, Hq, Hk, D, rot = size
    g = torch.Generator(DEV).manual_seed(4)
    q, k = (torch.randn(B, L, H, D, generator=g, device=DEV).to(dtype) for H in (Hq, Hk))
    freqs, scale = layers.rotary_frequencies(rot, scaling="by_turns", factor=4.0, trained_length=100, device=DEV)
    u = half_step(dtype)
    for positions in (torch.arange(L, device=DEV), torch.randint(-10 ** 6, 10 ** 6, (B, L), generator=g, device=DEV),
                      (torch.arange(B * L, device=DEV).view(B, L) + 2 ** 31 - 5 * B * L).int()):
        got = layers.rotary(q, positions, freqs, k=k, interleaved=interleaved, scale=scale, inverse=inverse)
        for x, y in zip((q, k), got):
            want, e = rotary64(x, positions, freqs, interleaved, scale, inverse)
            near(y, want, e + u * (want.abs() + e) + tiny(dtype), "rotated")
        alone = layers.rotary(q, positions, freqs, interleaved=interleaved, scale=scale, inverse=inverse)
        assert torch.equal(alone, got[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_in_place_in_windows_of_a_projection(dtype):
    g = torch.Generator(DEV).manual_seed(6)
    B, L, H, D = 2, 11, 4, 32
    freqs, scale = layers.rotary_frequencies(16, device=DEV)
    positions = torch.arange(L, device=DEV) + 3
    for off in (0, 1):                                    # on the 16-byte grid, and off it
        room = torch.randn(B * L * 3 * H * D + 1, generator=g, device=DEV).to(dtype)
        qkv = room[off:off + B * L * 3 * H * D].view(B, L, 3 * H, D)
        before = qkv.clone()
        q, k = qkv[:, :, :H], qkv[:, :, H:2 * H]
        want = layers.rotary(q, positions, freqs, k=k)
        got = layers.rotary(q, positions, freqs, k=k, inplace=True)
        assert got[0] is q and got[1] is k
        assert torch.equal(qkv[:, :, :H], want[0]) and torch.equal(qkv[:, :, H:2 * H], want[1])
        assert torch.equal(qkv[:, :, 2 * H:], before[:, :, 2 * H:])
        assert torch.equal(want[0][..., 16:], before[:, :, :H, 16:])


def test_rotary_in_place_beside_each_other_in_a_head():
    """q and k as the two halves of every head's row: windows of one layout that do not overlap."""
    g = torch.Generator(DEV).manual_seed(6)
    room = torch.randn(2, 5, 3, 2, 16, generator=g, device=DEV)
    q, k = room[:, :, :, 0], room[:, :, :, 1]
    freqs, _ = layers.rotary_frequencies(16, device=DEV)
    want = layers.rotary(q, torch.arange(5, device=DEV), freqs, k=k)
    layers.rotary(q, torch.arange(5, device=DEV), freqs, k=k, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_rotary_gradient_is_the_transpose():
    """<R x, y> = <x, R' y>, both sides in 64 bits of fp32 results: bounds of the two add up."""
    g = torch.Generator(DEV).manual_seed(7)
    x, y = (torch.randn(2, 9, 3, 48, generator=g, device=DEV) for _ in range(2))
    freqs, _ = layers.rotary_frequencies(32, device=DEV)
    positions = torch.randint(0, 10 ** 6, (2, 9), generator=g, device=DEV)
    for interleaved in (False, True):
        kw = dict(interleaved=interleaved, scale=1.25)
        a = (layers.rotary(x, positions, freqs, **kw).double() * y.double()).sum()
        b = (x.double() * layers.rotary(y, positions, freqs, inverse=True, **kw).double()).sum()
        room = 0.0
        for s, t, inv in ((x, y, False), (y, x, True)):
            want, e = rotary64(s, positions, freqs, interleaved, 1.25, inv)
            room += float(((e + F * want.abs()) * t.double().abs()).sum())
        assert abs(float(a - b)) <= room


def test_rotary_of_nothing():
    freqs, _ = layers.rotary_frequencies(32, device=DEV)
    assert layers.rotary(torch.zeros(2, 0, 3, 32, device=DEV), torch.arange(0, device=DEV), freqs).shape == (2, 0, 3, 32)


# ---------------------------------------------------------------------------------------------- norms ----

def norm64(x, y, gate, post, weight, bias, kind, alpha, eps, rpc, dh=None, dz=None):
    """Values by the formulas in 64 bits, gradients by autograd in 64 bits; bounds by the same formulas over magnitudes."""
    R, C = x.shape
    leaf = lambda t: None if t is None else t.detach().double().requires_grad_(True)
    X, Y, Gt, Pw, W, Bi = (leaf(t) for t in (x, y, gate, post, weight, bias))
    group = torch.arange(R, device=DEV) // rpc

    def row(t):
        return t if t is None or t.dim() == 1 or t.shape[0] == 1 else t[group]

    def norm(t):
        c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)

    with torch.enable_grad():
        if Y is None:
            h = X
        else:
            u = norm(Y) if Pw is not None else Y
            u = u * Pw if Pw is not None else u
            h = alpha * X + (u if Gt is None else row(Gt) * u)
        z = norm(h)
        z = z if W is None else z * row(W)
        z = z if Bi is None else z + row(Bi)
        res = {"h": h.detach(), "z": z.detach()}
        if dh is not None or dz is not None:
            loss = 0.0
            loss = loss + (h * dh.double()).sum() if dh is not None else loss
            loss = loss + (z * dz.double()).sum() if dz is not None else loss
            named = [(n, t) for n, t in (("dx", X), ("dy", Y), ("dgate", Gt), ("dpost_weight", Pw), ("dweight", W),
                                         ("dbias", Bi)) if t is not None]
            for (n, _), gr in zip(named, torch.autograd.grad(loss, [t for _, t in named], allow_unused=True)):
                res[n] = gr
    # magnitudes.  A sum over a row runs over at most 16 elements a lane and 6 + 16 partial sums, a moment is used as its
    # inverse root: 64 f covers a norm's factor, and the rest of a formula's ten or so operations.
    e = 64 * F
    with torch.no_grad():
        def scales(t, tabs):
            c = t - t.mean(-1, keepdim=True) if kind == "layer" else t
            r = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
            big = tabs + tabs.mean(-1, keepdim=True) if kind == "layer" else tabs
            # relative error of the factor: that of the moment, whose own terms |c| may be off by e big
            loose = 1 + (c.abs() * big).mean(-1, keepdim=True) * r * r
            return c * r, r, big * r, loose

        if Y is None:
            hab = X.abs()
        else:
            if Pw is not None:
                yn, yr, ynab, yl = scales(Y, Y.abs())
                uab = (ynab + yn.abs() * yl) * Pw.abs()
            else:
                uab = Y.abs()
            gab = torch.ones(1, device=DEV, dtype=torch.float64) if Gt is None else row(Gt).abs()
            hab = abs(alpha) * X.abs() + gab * uab
        n, r, nab, loose = scales(h.detach(), hab)
        nab = nab + n.abs() * loose
        wab = torch.ones(1, device=DEV, dtype=torch.float64) if W is None else row(W).abs()
        bab = 0.0 if Bi is None else row(Bi).abs()
        bounds = {"h": e * hab, "z": e * (nab * wab + bab)}
        if dh is not None or dz is not None:
            dab = torch.zeros_like(X) if dh is None else dh.double().abs()
            if dz is not None:
                a = dz.double().abs() * wab
                dab = dab + r * loose * (a + (a.mean(-1, keepdim=True) if kind == "layer" else 0)
                                         + 2 * nab * (a * nab).mean(-1, keepdim=True))
            dab = 2 * dab
            sums = lambda t, p: t.view(1, R, C).sum(1).view(p.shape) if p.dim() == 1 or p.shape[0] == 1 else \
                torch.zeros_like(p, dtype=torch.float64).index_add_(0, group, t)
            bounds["dx"] = e * dab * (1 if Y is None else abs(alpha))
            seq = (64 + R) * F                            # a column's sum: its terms' error and R additions
            if W is not None and dz is not None:
                bounds["dweight"] = seq * sums(dz.double().abs() * nab, W)
            if Bi is not None and dz is not None:
                bounds["dbias"] = seq * sums(dz.double().abs(), Bi)
            if Y is not None:
                duab = dab * gab
                if Gt is not None:
                    bounds["dgate"] = 2 * seq * sums(dab * uab, Gt)
                if Pw is not None:
                    ynab = ynab + yn.abs() * yl
                    bounds["dpost_weight"] = 2 * seq * sums(duab * ynab, Pw)
                    b = duab * Pw.abs()
                    duab = 2 * yr * yl * (b + (b.mean(-1, keepdim=True) if kind == "layer" else 0)
                                          + 2 * ynab * (b * ynab).mean(-1, keepdim=True))
                bounds["dy"] = e * duab
    return res, bounds


def norm_inputs(dtype, stream, R, C, groups, seed=0):
    g = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s, t=torch.float32: torch.randn(*s, generator=g, device=DEV).to(t)
    return dict(x=r(R, C, t=stream) * 2 + 0.25, y=r(R, C, t=dtype), gate=r(groups, C), post=r(C) * 0.2 + 1,
                weight=r(groups, C) * 0.2 + 1, bias=r(groups, C)), r(R, C, t=stream), r(R, C, t=dtype)


def check_norm(a, dh, dz, kind, alpha, rpc, eps=1e-5, norm=True):
    names = dict(gate=a["gate"], post_weight=a["post"], weight=a["weight"], bias=a["bias"], kind=kind, residual_scale=alpha,
                 eps=eps, rows_per_cond=rpc)
    h, z = layers.residual_norm(a["x"], a["y"], **names) if norm else \
        layers.residual_norm(a["x"], a["y"], norm=False, **{k: v for k, v in names.items() if k not in ("weight", "bias")})
    got = layers.residual_norm_backward(dh, dz, a["x"], a["y"], **names)
    res, bounds = norm64(a["x"], a["y"], a["gate"], a["post"], a["weight"], a["bias"], kind, alpha, eps, rpc, dh, dz)
    if a["y"] is None:
        assert h is a["x"]
    got.update(h=h, z=z)
    for name, t in got.items():
        if t is None or res.get(name) is None:
            if t is not None and name in ("dweight", "dbias"):
                assert bool((t == 0).all())
            continue
        near(t, res[name], bounds[name] + half_step(t.dtype) * (res[name].abs() + bounds[name]) + tiny(t.dtype), name)
    return got


PAIRS = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
         (torch.bfloat16, torch.float32), (torch.float16, torch.float32)]


@pytest.mark.parametrize("dtype, stream", PAIRS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("R, C, rpc", [(1, 1, 1), (52, 256, 52), (130, 64, 13), (37, 257, 10), (9, 1024, 9), (21, 1025, 5),
                                       (6, 4096, 3), (5, 4100, 5), (3, 16384, 2), (2, 9999, 2), (700, 24, 3)])
def test_residual_norm_and_gradient(dtype, stream, kind, R, C, rpc):
    groups = -(-R // rpc)
    a, dh, dz = norm_inputs(dtype, stream, R, C, groups)
    for post in (True, False):
        check_norm({**a, "post": a["post"] if post else None}, dh, dz, kind, 0.75, rpc)
    # one gate, weight and bias for all rows; a conditioned gate beside a shared weight
    check_norm({**a, "gate": a["gate"][0], "weight": a["weight"][:1], "bias": a["bias"][:1]}, dh, dz, kind, 1.0, rpc)
    check_norm({**a, "weight": a["weight"][0], "bias": None}, dh, dz, kind, -1.5, rpc)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_parts(kind):
    """The norm before the first block, the residual after the last, gradients of one of the results only."""
    a, dh, dz = norm_inputs(torch.bfloat16, torch.bfloat16, 50, 192, 5)
    none = dict(y=None, gate=None, post=None)
    check_norm({**a, **none}, None, dz, kind, 1.0, 10)
    check_norm({**a, **none}, dh, dz, kind, 1.0, 10)
    check_norm({**a, **none, "weight": None, "bias": None}, None, dz, kind, 1.0, 10)
    check_norm({**a, "weight": None, "bias": None}, dh, None, kind, 0.5, 10, norm=False)
    check_norm(a, dh, None, kind, 0.5, 10)
    check_norm({**a, "gate": None}, None, dz, kind, 0.5, 10)
    check_norm({**a, "gate": None, "post": None, "weight": None, "bias": None}, dh, dz, kind, 0.5, 10)


def test_residual_norm_strides_and_shapes():
    g = torch.Generator(DEV).manual_seed(3)
    room = torch.randn(4, 10, 3 * 64 + 1, generator=g, device=DEV)
    gate = torch.randn(4, 64, generator=g, device=DEV)
    for off in (0, 1):
        x, y = room[:, :, off:off + 64], room[:, :, off + 64:off + 128]
        dz, dh = room[:, :, off + 128:off + 192], y
        h, z = layers.residual_norm(x, y, gate=gate, rows_per_cond=10)
        h2, z2 = layers.residual_norm(x.contiguous(), y.contiguous(), gate=gate, rows_per_cond=10)
        assert h.shape == x.shape and torch.allclose(h, h2, rtol=0, atol=0) and (z - z2).abs().max() < 64 * F * 10
        got = layers.residual_norm_backward(dh, dz, x, y, gate=gate, rows_per_cond=10)
        res, bounds = norm64(x.reshape(40, 64), y.reshape(40, 64), gate, None, None, None, "rms", 1.0, 1e-5, 10,
                             dh.reshape(40, 64), dz.reshape(40, 64))
        for name in ("dx", "dy", "dgate"):
            t = got[name].reshape(res[name].shape)
            near(t, res[name], bounds[name] + F * res[name].abs(), name)


def test_residual_norm_of_extreme_rows():
    """Rows of zeros (the factor is eps^-1/2), of one value (layer norm: zero), far from zero (the mean leaves no room for a
    one-pass variance), and a row with NaN, which stays in its row."""
    x = torch.randn(6, 512, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    x[0] = 0
    x[1] = 3.0
    x[2] = x[2] * 0.01 + 1000.0
    for kind in ("rms", "layer"):
        check_norm(dict(x=x, y=None, gate=None, post=None, weight=None, bias=None), None, torch.ones_like(x), kind, 1.0, 6)
    x[3, 100] = math.nan
    _, z = layers.residual_norm(x, kind="layer")
    assert bool(torch.isnan(z[3]).all()) and bool(torch.isfinite(z[[0, 1, 2, 4, 5]]).all())


def test_residual_norm_of_more_rows_than_one_launch_holds():
    """2^23 rows of one column go out in a launch."""
    x = torch.randn(2 ** 23 + 5, 1, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    _, z = layers.residual_norm(x, kind="rms")
    want = x.double() / torch.sqrt(x.double() ** 2 + 1e-5)
    near(z, want, 8 * F * want.abs(), "z")


def test_residual_norm_of_nothing():
    x = torch.zeros(0, 32, device=DEV)
    w = torch.ones(32, device=DEV)
    h, z = layers.residual_norm(x, x, gate=w, weight=w)
    assert h.shape == z.shape == (0, 32)
    got = layers.residual_norm_backward(x, x, x, x, gate=w, weight=w)
    assert bool((got["dgate"] == 0).all()) and bool((got["dweight"] == 0).all()) and got["dx"].shape == (0, 32)


def test_residual_norm_gives_the_same_bits_again():
    a, dh, dz = norm_inputs(torch.float32, torch.float32, 5200, 256, 100)
    first = check_norm(a, dh, dz, "layer", 1.0, 52)
    again = check_norm(a, dh, dz, "layer", 1.0, 52)
    shared = [check_norm({**a, "gate": a["gate"][0], "weight": a["weight"][0], "bias": a["bias"][0]}, dh, dz, "layer", 1.0, 52)
              for _ in range(2)]
    for p, q in ((first, again), shared):
        assert all(torch.equal(p[n], q[n]) for n in p)


# --------------------------------------------------------------------------------- together, in graphs ----

def block(p, x, cond, keep):
    """One attention block over the tokens of x (B, L, C), the plain products by torch: norm, projection, rotary, attention,
    projection, gated residual and norm.  Returns h and z; `keep` gets what the gradient needs."""
    B, L, C = x.shape
    H, D = 4, C // 4
    _, z0 = layers.residual_norm(x, weight=cond[0], bias=cond[1], kind="layer", rows_per_cond=L)
    qkv = (z0.view(-1, C) @ p["in"]).view(B, L, 3 * H, D)
    q, k = layers.rotary(qkv[:, :, :H], p["pos"], p["freqs"], k=qkv[:, :, H:2 * H])
    v = qkv[:, :, 2 * H:]
    o, lse = layers.attention(q, k, v, key_mask=p["mask"])
    y = (o.view(-1, C) @ p["out"]).view(B, L, C)
    h, z = layers.residual_norm(x, y, gate=cond[2], weight=p["w"], kind="layer", rows_per_cond=L)
    keep.update(x=x, q=q, k=k, v=v, o=o, lse=lse, y=y)
    return h, z


def block_backward(p, dh, dz, cond, s):
    B, L, C = s["x"].shape
    g = layers.residual_norm_backward(dh, dz, s["x"], s["y"], gate=cond[2], weight=p["w"], kind="layer", rows_per_cond=L)
    do = (g["dy"].view(-1, C) @ p["out"].t().contiguous()).view(s["o"].shape)
    dq, dk, dv = layers.attention_backward(do, s["q"], s["k"], s["v"], s["o"], s["lse"], key_mask=p["mask"])
    dq, dk = layers.rotary(dq, p["pos"], p["freqs"], k=dk, inverse=True)
    dz0 = (torch.cat([dq, dk, dv], 2).view(-1, 3 * C) @ p["in"].t().contiguous()).view(B, L, C)
    g0 = layers.residual_norm_backward(g["dx"], dz0, s["x"], weight=cond[0], bias=cond[1], kind="layer", rows_per_cond=L)
    return g0["dx"], g["dgate"], g0["dweight"], g0["dbias"], g["dweight"]


def block_setup(seed=0, B=6, L=52, C=128):
    g = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    freqs, _ = layers.rotary_frequencies(16, device=DEV)
    mask = torch.rand(B, L, generator=g, device=DEV) < 0.8
    mask[0] = False
    p = {"in": r(C, 3 * C) / C ** 0.5, "out": r(C, C) / C ** 0.5, "w": 1 + 0.1 * r(C), "pos": torch.arange(L, device=DEV),
         "freqs": freqs, "mask": mask}
    cond = [1 + 0.1 * r(B, C), 0.1 * r(B, C), r(B, C)]
    return p, cond, r(B, L, C), r(B, L, C), r(B, L, C)


def test_block_and_its_gradient_against_autograd_in_64_bits():
    """fp32 through the whole block.  Every operator is right to about 1e-6 of its result's size (sums of 128 terms: 128 f =
    8e-6 at the very most) and none amplifies an error by more than a few: the norms divide by a spread of about 1, the softmax's
    scores are of order 1.  Eight operators each way, a factor of 4 apiece for the gradient: 8 * 4 * 8e-6 < 3e-4 in the 2-norm."""
    p, cond, x, dh, dz = block_setup()
    keep = {}
    h, z = block(p, x, cond, keep)
    got = block_backward(p, dh, dz, cond, keep)
    B, L, C = x.shape
    leaves = [t.double().requires_grad_(True) for t in (x, cond[2], cond[0], cond[1], p["w"])]
    X, G, W0, B0, W = leaves

    def ln(t):
        c = t - t.mean(-1, keepdim=True)
        return c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5)

    with torch.enable_grad():
        z0 = ln(X) * W0[:, None] + B0[:, None]
        qkv = (z0.view(-1, C) @ p["in"].double()).view(B, L, 12, C // 4).permute(0, 2, 1, 3)
        w = p["pos"].double()[:, None] * p["freqs"]

        def turn(t):
            a, b = t[..., :8], t[..., 8:16]
            return torch.cat([a * w.cos() - b * w.sin(), b * w.cos() + a * w.sin(), t[..., 16:]], -1)

        q, k, v = turn(qkv[:, :4]), turn(qkv[:, 4:8]), qkv[:, 8:].contiguous()
        S = q @ k.transpose(2, 3).contiguous() * (C // 4) ** -0.5
        E = torch.exp(S - S.detach().amax(-1, keepdim=True)) * p["mask"][:, None, None]
        t = E.sum(-1, keepdim=True)
        o = (E / torch.where(t == 0, 1.0, t)) @ v
        y = (o.permute(0, 2, 1, 3).reshape(-1, C) @ p["out"].double()).view(B, L, C)
        h64 = X + G[:, None] * y
        z64 = ln(h64) * W
        want = torch.autograd.grad((h64 * dh.double()).sum() + (z64 * dz.double()).sum(), leaves)
    for name, a, b in (("h", h, h64.detach()), ("z", z, z64.detach())) + tuple(
            zip(("dx", "dgate", "dscale", "dshift", "dweight"), got, want)):
        assert float((a.double() - b).norm() / b.norm()) < 3e-4, name


def test_block_in_graphs():
    """Two captured graphs of the block and its gradient, replayed in turn with new inputs and eager calls in between: every
    replay gives the eager call's bits."""
    made = []
    side = torch.cuda.Stream()
    for seed in (1, 2):
        p, cond, x, dh, dz = block_setup(seed)

        def call(p=p, cond=cond, x=x, dh=dh, dz=dz):           # of this setup, not the loop's next
            keep = {}
            h, z = block(p, x, cond, keep)
            return (h, z) + block_backward(p, dh, dz, cond, keep)

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = call()
        made.append((graph, held, call, x, cond))
    g = torch.Generator(DEV).manual_seed(8)
    for turn in range(4):
        for graph, held, call, x, cond in made:
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
            cond[2].copy_(torch.randn(cond[2].shape, generator=g, device=DEV))
            want = call()
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(want, held):
                assert torch.equal(a, b)
