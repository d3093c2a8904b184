"""Operators of attention blocks on the library's kernels (include/trace_hip.h): attention, rotary positions, and the
norms before and after a block fused with its gate and the residual connection -- what a denoiser that attends along the
horizon, or over the agents of a scene, runs between its plain products.

Each comes as a forward and an explicit gradient, as the sampler's own steps do (clean guidance differentiates the denoiser,
tbsim/models/trace.py:630,640-649); nothing is recorded for autograd, and a tensor that asks for it is refused.
Tensors are fp32, bf16 or fp16 on one GPU.  Calls only enqueue, on the current stream of that GPU; results and workspaces come
from torch's allocator, so a call can be captured into a graph.  The same call gives the same bits.
"""
import ctypes as C
import math

import torch
from torch.autograd import forward_ad

from . import _cabi

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_NORMS = {"rms": 0, "layer": 1}


def _refuse(text, *args):
    raise ValueError(text % args if args else text)


def _check(name, t, dtype=None, device=None, shape=None, dims=None):
    """Refuses what a kernel cannot take: another type (dtype None: one of the three), device or shape, an innermost
    dimension that is not contiguous, a tensor that autograd would have to record or carry a tangent on for.  (Plain ifs: a small
    call is bound by its time on the host.)"""
    if not isinstance(t, torch.Tensor):
        _refuse("%s must be a tensor", name)
    if t.requires_grad and torch.is_grad_enabled():
        _refuse("%s requires grad: these operators record nothing for autograd; call them under torch.no_grad() and use "
                "their backward functions", name)
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:   # no level: no call
        _refuse("%s has a forward-mode tangent, which these operators do not carry on", name)
    if dtype is None:
        if t.dtype not in _DTYPES:
            _refuse("%s has type %s (float32, bfloat16 or float16)", name, t.dtype)
    elif t.dtype is not dtype:
        _refuse("%s has type %s, expected %s", name, t.dtype, dtype)
    if device is not None and t.device != device:
        _refuse("%s is on %s, expected %s", name, t.device, device)
    s = t.shape
    if shape is not None and s != shape:
        _refuse("%s has shape %s, expected %s", name, tuple(s), tuple(shape))
    if dims is not None and len(s) != dims:
        _refuse("%s has %d dimensions, expected %d", name, len(s), dims)
    if s and s[-1] > 1 and t.stride(-1) != 1:
        _refuse("the last dimension of %s must be contiguous", name)


def _gpu(t):
    if t.device.type != "cuda":
        raise _cabi.TraceHipError("the attention-block operators need GPU tensors (got %s); there is no CPU fallback"
                                  % t.device)


def _enqueue(what, device, *args):
    """The C call `what` on the device's current stream, with the device current."""
    fn = getattr(_cabi.lib(), what)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if rc:
        _cabi.check(rc, what)


def _at(t):
    return None if t is None else t.data_ptr()


# ------------------------------------------------------------------------------------------ attention ----

def _attention_desc(q, k, v, causal, query_start, key_lengths, key_mask, scale, rest):
    _check("q", q, dims=4)
    dtype, device = q.dtype, q.device
    _check("k", k, dtype, device, dims=4)
    B, Lq, Hq, D = q.shape
    _, Lk, Hk, _ = k.shape
    if not 1 <= D <= 128:
        _refuse("head dimension %d unsupported (1..128)", D)
    if k.shape != (B, Lk, Hk, D):
        _refuse("k has shape %s, q %s", tuple(k.shape), tuple(q.shape))
    _check("v", v, dtype, device, k.shape)
    if Hk < 1 or Hq < 1 or Hq % Hk:
        _refuse("%d query heads cannot share %d key heads", Hq, Hk)
    if Lq > 1 << 30 or Lk > 1 << 30:
        _refuse("more than 2^30 tokens")
    scale = D ** -0.5 if scale is None else float(scale)
    if not (math.isfinite(scale) and scale > 0):
        _refuse("scale %g must be positive and finite", scale)
    start = lengths = mask = None
    if query_start is not None:
        if not causal:
            _refuse("query_start has a meaning for causal attention only")
        _check("query_start", query_start, torch.int32, device, (B,))
        start = query_start.data_ptr()
    if key_lengths is not None:
        _check("key_lengths", key_lengths, torch.int32, device, (B,))
        lengths = key_lengths.data_ptr()
    if key_mask is not None:
        _check("key_mask", key_mask, torch.bool, device, (B, Lk))
        mask = key_mask.data_ptr()
    strides = q.stride()[:3] + k.stride()[:3] + v.stride()[:3]
    for t in rest:
        strides += t.stride()[:3]
    return _cabi.AttentionDesc(_DTYPES[dtype], B, Lq, Lk, Hq, Hk, D, scale, 1 if causal else 0, start, lengths, mask,
                               0 if mask is None else key_mask.stride(0), *strides)


def _workspace(desc, backward, device):
    n = _cabi.lib().trace_attention_workspace_bytes(C.byref(desc), backward)
    if n < 0:
        _cabi.check(int(n), "trace_attention_workspace_bytes")
    return (torch.empty(n, dtype=torch.uint8, device=device), n) if n else (None, 0)


def attention(q, k, v, causal=False, query_start=None, key_lengths=None, key_mask=None, scale=None):
    """softmax(scale q k^T) v over the visible keys.

    q (B, Lq, Hq, D), k and v (B, Lk, Hk, D): Hq / Hk consecutive query heads share a key head; D <= 128; any strides with
    the head elements contiguous (windows of one projection's output, say).  scale: D ** -0.5 if None.
    Query i sees key j iff j < key_lengths[b] (int32), key_mask[b, j] (bool) and, if causal, j <= i + query_start[b]
    (int32; None: the last query is at the last key, Lk - Lq).  For one new token a sequence on a cache: Lq = 1 and
    key_lengths.  Keys that no length or mask admits may hold anything, NaN included; keys that only causality hides
    from some queries have to be finite.  Results that an infinite value enters are infinite or NaN.

    Returns out (B, Lq, Hq, D) and lse (B, Hq, Lq) fp32, the log of the softmax's denominator: what attention_backward
    needs.  A query that sees no key gets 0 and -inf."""
    desc = _attention_desc(q, k, v, causal, query_start, key_lengths, key_mask, scale, ())
    _gpu(q)
    device = q.device
    B, Lq, Hq, D = q.shape
    out = torch.empty((B, Lq, Hq, D), dtype=q.dtype, device=device)
    lse = torch.empty((B, Hq, Lq), dtype=torch.float32, device=device)
    desc.out_batch, desc.out_token, desc.out_head = Lq * Hq * D, Hq * D, D
    ws, n = _workspace(desc, 0, device)
    _enqueue("trace_attention", device, C.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
             lse.data_ptr(), _at(ws), n)
    return out, lse


def attention_backward(dout, q, k, v, out, lse, causal=False, query_start=None, key_lengths=None, key_mask=None,
                       scale=None):
    """Gradients (dq, dk, dv) of attention() given dout, its inputs and its results; the probabilities are recomputed.
    Gradients of shared key heads are summed over their query heads.  Queries that see no key and keys that no query sees get
    zero, whatever they (and dout) hold there."""
    _check("q", q, dims=4)
    _check("dout", dout, q.dtype, q.device, q.shape)
    _check("out", out, q.dtype, q.device, q.shape)
    _check("lse", lse, torch.float32, q.device, (q.shape[0], q.shape[2], q.shape[1]))
    if not lse.is_contiguous():
        _refuse("lse must be contiguous")
    desc = _attention_desc(q, k, v, causal, query_start, key_lengths, key_mask, scale, (out, dout))
    _gpu(q)
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    desc.dq_batch, desc.dq_token, desc.dq_head = dq.stride()[:3]
    desc.dk_batch, desc.dk_token, desc.dk_head = dk.stride()[:3]
    desc.dv_batch, desc.dv_token, desc.dv_head = dv.stride()[:3]
    ws, n = _workspace(desc, 1, q.device)
    _enqueue("trace_attention_backward", q.device, C.byref(desc), dout.data_ptr(), q.data_ptr(), k.data_ptr(),
             v.data_ptr(), out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _at(ws), n)
    return dq, dk, dv


# --------------------------------------------------------------------------------------------- rotary ----

def rotary_frequencies(rot, base=10000.0, scaling="none", factor=1.0, trained_length=None, turns_kept=32.0,
                       turns_stretched=1.0, device="cuda"):
    """Angles a position, for rotary(): (freqs (rot / 2) float64 on `device`, scale).  Pair p turns by
    base ** (-2 p / rot) a position.  For contexts `factor` times the trained length:
      "linear"    every angle divided by the factor
      "base"      the base raised by factor ** (rot / (rot - 2)): the slowest pair is stretched by the factor, the fastest not
      "by_turns"  pairs that make at least turns_kept turns over trained_length stay, those below turns_stretched are
                  divided by the factor, a linear ramp in between; scale = 1 + ln(factor) / 10 sharpens the scores"""
    if not (isinstance(rot, int) and rot >= 2 and rot % 2 == 0):
        _refuse("rot %r must be even and positive", rot)
    if scaling not in ("none", "linear", "base", "by_turns"):
        _refuse("unknown scaling %r", scaling)
    if not (base > 1 and factor >= 1):
        _refuse("base %g must be above 1 and factor %g at least 1", base, factor)
    if scaling == "base" and rot == 2:
        _refuse("scaling by the base needs two pairs")
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2))
    f = float(base) ** (-2 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    scale = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "by_turns":
        if trained_length is None or trained_length < 1:
            _refuse("scaling by turns needs the trained length")
        if not turns_kept > turns_stretched:
            _refuse("turns_kept %g must be above turns_stretched %g", turns_kept, turns_stretched)
        ramp = ((trained_length * f / (2 * math.pi) - turns_stretched) / (turns_kept - turns_stretched)).clamp(0, 1)
        f = f * ramp + f / factor * (1 - ramp)
        scale = 1 + 0.1 * math.log(factor)
    return f.to(device), scale


def _extent(t):
    """Elements from the first of t to behind the last."""
    return 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())) if t.numel() else 0


def _folds(t):
    """Whether two elements of t may be the same memory: a dimension that does not reach over those within it."""
    reach = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1) if t.numel() else ():
        if s < reach:
            return True
        reach += (n - 1) * s
    return False


def _share(q, k):
    """Whether q and k (B, L, heads, D), neither of which folds, have an element in common.  Windows of one layout: whether their
    distance is a sum of strides, as often as indices can differ; other pairs count as sharing what they both reach over."""
    size, apart = q.element_size(), k.data_ptr() - q.data_ptr()
    if not (q.numel() and k.numel() and -_extent(k) * size < apart < _extent(q) * size):
        return False
    steps = []
    for sq, nq, sk, nk in zip(q.stride(), q.shape, k.stride(), k.shape):
        if nq > 1 and nk > 1 and sq != sk or apart % size:
            return True
        if nq > 1 or nk > 1:
            steps.append((sq if nq > 1 else sk, 1 - nk, nq - 1))

    def meet(rest, steps):
        if not steps:
            return rest == 0
        s, low, high = steps[0]
        return any(low <= d <= high and meet(rest - d * s, steps[1:]) for d in (rest // s, rest // s + 1))

    return meet(apart // size, sorted(steps, reverse=True))


def rotary(q, positions, freqs, k=None, interleaved=False, scale=1.0, inverse=False, inplace=False):
    """Rotates the first 2 len(freqs) elements of every head of q (B, L, Hq, D), and of k (B, L, Hk, D), by their
    positions: pair (a, b) number p at position t becomes scale (a cos w - b sin w, b cos w + a sin w), w = t freqs[p],
    angles in 64 bits.  Pairs are the two halves' elements p, or elements 2p, 2p + 1 if interleaved.  inverse: -w, which
    is also the gradient (of the same scale).  positions (L) or (B, L), int32 or int64, of any sign; freqs float64.
    inplace: the results replace q and k, which may be windows of one tensor but share no element.  Returns the rotated q, or
    (q, k)."""
    _check("q", q, dims=4)
    device = q.device
    B, L, Hq, D = q.shape
    if k is not None:
        _check("k", k, q.dtype, device, dims=4)
        if k.shape[0] != B or k.shape[1] != L or k.shape[3] != D:
            _refuse("k has shape %s, q %s", tuple(k.shape), tuple(q.shape))
    _check("freqs", freqs, torch.float64, device, dims=1)
    rot = 2 * freqs.shape[0]
    if not 2 <= rot <= D <= 1024:
        _refuse("%d rotated of %d head elements (at most 1024)", rot, D)
    if not (isinstance(positions, torch.Tensor) and positions.dtype in (torch.int32, torch.int64)):
        _refuse("positions must be an int32 or int64 tensor")
    _check("positions", positions, positions.dtype, device)
    if positions.shape != (L,) and positions.shape != (B, L):
        _refuse("positions have shape %s, expected (%d,) or (%d, %d)", tuple(positions.shape), L, B, L)
    if not math.isfinite(scale):
        _refuse("scale is not finite")
    if inplace:
        for name, t in (("q", q), ("k", k)):
            if t is not None and _folds(t):
                _refuse("%s is broadcast or overlaps itself: it cannot be rotated in place", name)
        if k is not None and _share(q, k):
            _refuse("q and k share memory: they cannot be rotated in place together")
    _gpu(q)
    oq = q if inplace else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ok = k if k is None or inplace else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    none = (0, 0, 0)
    desc = _cabi.RotaryDesc(_DTYPES[q.dtype], B, L, Hq, 0 if k is None else k.shape[2], D, rot, 1 if interleaved else 0,
                            1 if inverse else 0, scale, 1 if positions.dtype == torch.int64 else 0,
                            positions.stride(0) if positions.dim() == 2 else 0, *q.stride()[:3],
                            *(none if k is None else k.stride()[:3]), *oq.stride()[:3],
                            *(none if k is None else ok.stride()[:3]))
    _enqueue("trace_rotary", q.device, C.byref(desc), q.data_ptr(), _at(k), positions.data_ptr(), freqs.data_ptr(),
             oq.data_ptr(), _at(ok))
    if inplace:
        for t in (q, k):
            if t is not None and not t.is_inference():
                torch.autograd.graph.increment_version(t)        # who saved it for a backward pass is told there
    return oq if k is None else (oq, ok)


# ---------------------------------------------------------------------------------------------- norms ----

def _row_stride(name, t):
    """The distance of the rows of t (..., C)."""
    if t.is_contiguous():
        return t.shape[-1]
    try:
        return t.view(-1, t.shape[-1]).stride(0)
    except RuntimeError:
        _refuse("%s: the rows of a tensor with strides %s are not evenly spaced", name, t.stride())


def _table(name, t, device, groups, columns):
    """A parameter of (C), (1, C) or a row for each conditioning group: whether it has one for each."""
    _check(name, t, torch.float32, device)
    s = t.shape
    if s != (columns,) and s != (1, columns) and s != (groups, columns):
        _refuse("%s has shape %s, expected (%d,) or (%d, %d)", name, tuple(s), columns, groups, columns)
    if not t.is_contiguous():
        _refuse("%s must be contiguous", name)
    return len(s) == 2 and groups > 1 and s[0] == groups


def _norm_desc(x, y, gate, post_weight, weight, bias, kind, residual_scale, eps, rows_per_cond):
    _check("x", x)
    shape, device = x.shape, x.device
    if not shape or not 1 <= shape[-1] <= 16384:
        _refuse("x has shape %s (1..16384 columns)", tuple(shape))
    columns = shape[-1]
    rows = x.numel() // columns
    if rows >= 1 << 31:
        _refuse("more than 2^31 rows")
    code = stream = _DTYPES[x.dtype]
    ys = 0
    if y is not None:
        _check("y", y, None, device, shape)
        code = _DTYPES[y.dtype]
        if stream and stream != code:
            _refuse("x is %s beside a block output of %s (float32, or the same)", x.dtype, y.dtype)
        ys = _row_stride("y", y)
    elif gate is not None or post_weight is not None:
        _refuse("gate and post_weight belong to a block output y")
    if kind not in _NORMS:
        _refuse("unknown norm %r", kind)
    if not (math.isfinite(eps) and eps >= 0 and math.isfinite(residual_scale)):
        _refuse("eps %g and residual_scale %g must be finite, eps not negative", eps, residual_scale)
    if rows_per_cond is not None and not (isinstance(rows_per_cond, int) and rows_per_cond >= 1):
        _refuse("rows_per_cond %r must be a positive number", rows_per_cond)
    per = min(rows_per_cond or max(rows, 1), max(rows, 1))
    groups = -(-rows // per) if rows else 1
    gate_cond = gate is not None and _table("gate", gate, device, groups, columns)
    if post_weight is not None:
        _table("post_weight", post_weight, device, 1, columns)
    w_cond = weight is not None and _table("weight", weight, device, groups, columns)
    b_cond = bias is not None and _table("bias", bias, device, groups, columns)
    if weight is not None and bias is not None and w_cond != b_cond:
        _refuse("weight and bias must both have a row for each group, or neither")
    return _cabi.NormDesc(code, stream, rows, columns, per, 1 if w_cond or b_cond else 0, 1 if gate_cond else 0,
                          _NORMS[kind], residual_scale, eps, _row_stride("x", x), ys, 0, 0)


def residual_norm(x, y=None, gate=None, post_weight=None, weight=None, bias=None, kind="rms", residual_scale=1.0,
                  eps=1e-5, rows_per_cond=None, norm=True):
    """The norm after a block, its gate, the residual connection and the norm before the next block, in one pass:
      u = N(y) * post_weight  (y itself without post_weight),  h = residual_scale * x + gate * u,  z = N(h) * weight + bias
    over the rows of x and y (..., C): N is the "rms" or "layer" norm of a row.  Without y (before the first block) h is x;
    norm=False (after the last) leaves z out.  gate, weight and bias (fp32) are (C), or (groups, C) with a row for each
    rows_per_cond consecutive rows of x: the scale, shift and gate that a conditioning gives to each trajectory.
    x, the residual stream, has y's type or fp32.  Returns (h, z); h is x where y is None, z None where norm is False."""
    desc = _norm_desc(x, y, gate, post_weight, weight, bias, kind, residual_scale, eps, rows_per_cond)
    if not norm:
        if y is None:
            _refuse("nothing to compute: no block output and no norm")
        if weight is not None or bias is not None:
            _refuse("weight and bias belong to the norm")
    _gpu(x)
    device = x.device
    h = x if y is None else torch.empty(x.shape, dtype=x.dtype, device=device)
    z = torch.empty(x.shape, dtype=x.dtype if y is None else y.dtype, device=device) if norm else None
    _enqueue("trace_residual_norm", device, C.byref(desc), x.data_ptr(), _at(y), _at(gate), _at(post_weight),
             _at(weight), _at(bias), None if y is None else h.data_ptr(), _at(z))
    return h, z


def residual_norm_backward(dh, dz, x, y=None, gate=None, post_weight=None, weight=None, bias=None, kind="rms",
                           residual_scale=1.0, eps=1e-5, rows_per_cond=None):
    """Gradients of residual_norm() given those of its results (either may be None: zero), recomputed from x and y.
    Returns a dict of dx, dy, dgate, dpost_weight, dweight and dbias; None for what the call does not have."""
    desc = _norm_desc(x, y, gate, post_weight, weight, bias, kind, residual_scale, eps, rows_per_cond)
    out = x if y is None else y
    if dh is None and dz is None:
        _refuse("neither dh nor dz")
    if dh is not None:
        _check("dh", dh, x.dtype, x.device, x.shape)
        desc.dh_stride = _row_stride("dh", dh)
    if dz is not None:
        _check("dz", dz, out.dtype, x.device, x.shape)
        desc.dz_stride = _row_stride("dz", dz)
    _gpu(x)
    new = torch.empty if desc.rows and dz is not None else torch.zeros
    got = {"dx": torch.empty(x.shape, dtype=x.dtype, device=x.device),
           "dy": None if y is None else torch.empty(y.shape, dtype=y.dtype, device=x.device)}
    for name, t, f in (("dgate", gate, torch.empty if desc.rows else torch.zeros),
                       ("dpost_weight", post_weight, torch.empty if desc.rows else torch.zeros),
                       ("dweight", weight, new), ("dbias", bias, new)):
        got[name] = None if t is None else f(t.shape, dtype=torch.float32, device=x.device)
    if not desc.rows:
        return got
    n = _cabi.lib().trace_residual_norm_workspace_bytes(C.byref(desc))
    if n < 0:
        _cabi.check(int(n), "trace_residual_norm_workspace_bytes")
    ws = torch.empty(n, dtype=torch.uint8, device=x.device)
    _enqueue("trace_residual_norm_backward", x.device, C.byref(desc), _at(dh), _at(dz), x.data_ptr(), _at(y), _at(gate),
             _at(post_weight), _at(weight), got["dx"].data_ptr(), _at(got["dy"]), _at(got["dgate"]),
             _at(got["dpost_weight"]), _at(got["dweight"]) if dz is not None else None,
             _at(got["dbias"]) if dz is not None else None, ws.data_ptr(), n)
    return got
