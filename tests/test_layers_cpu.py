"""Refusals of the attention-block operators (trace_amd/layers.py, include/trace_hip.h) and the angles of rotary positions:
nothing here needs a GPU, no kernel is launched."""
import ctypes as C
import math

import pytest
import torch

from trace_amd import _cabi, layers

EINVAL, ENOMEM = -1, -3


def _qkv(B=2, Lq=3, Lk=5, Hq=4, Hk=2, D=16, dtype=torch.float32):
    return torch.zeros(B, Lq, Hq, D, dtype=dtype), torch.zeros(B, Lk, Hk, D, dtype=dtype), torch.zeros(B, Lk, Hk, D, dtype=dtype)


def test_tensors_off_the_gpu_are_refused():
    q, k, v = _qkv()
    with pytest.raises(_cabi.TraceHipError, match="no CPU fallback"):
        layers.attention(q, k, v)
    with pytest.raises(_cabi.TraceHipError, match="no CPU fallback"):
        layers.attention_backward(q, q, k, v, q, torch.zeros(2, 4, 3))
    with pytest.raises(_cabi.TraceHipError, match="no CPU fallback"):
        layers.rotary(q, torch.arange(3), torch.ones(8, dtype=torch.float64))
    with pytest.raises(_cabi.TraceHipError, match="no CPU fallback"):
        layers.residual_norm(torch.zeros(3, 8))
    with pytest.raises(_cabi.TraceHipError, match="no CPU fallback"):
        layers.residual_norm_backward(None, torch.zeros(3, 8), torch.zeros(3, 8))


@pytest.mark.parametrize("change, text", [
    (lambda a: a.update(q=a["q"][0]), "dimensions"),
    (lambda a: a.update(k=a["k"][:, :, :, :8]), "shape"),
    (lambda a: a.update(k=a["k"][:1], v=a["v"][:1]), "shape"),
    (lambda a: a.update(v=a["v"][:, :4]), "shape"),
    (lambda a: a.update(v=a["v"].half()), "type"),
    (lambda a: a.update(q=a["q"].double()), "type"),
    (lambda a: a.update(q=a["q"][:, :, :3]), "share"),
    (lambda a: a.update(q=torch.zeros(2, 3, 16, 4).transpose(2, 3)), "contiguous"),
    (lambda a: a.update(q=a["q"].requires_grad_()), "autograd"),
    (lambda a: a.update(scale=0.0), "positive"),
    (lambda a: a.update(scale=float("nan")), "positive"),
    (lambda a: a.update(scale=-1.0), "positive"),
    (lambda a: a.update(query_start=torch.zeros(2, dtype=torch.int32)), "causal"),
    (lambda a: a.update(causal=True, query_start=torch.zeros(2)), "type"),
    (lambda a: a.update(key_lengths=torch.zeros(2, dtype=torch.int64)), "type"),
    (lambda a: a.update(key_lengths=torch.zeros(3, dtype=torch.int32)), "shape"),
    (lambda a: a.update(key_mask=torch.ones(2, 5)), "type"),
    (lambda a: a.update(key_mask=torch.ones(2, 4, dtype=torch.bool)), "shape"),
    (lambda a: a.update(zip("qkv", _qkv(D=129))), "head dimension"),
])
def test_attention_refuses(change, text):
    a = dict(zip("qkv", _qkv()))
    change(a)
    with pytest.raises(ValueError, match=text):
        layers.attention(**a)
    q = a["q"].detach()
    if q.dim() == 4 and text != "autograd":
        with pytest.raises(ValueError, match=text):
            layers.attention_backward(dout=q, out=q, lse=torch.zeros(q.shape[0], q.shape[2], q.shape[1]), **a)


def test_attention_backward_refuses_results_of_another_call():
    q, k, v = _qkv()
    lse = torch.zeros(2, 4, 3)
    for bad in (dict(dout=q[:, :2]), dict(out=q.half()), dict(lse=lse.half()), dict(lse=lse.transpose(1, 2)),
                dict(lse=torch.zeros(2, 3, 4).transpose(1, 2))):
        with pytest.raises(ValueError):
            layers.attention_backward(**{**dict(dout=q, q=q, k=k, v=v, out=q, lse=lse), **bad})


@pytest.mark.parametrize("change, text", [
    (lambda a: a.update(q=a["q"][0]), "dimensions"),
    (lambda a: a.update(k=a["k"][:, :2]), "shape"),
    (lambda a: a.update(freqs=a["freqs"].float()), "type"),
    (lambda a: a.update(freqs=torch.ones(9, dtype=torch.float64)), "rotated"),
    (lambda a: a.update(freqs=torch.ones(0, dtype=torch.float64)), "rotated"),
    (lambda a: a.update(positions=torch.zeros(3)), "int32 or int64"),
    (lambda a: a.update(positions=torch.arange(4)), "shape"),
    (lambda a: a.update(positions=torch.zeros(3, 3, dtype=torch.int64)), "shape"),
    (lambda a: a.update(scale=float("inf")), "finite"),
    (lambda a: a.update(k=a["k"][:, :, :1].expand(2, 3, 2, 16), inplace=True), "broadcast"),
    (lambda a: a.update(k=a["q"], inplace=True), "share memory"),
    (lambda a: a.update(k=a["q"][:, :, 2:], inplace=True), "share memory"),
])
def test_rotary_refuses(change, text):
    a = dict(q=torch.zeros(2, 3, 4, 16), k=torch.zeros(2, 3, 2, 16), positions=torch.arange(3),
             freqs=torch.ones(8, dtype=torch.float64))
    change(a)
    with pytest.raises(ValueError, match=text):
        layers.rotary(**a)


@pytest.mark.parametrize("change, text", [
    (lambda a: a.update(y=a["y"][:5]), "shape"),
    (lambda a: a.update(x=a["x"].half()), "beside"),
    (lambda a: a.update(y=None), "belong"),
    (lambda a: a.update(gate=torch.ones(2, 8)), "shape"),
    (lambda a: a.update(gate=torch.ones(3, 8, dtype=torch.float16)), "type"),
    (lambda a: a.update(weight=torch.ones(8, 3).t()), "contiguous"),
    (lambda a: a.update(weight=torch.ones(3, 8), bias=torch.ones(8)), "both"),
    (lambda a: a.update(post_weight=torch.ones(3, 8)), "post_weight"),
    (lambda a: a.update(kind="group"), "unknown"),
    (lambda a: a.update(eps=-1.0), "eps"),
    (lambda a: a.update(residual_scale=float("nan")), "residual_scale"),
    (lambda a: a.update(rows_per_cond=0), "rows_per_cond"),
    (lambda a: a.update(x=torch.zeros(6, 16)[:, ::2], y=torch.zeros(6, 16)[:, ::2]), "contiguous"),
    (lambda a: a.update(x=torch.zeros(3, 4, 8)[:, :2], y=torch.zeros(3, 2, 8)), "evenly"),
    (lambda a: a.update(x=torch.zeros(1, 16385), y=torch.zeros(1, 16385)), "16384"),
])
def test_residual_norm_refuses(change, text):
    a = dict(x=torch.zeros(6, 8), y=torch.zeros(6, 8), gate=torch.ones(3, 8), rows_per_cond=2)
    change(a)
    with pytest.raises(ValueError, match=text):
        layers.residual_norm(**a)
    with pytest.raises(ValueError, match=text):
        layers.residual_norm_backward(torch.zeros(a["x"].shape), None, **a)


def test_residual_norm_refuses_calls_without_work():
    with pytest.raises(ValueError, match="nothing"):
        layers.residual_norm(torch.zeros(3, 8), norm=False)
    with pytest.raises(ValueError, match="belong"):
        layers.residual_norm(torch.zeros(3, 8), torch.zeros(3, 8), weight=torch.ones(8), norm=False)
    with pytest.raises(ValueError, match="neither"):
        layers.residual_norm_backward(None, None, torch.zeros(3, 8))


def test_rotary_frequencies():
    f, scale = layers.rotary_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and scale == 1.0
    assert float(f[0]) == 1.0 and abs(float(f[16]) - 1e-2) < 1e-17
    g, _ = layers.rotary_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(g, f / 4)
    g, _ = layers.rotary_frequencies(64, scaling="base", factor=4.0, device="cpu")
    assert float(g[0]) == 1.0 and abs(float(f[-1] / g[-1]) - 4.0) < 1e-12
    g, scale = layers.rotary_frequencies(64, scaling="by_turns", factor=8.0, trained_length=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.equal(g[turns <= 1], f[turns <= 1] / 8)
    assert bool((g[1:] < g[:-1]).all()) and scale == 1 + 0.1 * math.log(8.0)
    for bad in (dict(rot=63), dict(rot=64, scaling="cubic"), dict(rot=64, factor=0.5), dict(rot=2, scaling="base"),
                dict(rot=64, scaling="by_turns"), dict(rot=64, base=0.5)):
        with pytest.raises(ValueError):
            layers.rotary_frequencies(device="cpu", **bad)


def _err(L):
    return L.trace_last_error().decode()


def test_c_entries_refuse_bad_descriptors():
    """Every call here ends in the host's checks."""
    L = _cabi.lib()
    buf = torch.zeros(64)
    p = buf.data_ptr()

    def attention(**kw):
        d = _cabi.AttentionDesc(0, 1, 1, 1, 1, 1, 16, 1.0)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    for kw, text in ((dict(dtype=3), "dtype"), (dict(D=0), "head dimension"), (dict(D=129), "head dimension"),
                     (dict(Hq=3, Hk=2), "multiple"), (dict(B=-1), "sizes"), (dict(scale=0.0), "scale"),
                     (dict(scale=float("inf")), "scale"), (dict(Lk=(1 << 30) + 1), "tokens")):
        d = attention(**kw)
        assert L.trace_attention(C.byref(d), p, p, p, p, p, None, 0, None) == EINVAL and text in _err(L)
        assert L.trace_attention_backward(C.byref(d), p, p, p, p, p, p, p, p, p, p, 256, None) == EINVAL and text in _err(L)
        assert L.trace_attention_workspace_bytes(C.byref(d), 1) == EINVAL
    d = attention()
    assert L.trace_attention(None, p, p, p, p, p, None, 0, None) == EINVAL and "null" in _err(L)
    assert L.trace_attention(C.byref(d), p, None, p, p, p, None, 0, None) == EINVAL and "null" in _err(L)
    long = attention(Lq=100, Lk=100)                         # a call that needs a workspace
    assert L.trace_attention_workspace_bytes(C.byref(long), 1) >= 400
    assert L.trace_attention_backward(C.byref(long), p, p, p, p, p, p, p, p, p, None, 0, None) == ENOMEM
    assert "workspace" in _err(L)
    assert L.trace_attention(C.byref(attention(B=0)), None, None, None, None, None, None, 0, None) == 0

    def rotary(**kw):
        d = _cabi.RotaryDesc(0, 1, 1, 1, 0, 16, 16)
        d.scale = 1.0
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    for kw, text in ((dict(dtype=-1), "dtype"), (dict(rot=15), "even"), (dict(rot=18), "rotated"), (dict(D=2048, rot=2), "rotated"),
                     (dict(L=-1), "sizes"), (dict(scale=float("nan")), "scale")):
        assert L.trace_rotary(C.byref(rotary(**kw)), p, None, p, p, p, None, None) == EINVAL and text in _err(L)
    assert L.trace_rotary(C.byref(rotary()), p, None, None, p, p, None, None) == EINVAL and "null" in _err(L)
    assert L.trace_rotary(C.byref(rotary(L=0)), None, None, None, None, None, None, None) == 0

    def norm(**kw):
        d = _cabi.NormDesc(0, 0, 2, 8, 1, 0, 0, 0, 1.0, 1e-5, 8, 8, 8, 8)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    for kw, text in ((dict(dtype=4), "dtype"), (dict(stream_dtype=1), "stream"), (dict(C=0), "columns"),
                     (dict(C=16385), "columns"), (dict(rows_per_cond=0), "rows_per_cond"), (dict(kind=2), "norm"),
                     (dict(eps=-1.0), "eps")):
        d = norm(**kw)
        assert L.trace_residual_norm(C.byref(d), p, None, None, None, None, None, None, p, None) == EINVAL and text in _err(L)
        assert L.trace_residual_norm_workspace_bytes(C.byref(d)) == EINVAL
    d = norm()
    assert L.trace_residual_norm(C.byref(d), p, None, p, None, None, None, None, p, None) == EINVAL and "belong" in _err(L)
    assert L.trace_residual_norm(C.byref(d), p, None, None, None, None, None, None, None, None) == EINVAL
    assert L.trace_residual_norm_backward(C.byref(d), p, None, p, None, None, None, None, p, None, None, None, None, None,
                                          None, 0, None) == ENOMEM and "workspace" in _err(L)
    assert L.trace_residual_norm(C.byref(norm(rows=0)), None, None, None, None, None, None, None, None, None) == 0
