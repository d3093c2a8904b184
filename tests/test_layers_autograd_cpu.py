"""The attention-block operators (trace_amd/layers.py) refuse tensors with a forward-mode tangent like those that require grad.  No kernel
is launched."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from trace_amd import layers


def _calls(t):
    q = torch.zeros(2, 3, 4, 16)
    lse, freqs, at = torch.zeros(2, 4, 3), torch.ones(8, dtype=torch.float64), torch.arange(3)
    x, w = torch.zeros(6, 16), torch.ones(16)
    d, e = t(q), t(x)
    return [lambda: layers.attention(d, q, q), lambda: layers.attention(q, d, q), lambda: layers.attention(q, q, d),
            lambda: layers.attention_backward(d, q, q, q, q, lse), lambda: layers.attention_backward(q, q, q, q, d, lse),
            lambda: layers.attention_backward(q, q, q, q, q, t(lse)),
            lambda: layers.rotary(d, at, freqs), lambda: layers.rotary(q, at, freqs, k=d), lambda: layers.rotary(q, at, t(freqs)),
            lambda: layers.rotary(d, at, freqs, inplace=True),
            lambda: layers.residual_norm(e), lambda: layers.residual_norm(x, e), lambda: layers.residual_norm(x, x, gate=t(w)),
            lambda: layers.residual_norm(x, weight=t(w)), lambda: layers.residual_norm_backward(None, e, x),
            lambda: layers.residual_norm_backward(e, None, x)]


@pytest.mark.parametrize("n", range(16))
def test_forward_mode_tangents_are_refused(n):
    with forward_ad.dual_level():
        for quiet in (False, True):                       # no_grad does not put forward mode off
            call = _calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))[n]
            with torch.set_grad_enabled(not quiet), pytest.raises(ValueError, match="tangent"):
                call()
