"""What a rotation in place (trace_amd/layers.py) tells autograd, and which tensors it refuses.  No kernel is launched."""
import pytest
import torch

from trace_amd import layers


@pytest.mark.parametrize("both", [False, True])
def test_rotation_in_place_raises_the_version(monkeypatch, both):
    monkeypatch.setattr(layers, "_gpu", lambda t: None)
    monkeypatch.setattr(layers, "_enqueue", lambda *a: None)
    room = torch.zeros(2, 3, 8, 16)
    q, k = room[:, :, :4], room[:, :, 4:] if both else None
    at, freqs = torch.arange(3), torch.ones(8, dtype=torch.float64)
    layers.rotary(q, at, freqs, k=k)
    assert room._version == 0
    layers.rotary(q, at, freqs, k=k, inplace=True)
    assert room._version > 0 and q._version > 0 and (k is None or k._version > 0)
    with torch.inference_mode():
        t = torch.zeros(2, 3, 4, 16)
    layers.rotary(t, at, freqs, inplace=True)             # keeps no version


def test_a_tensor_that_was_saved_is_not_rotated_unnoticed(monkeypatch):
    monkeypatch.setattr(layers, "_gpu", lambda t: None)
    monkeypatch.setattr(layers, "_enqueue", lambda *a: None)
    w = torch.ones(2, 3, 4, 16, requires_grad=True)
    q = torch.ones(2, 3, 4, 16)
    y = (w * q).sum()
    layers.rotary(q, torch.arange(3), torch.ones(8, dtype=torch.float64), inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
