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


def _windows(room, *at):
    return [room[w] for w in at]


S = slice
ROOM = (2, 6, 8, 16)


@pytest.mark.parametrize("q, k", [
    ((S(None), S(0, 5)), (S(None), S(1, 6))),                             # the next token's heads
    ((S(0, 1),), (S(0, 1), S(None), S(None, None, 2))),                   # every other head of q
    ((S(None), S(None), S(0, 4)), (S(None), S(None), S(3, 7))),           # a head in common
    ((S(None), S(0, 2)), (S(None), S(0, 4, 2))),                          # other tokens
])
def test_queries_and_keys_that_share_memory_are_not_rotated_in_place(monkeypatch, q, k):
    monkeypatch.setattr(layers, "_gpu", lambda t: None)
    monkeypatch.setattr(layers, "_enqueue", lambda *a: None)
    room = torch.zeros(ROOM)
    q, k = _windows(room, q, k)
    at, freqs = torch.arange(q.shape[1]), torch.ones(8, dtype=torch.float64)
    layers.rotary(q, at, freqs, k=k)                      # elsewhere: any windows
    with pytest.raises(ValueError, match="share memory"):
        layers.rotary(q, at, freqs, k=k, inplace=True)
    with pytest.raises(ValueError, match="share memory"):
        layers.rotary(k, at, freqs, k=q, inplace=True)


@pytest.mark.parametrize("sizes, strides", [((2, 5, 4, 16), (64, 16, 16, 1)), ((1, 5, 4, 16), (0, 32, 16, 1)), ((2, 3, 2, 16), (96, 32, 8, 1)),
                                            ((2, 3, 4, 16), (0, 64, 16, 1))])
def test_a_tensor_that_overlaps_itself_is_not_rotated_in_place(monkeypatch, sizes, strides):
    monkeypatch.setattr(layers, "_gpu", lambda t: None)
    monkeypatch.setattr(layers, "_enqueue", lambda *a: None)
    q = torch.zeros(1000).as_strided(sizes, strides)
    other = torch.zeros(sizes)
    at, freqs = torch.arange(sizes[1]), torch.ones(8, dtype=torch.float64)
    for call in (lambda **kw: layers.rotary(q, at, freqs, **kw), lambda **kw: layers.rotary(other, at, freqs, k=q, **kw)):
        call()
        with pytest.raises(ValueError, match="overlap|broadcast"):
            call(inplace=True)


@pytest.mark.parametrize("q, k", [
    ((S(None), S(None), S(0, 4)), (S(None), S(None), S(4, 8))), ((S(None), S(None), S(4, 8)), (S(None), S(None), S(0, 4))),
    ((S(None), S(None), S(0, 7)), (S(None), S(None), S(7, 8))), ((S(None), S(0, 3)), (S(None), S(3, 6))),
    ((S(None), S(None, None, 2)), (S(None), S(1, None, 2))), ((S(None), S(None), S(0, None, 2)), (S(None), S(None), S(1, None, 2))),
    ((S(0, 1),), (S(1, 2),)),
])
def test_windows_that_share_nothing_are_rotated_in_place(monkeypatch, q, k):
    monkeypatch.setattr(layers, "_gpu", lambda t: None)
    monkeypatch.setattr(layers, "_enqueue", lambda *a: None)
    for room in (torch.zeros(ROOM), torch.zeros(2, 8, 6, 16).transpose(1, 2)):
        a, b = _windows(room, q, k)
        layers.rotary(a, torch.arange(a.shape[1]), torch.ones(8, dtype=torch.float64), k=b, inplace=True)
    halves = torch.zeros(2, 5, 3, 2, 16)
    layers.rotary(halves[:, :, :, 0], torch.arange(5), torch.ones(8, dtype=torch.float64), k=halves[:, :, :, 1], inplace=True)
