"""The attention-block operators (trace_amd/layers.py) enqueue on the device of their tensors, with that device current, and on its current
stream, whichever device is current at the call.  Device and stream calls are recorded here; no kernel is launched."""
import pytest
import torch

from trace_amd import _cabi, layers


class _Device:
    """Stands for torch.cuda: which device is current, and which stream each has."""

    def __init__(self, current):
        self.now = current

    def current_device(self):
        return self.now

    def current_stream(self, device):
        return type("Stream", (), {"cuda_stream": 1000 + device.index})

    def device(self, device):
        outer = self

        class Guard:
            def __enter__(self):
                self.was, outer.now = outer.now, device.index

            def __exit__(self, *a):
                outer.now = self.was

        return Guard()


@pytest.mark.parametrize("current", [0, 1])
@pytest.mark.parametrize("fails", [False, True])
def test_calls_go_to_the_device_of_their_tensors(monkeypatch, current, fails):
    calls = []
    cuda = _Device(current)

    class Lib:
        @staticmethod
        def trace_rotary(*args):
            calls.append((cuda.now, args))
            return -2 if fails else 0

        @staticmethod
        def trace_last_error():
            return b"refused"

    monkeypatch.setattr(layers.torch, "cuda", cuda)
    monkeypatch.setattr(_cabi, "lib", lambda: Lib)
    device = torch.device("cuda", 1)
    if fails:
        with pytest.raises(_cabi.TraceHipError):
            layers._enqueue("trace_rotary", device, 7)
    else:
        layers._enqueue("trace_rotary", device, 7)
    assert calls == [(1, (7, 1001))] and cuda.now == current
