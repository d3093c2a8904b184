"""Attention-block operators (trace_amd/layers.py) at sizes and values that nothing else reaches."""
import math

import pytest
import torch

from test_gpu_layers import DEV, F, half_step, near, rotary64, tiny
from trace_amd import layers

pytestmark = pytest.mark.gpu


def test_rotary_of_more_elements_than_32_bits_count():
    """256 tokens, one rotated pair of 1024 elements, 8300 heads: what one workgroup would do, counted in elements, passes 2^31."""
    B, L, H, D = 1, 256, 8300, 1024
    q = torch.empty(B, L, H, D, dtype=torch.float16, device=DEV)
    g = torch.Generator(DEV).manual_seed(1)
    for l in range(L):
        q[0, l] = torch.randn(H, D, generator=g, device=DEV)
    freqs = torch.ones(1, dtype=torch.float64, device=DEV)
    at = torch.arange(L, device=DEV)
    got = layers.rotary(q, at, freqs)
    for l in range(0, L, 32):
        assert torch.equal(got[:, l:l + 32, :, 2:], q[:, l:l + 32, :, 2:])
    want, e = rotary64(q[..., :2], at, freqs, False, 1.0, False)
    near(got[..., :2], want, e + half_step(q.dtype) * (want.abs() + e) + tiny(q.dtype), "rotated")
