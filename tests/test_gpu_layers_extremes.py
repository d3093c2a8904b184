"""Attention-block operators (trace_amd/layers.py) at sizes and values that nothing else reaches."""
import math

import pytest
import torch

from attention_formulas import backward64, forward64
from test_gpu_layers import DEV, half_step, inputs, near, rotary64, tiny
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq, Lk", [(1, 700), (3, 40), (40, 300)])
def test_scores_that_are_infinite_or_nan_stay_in_their_rows(dtype, Lq, Lk):
    """A query with a NaN, and one whose scores reach +inf (inf - inf: NaN, as in the formula): NaN in those rows alone.  A query whose
    scores are all -inf sees nothing of weight."""
    g = torch.Generator(DEV).manual_seed(3)
    B, H, D = 4, 2, 64
    q = torch.randn(B, Lq, 2 * H, D, generator=g, device=DEV).to(dtype)
    k, v = (torch.randn(B, Lk, H, D, generator=g, device=DEV).to(dtype) for _ in range(2))
    k[..., 0] = 1.0
    want, want_lse = layers.attention(q, k, v)
    q[0, 0, 1, 5] = math.nan
    q[1, 0, 2, 0] = math.inf
    q[2, 0, 3, 0] = -math.inf
    out, lse = layers.attention(q, k, v)
    assert bool(out[0, 0, 1].isnan().all()) and bool(lse[0, 1, 0].isnan())
    assert bool(out[1, 0, 2].isnan().all()) and not bool(lse[1, 2, 0].isfinite())
    assert bool((out[2, 0, 3] == 0).all()) and float(lse[2, 3, 0]) == -math.inf
    same = torch.ones(B, Lq, 2 * H, dtype=torch.bool, device=DEV)
    same[0, 0, 1] = same[1, 0, 2] = same[2, 0, 3] = False
    assert torch.equal(out[same], want[same]) and torch.equal(lse.transpose(1, 2)[same], want_lse.transpose(1, 2)[same])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Lq", [1, 40])
def test_an_infinite_value_reaches_its_element_alone(dtype, Lq):
    """Results that an infinite value enters are infinite or NaN (its probability is a sum of two operands, one of which may be zero);
    no others are."""
    g = torch.Generator(DEV).manual_seed(3)
    q = torch.randn(1, Lq, 2, 32, generator=g, device=DEV).to(dtype)
    k, v = (torch.randn(1, 90, 2, 32, generator=g, device=DEV).to(dtype) for _ in range(2))
    want = layers.attention(q, k, v)[0]
    v[0, 66, 1, 5] = math.inf
    out = layers.attention(q, k, v)[0]
    assert not bool(out[0, :, 1, 5].isfinite().any())
    out[0, :, 1, 5] = want[0, :, 1, 5] = 0
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [(1, 33, 6001, 2, 1, 64), (1, 6001, 33, 2, 1, 64), (1, 2500, 2500, 1, 1, 128)])
def test_gradients_of_long_rows(dtype, size):
    """Rows, and columns, of thousands of terms."""
    q, k, v = inputs(dtype, *size)
    dout = inputs(dtype, *size, seed=3)[0]
    out, lse = layers.attention(q, k, v)
    near(out, *forward64(q, k, v)["out"], what="out")
    want = backward64(dout, q, k, v, out, lse)
    for name, got in zip(("dq", "dk", "dv"), layers.attention_backward(dout, q, k, v, out, lse)):
        near(got, *want[name], what=name)


def test_residual_norm_gradient_of_the_most_rows():
    """2^31 - 1 rows of one element, one group: without dz the gradient of x is dh."""
    dh = torch.empty(2 ** 31 - 1, 1, dtype=torch.bfloat16, device=DEV)
    part = torch.randn(2 ** 24 + 3, device=DEV, generator=torch.Generator(DEV).manual_seed(1)).to(dh.dtype)
    for at in range(0, dh.shape[0], part.shape[0]):
        n = min(part.shape[0], dh.shape[0] - at)
        dh[at:at + n, 0] = part[:n]
    got = layers.residual_norm_backward(dh, None, dh)
    assert torch.equal(got["dx"], dh) and got["dy"] is None
