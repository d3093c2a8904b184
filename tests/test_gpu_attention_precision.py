"""Attention loses nothing of its probabilities and score gradients that a result in its type could show: one rounding, the result's,
is all that tests/attention_formulas.py leaves, on every kernel (few queries, tiles, short sequences, shares)."""
import pytest
import torch

from attention_formulas import backward64, forward64
from test_gpu_layers import DEV, inputs, near
from trace_amd import layers

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(q, k, v, dout, backward=True, **masks):
    out, lse = layers.attention(q, k, v, **masks)
    near(out, *forward64(q, k, v, **masks)["out"], what="out")
    if not backward:
        return
    want = backward64(dout, q, k, v, out, lse, **masks)
    for name, got in zip(("dq", "dk", "dv"), layers.attention_backward(dout, q, k, v, out, lse, **masks)):
        near(got, *want[name], what=name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [
    (2, 1, 300, 8, 2, 64), (1, 16, 500, 2, 2, 128), (2, 52, 52, 4, 2, 64), (2, 64, 40, 2, 2, 128), (1, 20, 33, 4, 4, 32),
    (1, 300, 300, 4, 1, 128), (2, 100, 257, 4, 2, 64), (1, 130, 70, 2, 2, 32), (1, 65, 900, 2, 1, 128), (40, 129, 200, 8, 8, 64),
    (1, 200, 80, 4, 4, 20)])
def test_one_rounding(dtype, causal, size):
    q, k, v = inputs(dtype, *size)
    check(q, k, v, inputs(dtype, *size, seed=3)[0], causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_rounding_under_masks(dtype):
    B, Lq, Lk = 4, 90, 256
    q, k, v = inputs(dtype, B, Lq, Lk, 4, 4, 32)
    mask = torch.rand(B, Lk, generator=torch.Generator(DEV).manual_seed(9), device=DEV) < 0.5
    lengths = torch.tensor([256, 100, 0, 1], dtype=torch.int32, device=DEV)
    dout = inputs(dtype, B, Lq, Lk, 4, 4, 32, seed=3)[0]
    check(q, k, v, dout, key_mask=mask)
    check(q, k, v, dout, key_mask=mask, key_lengths=lengths)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [16, 20, 40, 72, 80])
@pytest.mark.parametrize("off", [0, 1])
def test_one_rounding_of_single_tokens_in_cut_ranges(dtype, D, off):
    """Head sizes below the padded ones, and caches off the 16-byte grid, where ranges of the keys are joined."""
    B, Lk, H = 2, 1500, 2
    g = torch.Generator(DEV).manual_seed(1)
    k, v = (torch.randn(B, Lk, H, D + 8, generator=g, device=DEV).to(dtype)[..., off:off + D] for _ in range(2))
    lengths = torch.tensor([Lk, 700], dtype=torch.int32, device=DEV)
    for Lq, Hq in ((1, 2), (1, 16), (4, 6)):
        q = torch.randn(B, Lq, Hq, D, generator=g, device=DEV).to(dtype)
        check(q, k, v, None, backward=False, key_lengths=lengths)


@pytest.mark.parametrize("size", [(2, 40, 40, 2, 2, 64), (2, 30, 20, 4, 4, 128), (2, 24, 30, 4, 2, 128), (1, 64, 20, 4, 1, 128), (2, 52, 52, 4, 2, 32),
                                  (2, 30, 33, 2, 2, 20), (1, 100, 70, 4, 2, 64), (1, 65, 900, 2, 1, 128), (40, 129, 200, 8, 8, 64)])
@pytest.mark.parametrize("v, dout, qk, causal", [(4.0, 1000.0, 1.0, False), (8.0, 8000.0, 0.02, True), (1.0, 2.0 ** 12, 0.5, False),
                                                 (1.0, 2.0 ** -10, 1.0, True)])
def test_fp16_gradients_of_a_scaled_loss(size, v, dout, qk, causal):
    """dout . v far above what fp16 holds (and far below 1), gradients that it holds: rows and heads of different sizes."""
    q, k, w = inputs(torch.float16, *size)
    d = inputs(torch.float16, *size, seed=3)[0].float() * dout
    d = d * torch.linspace(0.1, 1, size[3], device=DEV)[:, None] * torch.linspace(1, 0.2, size[1], device=DEV)[:, None, None]
    check(q * qk, k * qk, w * v, d.half(), causal=causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(1, 40, 40, 2, 2, 64), (1, 30, 20, 4, 4, 128), (1, 100, 170, 4, 2, 64)])
def test_a_row_of_infinite_gradients_is_alone_in_dq(dtype, size):
    """dout infinite in one row: the other rows' dq keep their bits (fp16's scale does not go by it)."""
    q, k, v = inputs(dtype, *size)
    dout = inputs(dtype, *size, seed=3)[0] * 100
    out, lse = layers.attention(q, k, v)
    want = layers.attention_backward(dout, q, k, v, out, lse)
    dout[0, 7, 1] = float("inf")
    got = layers.attention_backward(dout, q, k, v, out, lse)
    assert not bool(torch.isfinite(got[0][0, 7, 1]).any())
    other = torch.ones(size[1], size[3], dtype=torch.bool, device=DEV)
    other[7, 1] = False
    assert torch.equal(got[0][0][other], want[0][0][other])
    heads = [h for h in range(size[4]) if h != 1 // (size[3] // size[4])]
    for a, b in zip(got[1:], want[1:]):
        assert torch.equal(a[:, :, heads], b[:, :, heads])
        assert not bool(torch.isfinite(a[:, :, 1 // (size[3] // size[4])]).any())
