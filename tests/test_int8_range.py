"""Norms in 8 bits of finite rows whose sums pass the range of fp32, on the CPU: their scale is NaN, not the zero that 1 / rms would be."""
import pytest
import torch

from tensor_parallel_b200.ops import functional as OF

BF16 = torch.bfloat16
MOST = torch.finfo(torch.float32).max


def far_rows(cols, dtype, device="cpu"):
    """Rows with sums beyond fp32, but for the last three."""
    x = torch.randn(8, cols, generator=torch.Generator().manual_seed(cols))
    x[0, 0] = 1e25                                     # one large channel
    x[1] = 3e38 * (torch.arange(cols) % 2 * 2.0 - 1)   # both ends of the range
    x[2] *= 1e30
    x[3] = torch.finfo(BF16).max                       # (nothing but its mean, whose sum is beyond)
    x[4] = x[4] * 1e20 + 1e22
    x[5] *= 1e16
    x[6] *= 1e-20
    return x.to(dtype).to(device)


def rms64(h):
    """Sums of squares in 64 bits, and which rows are beyond fp32 by any order of summation, or by none."""
    squares = h.double().square().sum(-1)
    return squares, squares > MOST * 1.001, squares < MOST * 0.999


def layer64(h):
    """The normalised row's parts in 64 bits: deviations and their squares' sums; and which rows are beyond fp32."""
    d = h.double()
    total = d.sum(-1)
    for _ in range(4):  # (each takes off what the mean before was rounded by)
        d = d - d.mean(-1, keepdim=True)
    squares = d.square().sum(-1)
    return d, squares, (squares > MOST * 1.001) | (total.abs() > MOST * 1.001)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("cols", [8, 33, 1000])
def test_rms_norm_rows_beyond_the_range_of_sums(cols, dtype):
    x = far_rows(cols, dtype)
    squares, beyond, within = rms64(x)
    assert beyond.tolist() == [True] * 5 + [False] * 3 and (beyond | within).all()
    for weight in (None, (1 - 0.5 * torch.rand(cols, generator=torch.Generator().manual_seed(1))).to(dtype)):
        (q, s), h = OF.rms_norm_int8(x, weight, 1e-5)
        assert torch.isnan(s[beyond]).all()
        v = x.double() if weight is None else x.double() * weight.double()
        want = v.abs().amax(-1).clamp_min(1e-30) / 127 * torch.rsqrt(squares / cols + 1e-5)
        # (a sum of squares of at most 1000 roundings of 2^-24, halved by the root, five more)
        torch.testing.assert_close(s[within].double(), want[within], rtol=505 * 2.0 ** -24, atol=0)
    w = OF.quantize_int8(torch.randn(16, cols, generator=torch.Generator().manual_seed(2)))
    out = OF.linear_int8(OF.rms_norm_int8(x, None)[0], w)
    assert torch.isnan(out[beyond]).all() and torch.isfinite(out[within]).all()  # (what is computed from such a row says so)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("cols", [8, 33, 1000])
def test_layer_norm_rows_beyond_the_range_of_sums(cols, dtype):
    x = far_rows(cols, dtype)
    d, squares, beyond = layer64(x)
    assert beyond.tolist() == [True] * 5 + [False] * 3
    gen = torch.Generator().manual_seed(2)
    w, b = (1 + 0.1 * torch.randn(cols, generator=gen)).to(dtype), (0.1 * torch.randn(cols, generator=gen)).to(dtype)
    for weight, bias in ((None, None), (w, b)):
        q, s = OF.layer_norm_int8(x, weight, bias, 1e-5)[0]
        assert torch.isnan(s[beyond]).all()
        y = d * torch.rsqrt(squares / cols + 1e-5)[:, None]
        y = y if weight is None else y * weight.double() + bias.double()
        step = y.abs().amax(-1, keepdim=True).clamp_min(1e-30) / 127
        back = q.double() * s.double()[:, None]
        assert ((back - y).abs() <= 0.501 * step)[~beyond].all()  # half a step, and roundings of 127 steps times a few 2^-24
