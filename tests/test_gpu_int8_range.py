"""Norms in 8 bits of finite rows whose sums pass the range of fp32, on the GPU: by every kernel, between ordinary rows."""
import pytest
import torch

from tensor_parallel_b200.ops import functional as OF
from test_int8_range import far_rows, layer64, rms64

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
# a row per warp and per few warps, of any alignment; a block per row with 16 and 32 columns a thread; rows that are read again; the ring; persistent blocks
SIZES = [(9, 64, BF16), (9, 250, BF16), (9, 64, torch.float32), (11, 1000, BF16), (9, 2731, BF16), (9, 2048, torch.float32), (700, 5255, BF16), (9, 20000, BF16),
         (9, 40001, BF16), (9, 40000, BF16), (9, 20001, torch.float32), (300, 8192, torch.float32), (300, 4100, torch.float32), (2400, 16640, BF16),
         (5000, 1024, BF16), (1200, 2048, BF16), (1200, 3592, BF16), (1200, 4096, BF16), (1200, 8192, BF16), (620, 11008, BF16), (5000, 8192, BF16)]


def _mixed(rows, cols, dtype):
    """Ordinary rows, and the far ones among them: several in the share of one persistent block, in the first and in the last row; one with a NaN."""
    x = torch.randn(rows, cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(0)).to(dtype)
    at = torch.tensor([0, 1, 2, rows // 3, rows // 2, rows - 3, rows - 2, rows - 1] if rows < 400 else [0, 1, 148, 149, 296, 444, rows - 2, rows - 1], device="cuda")
    x[at] = far_rows(cols, dtype, "cuda")
    x[at[2] + 1, cols // 2] = float("nan")
    return x


def _call(x, norm, weight, bias, residual, dtype):
    """(integers, scales), and what was normalised"""
    from tensor_parallel_b200.ops import native

    if residual is None:
        return (OF.layer_norm_int8(x, weight, bias, 1e-5) if norm else OF.rms_norm_int8(x, weight, 1e-5))
    res = torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    if residual == "apart":
        return OF.layer_norm_int8(x, weight, bias, 1e-5, res) if norm else OF.rms_norm_int8(x, weight, 1e-5, res)
    h = x.clone()
    return native.rows_int8(h, weight, bias, 1e-5, norm, res, h), h


@pytest.mark.parametrize("residual", [None, "apart", "in place"])
@pytest.mark.parametrize("rows,cols,dtype", SIZES)
def test_rms_norm(rows, cols, dtype, residual):
    x = _mixed(rows, cols, dtype)
    w = (1 - 0.5 * torch.rand(cols, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))).to(dtype)
    (q, s), h = _call(x, 0, w, None, residual, dtype)
    assert torch.equal(q, OF.rms_norm_int8_ref(h, w, 1e-5)[0].values)
    squares, beyond, within = rms64(h)
    assert beyond.sum() >= 4 and within.sum() >= rows - 6 and torch.isnan(s[~within]).all()
    want = (h.double() * w.double()).abs().amax(1).clamp_min(1e-30) / 127 * torch.rsqrt(squares / cols + 1e-5)
    # (as for other rows: a sum of squares of 80 roundings of 2^-24 one after the other at most, halved by the root, the root, five more)
    torch.testing.assert_close(s[within].double(), want[within], rtol=64 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("residual", [None, "apart", "in place"])
@pytest.mark.parametrize("rows,cols,dtype", SIZES)
def test_layer_norm(rows, cols, dtype, residual):
    x = _mixed(rows, cols, dtype)
    gen = torch.Generator(device="cuda").manual_seed(2)
    w, b = (1 + 0.1 * torch.randn(cols, device="cuda", generator=gen)).to(dtype), (0.1 * torch.randn(cols, device="cuda", generator=gen)).to(dtype)
    (q, s), h = _call(x, 1, w, b, residual, dtype)
    for lo in range(0, rows, 512):
        part = slice(lo, lo + 512)
        d, squares, beyond = layer64(h[part])
        fine = torch.isfinite(h[part]).all(1) & ~beyond
        assert torch.isnan(s[part][~fine]).all() and torch.isfinite(s[part][fine]).all()
        rstd = torch.rsqrt(squares / cols + 1e-5)[:, None]
        y = d * rstd * w.double() + b.double()
        step = y.abs().amax(1, keepdim=True).clamp_min(1e-30) / 127
        back = q[part].double() * s[part].double()[:, None]
        # half a step and the roundings of y, of the quotient and of the scale; the mean is a sum of 80 roundings of 2^-24 one after the other at most, and what it is
        # off by a small deviation magnifies (weights are below 1.5)
        slack = 80 * 2.0 ** -24 * h[part].double().abs().amax(1, keepdim=True) * rstd * 1.5
        assert ((back - y).abs() <= 0.501 * step + slack)[fine].all()
