"""8-bit operators of tensors whose memory holds the negatives of their values (views of conjugates), on the GPU."""
import pytest
import torch

from tensor_parallel_b200.ops import functional as OF

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def _negative(t):
    """The values of ``t``, over memory that holds their negatives."""
    out = torch._neg_view(-t)
    assert out.is_neg() and torch.equal(out.clone(), t)
    return out


@pytest.mark.parametrize("cols", [1, 2, 64])
def test_the_imaginary_part_of_a_conjugate(cols):
    part = torch.complex(_randn(6, cols), _randn(6, cols, seed=1)).conj().imag
    assert part.is_neg()
    got, want = OF.quantize_int8(part), OF.quantize_int8_ref(part.clone())
    assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales) and got.values.any()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
def test_norms(which, dtype):
    args = dict(x=_randn(5, 64, dtype=dtype), weight=_randn(64, seed=1, dtype=dtype), bias=_randn(64, seed=2, dtype=dtype), residual=_randn(5, 64, seed=3, dtype=dtype))
    given = {**args, which: _negative(args[which])}
    for call, names in ((OF.rms_norm_int8, ("weight",)), (OF.layer_norm_int8, ("weight", "bias"))):
        want, got = (call(a["x"], *(a[n] for n in names), 1e-5, a["residual"]) for a in (args, given))
        assert all(torch.equal(a, b) for a, b in zip((*got[0], got[1]), (*want[0], want[1])))  # (the same kernel on the same values)


@pytest.mark.parametrize("which", ["x scales", "weight scales", "bias", "residual"])
def test_the_product(which):
    x, w = OF.quantize_int8(_randn(7, 64)), OF.quantize_int8(_randn(32, 64, seed=1))
    bias, residual = _randn(32, seed=2, dtype=BF16), _randn(7, 32, seed=3, dtype=BF16)
    want = OF.linear_int8(x, w, bias, "gelu", residual)
    if which == "x scales":
        x = OF.Int8Rows(x.values, _negative(x.scales))
    if which == "weight scales":
        w = OF.Int8Rows(w.values, _negative(w.scales))
    got = OF.linear_int8(x, w, _negative(bias) if which == "bias" else bias, "gelu", _negative(residual) if which == "residual" else residual)
    assert torch.equal(got, want)
