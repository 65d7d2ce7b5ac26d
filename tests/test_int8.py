"""8-bit rows and their matrix product on the CPU: the definitions against 64 bits, and what is refused."""
import math

import pytest
import torch

from tensor_parallel_b200 import build
from tensor_parallel_b200.ops import functional as OF

BF16 = torch.bfloat16


def _rows64(v):
    """(values before rounding, scales) in 64 bits."""
    most = v.abs().amax(-1, keepdim=True).clamp_min(1e-30)
    return v / most * 127, (most / 127)[..., 0]


def assert_integers(q, want):
    """``q`` is ``want`` rounded: 64-bit values within 127 * 3 * 2^-24 of a tie (the quotient and the product are rounded once each in fp32, a
    weighted norm's product once more) may go to either side."""
    assert (q.double() - want).abs().max().item() <= 0.5 + 127 * 3 * 2.0 ** -24
    assert q.abs().max() <= 127


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 33), (64,)])
def test_rows_are_rounded_quotients(shape, dtype):
    torch.manual_seed(0)
    x = (torch.randn(shape) * 3).to(dtype)
    q, s = OF.quantize_int8(x)
    want, scale = _rows64(x.double())
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == x.shape and s.shape == x.shape[:-1]
    assert_integers(q, want)
    torch.testing.assert_close(s.double(), scale, rtol=2.0 ** -24, atol=0)
    # every value comes back to within half a step, and the two roundings of the fp32 product
    back = OF.Int8Rows(q, s).dequantize(torch.float64)
    assert ((back - x.double()).abs() <= scale[..., None] * 0.5001).all()


def test_ties_go_to_even_and_extremes_are_127():
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -127.0]])
    q, s = OF.quantize_int8(x)
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, -127]] and s.tolist() == [1.0]


def test_rows_without_values_and_rows_that_are_not_finite():
    x = torch.tensor([[0.0, 0.0, 0.0], [1.0, float("nan"), 2.0], [float("inf"), 1.0, 1.0], [3.4e38, -3.4e38, 1.0], [1e-40, -1e-40, 0.0]])
    q, s = OF.quantize_int8(x)
    assert q.tolist() == [[0, 0, 0], [0, 0, 0], [0, 0, 0], [127, -127, 0], [0, 0, 0]]
    assert math.isfinite(s[0]) and torch.isnan(s[1:3]).all() and torch.isfinite(s[3:]).all()
    q, s = OF.rms_norm_int8(x[:3], torch.ones(3), 1e-6)[0]
    assert not q.any() and math.isfinite(s[0]) and torch.isnan(s[1:]).all()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norms_in_8_bits(dtype, with_residual):
    torch.manual_seed(1)
    x = torch.randn(5, 3, 40).to(dtype)
    res = torch.randn(5, 3, 40).to(dtype) if with_residual else None
    w, b = (1 + 0.1 * torch.randn(40)).to(dtype), (0.1 * torch.randn(40)).to(dtype)
    h = x if res is None else (x.double() + res.double()).to(dtype)
    (q, s), got = OF.rms_norm_int8(x, w, 1e-5, res)
    assert torch.equal(got, h) and (res is not None or got is x)
    hd = h.double()
    v = hd * w.double()
    want, scale = _rows64(v)
    assert_integers(q, want)
    torch.testing.assert_close(s.double(), scale * torch.rsqrt(hd.square().mean(-1) + 1e-5), rtol=2e-6, atol=0)
    (q, s), got = OF.layer_norm_int8(x, w, b, 1e-5, res)
    assert torch.equal(got, h)
    y = torch.nn.functional.layer_norm(hd, (40,), w.double(), b.double(), 1e-5)
    back = OF.Int8Rows(q, s).dequantize(torch.float64)
    assert ((back - y).abs() <= _rows64(y)[1][..., None] * 0.501).all()


@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu", "swiglu16"])
def test_product_of_8_bit_rows(act):
    torch.manual_seed(2)
    x, w = OF.quantize_int8(torch.randn(2, 3, 50)), OF.quantize_int8(torch.randn(64, 50) / 7)
    bias = torch.randn(64).to(BF16)
    residual = None if act == "swiglu16" else torch.randn(2, 3, 64).to(BF16)
    out = OF.linear_int8(x, w, bias, act, residual)
    v = x.dequantize(torch.float64) @ w.dequantize(torch.float64).t() + bias.double()
    if act == "swiglu16":
        g = v.unflatten(-1, (2, 2, 16))
        v = (torch.nn.functional.silu(g[..., 0, :]) * g[..., 1, :]).flatten(-2)
    elif act:
        v = {"relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[act](v)
    if residual is not None:
        v = v + residual.double()
    assert out.dtype == BF16 and out.shape == v.shape
    torch.testing.assert_close(out.double(), v, rtol=2.0 ** -8, atol=1e-4)  # one bf16 rounding, and fp32 around it


def test_sums_of_products_are_exact_to_the_longest_contraction():
    k = OF.INT8_MAX_K
    x = OF.Int8Rows(torch.full((1, k), -128, dtype=torch.int8), torch.ones(1))
    w = OF.Int8Rows(torch.full((1, k), -128, dtype=torch.int8), torch.ones(1))
    assert k * 128 * 128 < 2 ** 31 <= (k + 1) * 128 * 128
    assert OF.linear_int8(x, w).item() == torch.tensor(float(k * 128 * 128)).to(BF16).item()


def _pair():
    return OF.quantize_int8(torch.randn(4, 64)), OF.quantize_int8(torch.randn(32, 64))


def test_refusals_of_rows():
    x = torch.randn(4, 64)
    with pytest.raises(TypeError):
        OF.quantize_int8(x.half())
    with pytest.raises(TypeError):
        OF.quantize_int8(torch.ones(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError):
        OF.quantize_int8(torch.empty(4, 0))
    with pytest.raises(ValueError):
        OF.quantize_int8(torch.tensor(1.0))
    for weight in (torch.ones(63), torch.ones(1, 64)):
        with pytest.raises(ValueError):
            OF.rms_norm_int8(x, weight)
    for residual in (torch.randn(4, 63), torch.randn(64), x.to(BF16)):
        with pytest.raises(ValueError):
            OF.rms_norm_int8(x, None, 1e-6, residual)
    with pytest.raises(ValueError):
        OF.layer_norm_int8(x, torch.ones(64), torch.ones(63))
    leaf = torch.randn(4, 64, requires_grad=True)
    for call in (lambda: OF.quantize_int8(leaf), lambda: OF.rms_norm_int8(leaf, None), lambda: OF.rms_norm_int8(x, torch.ones(64, requires_grad=True)),
                 lambda: OF.layer_norm_int8(x, None, None, residual=leaf)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()


def test_refusals_of_the_product():
    x, w = _pair()
    bad = [
        (x, OF.Int8Rows(w.values[:, :32], w.scales)),                 # another contraction
        (x, OF.Int8Rows(w.values, w.scales[:5])),                     # scales of other rows
        (x, OF.Int8Rows(w.values, w.scales.double())),
        (x, OF.Int8Rows(w.values.to(torch.uint8), w.scales)),
        (OF.Int8Rows(x.values.float(), x.scales), w),
        (OF.Int8Rows(x.values[0], x.scales[0]), w),                   # a single row without its dimension
        (x, OF.Int8Rows(w.values[None], w.scales[None])),
        (OF.Int8Rows(x.values[:, :0], x.scales), OF.Int8Rows(w.values[:, :0], w.scales)),
        (x, OF.Int8Rows(w.values[:0], w.scales[:0])),
    ]
    for a, b in bad:
        with pytest.raises(ValueError):
            OF.linear_int8(a, b)
    long = [OF.Int8Rows(torch.zeros(1, OF.INT8_MAX_K + 1, dtype=torch.int8), torch.ones(1)) for _ in range(2)]
    with pytest.raises(ValueError):
        OF.linear_int8(*long)
    for kw in (dict(bias=torch.zeros(31, dtype=BF16)), dict(bias=torch.zeros(32)), dict(residual=torch.zeros(4, 31, dtype=BF16)), dict(residual=torch.zeros(4, 32)),
               dict(act="tanh"), dict(act="swiglu16", residual=torch.zeros(4, 16, dtype=BF16))):
        with pytest.raises(ValueError):
            OF.linear_int8(x, w, **kw)
    with pytest.raises(ValueError):
        OF.linear_int8(x, OF.Int8Rows(w.values[:30], w.scales[:30]), act="swiglu16")
    with pytest.raises(RuntimeError, match="no gradient"):
        OF.linear_int8(x, w, torch.zeros(32, dtype=BF16, requires_grad=True))


def test_no_tokens():
    x, w = _pair()
    assert OF.linear_int8(OF.Int8Rows(x.values[:0], x.scales[:0]), w).shape == (0, 32)
    q, s = OF.quantize_int8(torch.empty(0, 3, 64))
    assert q.shape == (0, 3, 64) and s.shape == (0, 3)


def test_tangents_are_refused_and_batches_go_through_the_steps():
    import torch.autograd.forward_ad as fwd

    x = torch.randn(4, 8)
    with fwd.dual_level(), pytest.raises(RuntimeError, match="no derivative"):
        OF.quantize_int8(fwd.make_dual(x, torch.ones_like(x)))
    got = torch.vmap(lambda t: tuple(OF.quantize_int8(t)))(x)
    assert torch.equal(got[0], OF.quantize_int8(x).values)


def test_generation_in_8_bits_needs_the_engine():
    import tensor_parallel_b200 as tp
    from tensor_parallel_b200.models.llama import LlamaConfig, LlamaForCausalLM

    model = LlamaForCausalLM(LlamaConfig(vocab_size=64, hidden_size=32, intermediate_size=48, num_hidden_layers=1, num_attention_heads=4)).eval()
    wrapped = tp.tensor_parallel(model, ["cpu"])
    ids = torch.randint(0, 64, (1, 5))
    with pytest.raises(ValueError, match="serving engine"):
        wrapped.generate(ids, max_new_tokens=2, quantize="int8")
    with pytest.raises(ValueError, match="quantize"):
        wrapped.generate(ids, max_new_tokens=2, quantize="fp4")
    assert wrapped.generate(ids, max_new_tokens=2, quantize="bf16").shape == (1, 7)


def _form(tokens, features, k, sms=148):
    import ctypes

    from tensor_parallel_b200.ops import native

    form = (ctypes.c_int * 2)()
    return native.LIB.tpb_gemm_int8_form(tokens, features, k, sms, form), form[0], form[1]


@pytest.mark.skipif(not build.LIB_PATH.exists(), reason="native library not built")
@pytest.mark.parametrize("sms", [148, 132, 20, 2])
def test_every_size_has_a_kernel_that_takes_it(sms):
    for tokens in (1, 2, 16, 17, 32, 33, 64, 65, 128, 129, 300, 512, 1000, 8192, 200000):
        for features in (1, 32, 33, 768, 4096, 4736, 4737, 12288, 22016, 151936):
            for k in (1, 128, 129, 500, 1024, 2048, 4096, 11008, OF.INT8_MAX_K):
                kind, bn, splits = _form(tokens, features, k, sms)
                if kind == 0:
                    assert tokens <= 64
                elif kind == 1:
                    tiles = -(-features // 128) * -(-tokens // bn)
                    assert (bn, splits) in {(32, 1), (32, 2), (32, 4), (64, 1), (64, 2), (64, 4), (64, 8), (128, 1), (128, 2)}
                    assert splits <= -(-k // 128) and (tiles * splits <= sms or (features % 8 and (bn, splits) == (128, 1)))  # (a k-block for every CTA, and one round of CTAs)
                else:
                    assert kind == 2 and tokens > 64 and bn in (128, 160, 192, 224, 256)
    assert _form(0, 1, 1)[0] == _form(1, 1, OF.INT8_MAX_K + 1)[0] == -1


@pytest.mark.skipif(not build.LIB_PATH.exists(), reason="native library not built")
def test_sizes_whose_last_tile_would_not_count_in_32_bits_are_refused():
    assert _form(2 ** 31 - 1, 1, 1)[0] == _form(1, 2 ** 31 - 1, 1)[0] == -1
    assert _form(2 ** 31 - 512, 1, 1)[0] == 2 and _form(1, 2 ** 31 - 512, 1)[0] == 0
