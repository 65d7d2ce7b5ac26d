"""Early reads behind the row kernels, on the GPU."""
import pytest
import torch

from tensor_parallel_b200.ops import functional as OF

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens", [4, 40])
def test_a_weight_written_two_kernels_before_an_early_product(tokens):
    """The weight's rows, the activation's rows, the product that reads its weight early: the kernel in front of the product is not the one that writes the weight, and
    has waited for that one."""
    from tensor_parallel_b200.ops import native

    gen = torch.Generator(device="cuda").manual_seed(0)
    wide = [torch.randn(8192, 4096, device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2)]
    x = torch.randn(tokens, 4096, device="cuda", generator=gen).to(torch.bfloat16)
    rows = native.rows_int8(x)
    want = [OF.linear_int8_ref(rows, OF.quantize_int8_ref(w)) for w in wide]
    weight, out = native.int8_rows_empty(8192, 4096, "cuda"), [torch.empty(tokens, 8192, device="cuda", dtype=torch.bfloat16) for _ in range(8)]
    torch.cuda.synchronize()
    for i in range(8):
        native.rows_int8(wide[i % 2], out=weight)
        native.rows_int8(x, out=rows)
        native.gemm_int8(rows, weight, out=out[i], early=True)
    torch.cuda.synchronize()
    for i in range(8):
        torch.testing.assert_close(out[i], want[i % 2], rtol=2.0 ** -7, atol=0)  # a rounding to bf16 on either side


def test_rows_that_are_asked_to_let_the_next_kernel_in_ahead():
    from tensor_parallel_b200.ops import native

    gen = torch.Generator(device="cuda").manual_seed(1)
    weight = OF.quantize_int8(torch.randn(4096, 2048, device="cuda", generator=gen).to(torch.bfloat16))
    for rows, cols in ((8, 2048), (5000, 2048), (6000, 11008), (2400, 16384)):  # a block per row, persistent blocks, the ring
        x = torch.randn(rows, cols, device="cuda", generator=gen).to(torch.bfloat16)
        torch.cuda.synchronize()
        y = x * 2  # (what the rows read is written by the kernel in front of them)
        got = native.rows_int8(y, ahead=True)
        normed = native.rows_int8(y, eps=1e-6, norm=0, ahead=True)
        want = OF.quantize_int8_ref(y)
        assert torch.equal(got.values, want.values) and torch.equal(got.scales, want.scales) and torch.equal(normed.values, want.values)
        if cols == 2048:
            product = native.gemm_int8(native.rows_int8(y, ahead=True), weight, early=True)
            torch.testing.assert_close(product, OF.linear_int8_ref(want, weight), rtol=2.0 ** -7, atol=0)
