"""8-bit operators under torch.compile and torch.export, on the CPU: one graph of their steps, whether the native module has been loaded or not."""
import pytest
import torch

from tensor_parallel_b200 import build
from tensor_parallel_b200.ops import functional as OF

needs_library = pytest.mark.skipif(not build.LIB_PATH.exists() or not build.AUTOGRAD_PATH.exists(), reason="native library not built")
CALLS = {
    "quantize_int8": lambda x, w: tuple(OF.quantize_int8(x)),
    "rms_norm_int8": lambda x, w: tuple(OF.rms_norm_int8(x, w[0], 1e-5, x)[0]),
    "layer_norm_int8": lambda x, w: tuple(OF.layer_norm_int8(x, w[0], w[1], 1e-5)[0]),
    "linear_int8": lambda x, w: (OF.linear_int8(OF.quantize_int8_ref(x), OF.quantize_int8_ref(w), act="silu"),),
}


def _inputs(seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(5, 64, generator=gen).to(torch.bfloat16), torch.randn(32, 64, generator=gen).to(torch.bfloat16)


def _load(loaded, monkeypatch):
    if loaded:
        from tensor_parallel_b200.ops import native

        monkeypatch.setattr(OF, "quantize_int8_directly", native.AUTOGRAD.quantize_int8)
        monkeypatch.setattr(OF, "norm_int8_directly", native.AUTOGRAD.norm_int8)
        monkeypatch.setattr(OF, "linear_int8_directly", native.AUTOGRAD.linear_int8)
    else:
        for name in ("quantize_int8_directly", "norm_int8_directly", "linear_int8_directly"):
            monkeypatch.setattr(OF, name, OF._not_taken)


def _same(got, want):
    # (the steps, the same operations in the same order)
    return all(torch.equal(a, b) for a, b in zip(got, want))


@needs_library
@pytest.mark.parametrize("loaded", [False, True])
@pytest.mark.parametrize("name", list(CALLS))
def test_one_graph_of_steps(name, loaded, monkeypatch):
    _load(loaded, monkeypatch)
    torch._dynamo.reset()
    call = CALLS[name]
    compiled = torch.compile(call, fullgraph=True, backend="eager")
    with torch.no_grad():
        for seed in (0, 1):
            args = _inputs(seed)
            assert _same(compiled(*args), call(*args))


@needs_library
@pytest.mark.parametrize("name", list(CALLS))
def test_one_graph_of_steps_for_tensors_that_kernels_would_take(name, monkeypatch):
    from tensor_parallel_b200.ops import native

    _load(True, monkeypatch)
    call = CALLS[name]
    with torch.no_grad():
        args = _inputs(2)
        want = call(*args)
        monkeypatch.setattr(OF, "_native", lambda x: native)  # (as for tensors on the GPU)
        torch._dynamo.reset()
        assert _same(torch.compile(call, fullgraph=True, backend="eager")(*args), want)


@needs_library
@pytest.mark.parametrize("strict", [False, True])
@pytest.mark.parametrize("name", list(CALLS))
def test_export(name, strict, monkeypatch):
    _load(True, monkeypatch)
    call = CALLS[name]

    class Model(torch.nn.Module):
        def forward(self, x, w):
            return call(x, w)

    with torch.no_grad():
        program = torch.export.export(Model(), _inputs(3), strict=strict)
        args = _inputs(4)
        assert _same(program.module()(*args), call(*args))
