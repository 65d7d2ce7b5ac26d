"""Operators inside graph capture and dispatch modes, on the GPU: a captured graph holds the operator's steps, not its first results."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from tensor_parallel_b200.ops import functional as OF

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _randn(*shape, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(BF16)


def _linear(linear):
    return lambda x, w, b: (linear(OF.quantize_int8_ref(x), OF.quantize_int8_ref(w), b, "gelu"),)


# the operator and its definition, of rows [6, 64], a weight [96, 64], a vector of 96 and one of 64
INT8 = {
    "quantize_int8": (lambda x, w, b, g: tuple(OF.quantize_int8(x)), lambda x, w, b, g: tuple(OF.quantize_int8_ref(x))),
    "rms_norm_int8": (lambda x, w, b, g: tuple(OF.rms_norm_int8(x, g, 1e-5, x)[0]), lambda x, w, b, g: tuple(OF.rms_norm_int8_ref(x, g, 1e-5, x)[0])),
    "layer_norm_int8": (lambda x, w, b, g: tuple(OF.layer_norm_int8(x, g, g, 1e-5)[0]), lambda x, w, b, g: tuple(OF.layer_norm_int8_ref(x, g, g, 1e-5)[0])),
    "linear_int8": (lambda x, w, b, g: _linear(OF.linear_int8)(x, w, b), lambda x, w, b, g: _linear(OF.linear_int8_ref)(x, w, b)),
}
CAPTURES = {
    "real": lambda f, *args: make_fx(f, tracing_mode="real")(*args),
    "before dispatch": lambda f, *args: make_fx(f, pre_dispatch=True)(*args),
    "functionalized": lambda f, *args: make_fx(torch.func.functionalize(f))(*args),
    "fake": lambda f, *args: make_fx(f, tracing_mode="fake")(*args),
}


def _inputs(rows, seed):
    return _randn(rows, 64, seed=seed), _randn(96, 64, seed=1), _randn(96, seed=2), _randn(64, seed=3)


@pytest.mark.parametrize("capture", list(CAPTURES))
@pytest.mark.parametrize("name", list(INT8))
def test_a_captured_graph_holds_the_steps_of_the_8_bit_operators(name, capture):
    call, steps = INT8[name]
    graph = CAPTURES[capture](call, *_inputs(6, 10))
    for seed in (11, 12):
        args = _inputs(6, seed)
        # (the graph's steps are the definition's, on the same device: the same bits)
        assert all(torch.equal(a, b) for a, b in zip(graph(*args), steps(*args)))


class _Watch(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("name", list(INT8))
def test_a_mode_sees_the_steps_of_the_8_bit_operators(name):
    call, steps = INT8[name]
    args = _inputs(6, 13)
    with _Watch() as base:
        want = steps(*args)
    with _Watch() as watch:
        got = call(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert [n for n in watch.names if n in set(base.names)] == base.names


OTHERS = {
    "linear": lambda x, w, b, g: OF.linear(x, w, b),
    "rms_norm": lambda x, w, b, g: OF.rms_norm(x, g, 1e-5),
    "layer_norm": lambda x, w, b, g: OF.layer_norm(x, g, g, 1e-5),
    "gelu": lambda x, w, b, g: OF.gelu(x),
    "relu": lambda x, w, b, g: OF.relu(x),
    "swiglu": lambda x, w, b, g: OF.swiglu(x, x * 2),
    "geglu": lambda x, w, b, g: OF.geglu(x, x * 2),
    "rope": lambda x, w, b, g: OF.apply_rope(x.view(1, -1, 1, 64), torch.arange(x.shape[0], device=x.device)[None]),
    "attention": lambda x, w, b, g: OF.attention(*(x.view(1, -1, 1, 64) * s for s in (1, 2, 3)), True),
}


@pytest.mark.parametrize("capture", list(CAPTURES))
@pytest.mark.parametrize("name", list(OTHERS))
def test_a_captured_graph_holds_the_steps_of_the_other_operators(name, capture):
    call = OTHERS[name]
    graph = CAPTURES[capture](call, *_inputs(128, 10))
    for seed in (11, 12):
        args = _inputs(128, seed)
        got, want = graph(*args).float(), call(*args).float()
        # steps against the kernel: a rounding to bf16 on either side (2^-8 of a value each); terms of a sum and probabilities are rounded to bf16 in between, 2^-8 of
        # values up to 16 each
        torch.testing.assert_close(got, want, rtol=2.0 ** -7, atol=2.0 ** -4)


@pytest.mark.parametrize("name", list(INT8))
def test_one_compiled_graph_of_the_8_bit_operators(name):
    call, steps = INT8[name]
    call(*_inputs(6, 14))  # (the native module is loaded)
    torch._dynamo.reset()
    compiled = torch.compile(call, fullgraph=True, backend="eager")
    with torch.no_grad():
        for seed in (15, 16):
            args = _inputs(6, seed)
            assert all(torch.equal(a, b) for a, b in zip(compiled(*args), steps(*args)))
