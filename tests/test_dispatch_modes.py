"""Calls inside transforms, dispatch modes and graph capture, on the CPU: what is asked before a kernel may take an operator."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from tensor_parallel_b200 import build
from tensor_parallel_b200.ops import functional as OF


class _Watch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _under_mode(f, x):
    with _Watch():
        f(x)


SURROUNDINGS = {
    "make_fx": lambda f, x: make_fx(f, tracing_mode="real")(x),
    "make_fx, before dispatch": lambda f, x: make_fx(f, pre_dispatch=True)(x),
    "functionalized": lambda f, x: torch.func.functionalize(f)(x),
    "a mode": _under_mode,
    "vmap": lambda f, x: torch.vmap(f)(x),
    "grad": lambda f, x: torch.func.grad(lambda t: f(t).sum())(x),
}


@pytest.mark.skipif(not build.AUTOGRAD_PATH.exists(), reason="native module not built")
@pytest.mark.parametrize("around", list(SURROUNDINGS))
def test_the_native_calls_know_what_goes_on_around_them(around):
    from tensor_parallel_b200.ops import native

    plain, seen = torch.ones(2, 4), []

    def f(x):
        # (asked of a tensor that the surroundings have not wrapped: what they do is known to the thread, not to the tensor)
        seen.append((native.AUTOGRAD.interposed(), OF.transformed(plain)))
        return x + 1

    SURROUNDINGS[around](f, torch.ones(2, 4))
    assert seen == [(True, True)]
    assert not native.AUTOGRAD.interposed() and not OF.transformed(plain)


class _OnGpu:
    is_cuda = True


CAPTURES = {
    "make_fx": lambda f, x: make_fx(f, tracing_mode="real")(x),
    "make_fx, before dispatch": lambda f, x: make_fx(f, pre_dispatch=True)(x),
    "fake tensors": lambda f, x: make_fx(f, tracing_mode="fake")(x),
    "functionalized": lambda f, x: make_fx(torch.func.functionalize(f))(x),
}


@pytest.mark.skipif(not build.LIB_PATH.exists(), reason="native library not built")
@pytest.mark.parametrize("asks", ["module", "python"])
@pytest.mark.parametrize("around", list(CAPTURES))
def test_no_kernel_is_taken_while_operators_are_captured(around, asks, monkeypatch):
    from tensor_parallel_b200.ops import native

    if asks == "python":  # (as without the C++ module)
        monkeypatch.setattr(native, "captured", native._captured)
    monkeypatch.setattr(OF, "_FORCE_TORCH", False)
    seen = []

    def f(x):
        seen.append(OF._native(_OnGpu()))
        return x + 1

    CAPTURES[around](f, torch.ones(2, 4))
    assert seen == [None]
    with _Watch():  # (a mode that captures nothing)
        assert OF._native(_OnGpu()) is native
    assert OF._native(_OnGpu()) is native


def test_no_kernel_is_taken_while_a_model_is_exported(monkeypatch):
    if not build.LIB_PATH.exists():
        pytest.skip("native library not built")
    monkeypatch.setattr(OF, "_FORCE_TORCH", False)
    seen = []

    class Model(torch.nn.Module):
        def forward(self, x):
            seen.append(OF._native(_OnGpu()))
            return x + 1

    torch.export.export(Model(), (torch.ones(2, 4),), strict=False)
    assert seen and set(seen) == {None}
