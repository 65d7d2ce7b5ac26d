"""Order of programmatic launches, checked on the CPU: when a kernel lets the next one in, and who asks for the exception."""
import re
import types

import pytest
import torch

from tensor_parallel_b200 import build
from tensor_parallel_b200.engine import DecoderEngine

needs_library = pytest.mark.skipif(not build.LIB_PATH.exists(), reason="native library not built")


def _code(path):
    return [line for line in (re.sub(r"//.*", "", raw).strip() for raw in path.read_text().splitlines()) if line]


def test_kernels_let_the_next_one_in_behind_their_own_wait():
    """A kernel that reads early promises that it reads nothing the one kernel in front of it writes: that is enough as long as no kernel lets its successor in
    before its own wait, unless it was asked to."""
    found = 0
    for path in sorted(build.CSRC.glob("*.cu")):
        lines = _code(path)
        for before, line in zip(lines, lines[1:]):
            if "pdl_trigger()" not in line:
                continue
            found += 1
            assert before == "pdl_wait();" or line == "if (ahead) pdl_trigger();", f"{path.name}: {before} / {line}"
    assert found >= 8


@needs_library
def test_rows_let_the_next_kernel_in_ahead_only_where_they_are_asked(monkeypatch):
    from tensor_parallel_b200.ops import native

    calls = []
    argtypes = native.LIB.tpb_rows_int8.argtypes
    monkeypatch.setattr(native, "LIB", types.SimpleNamespace(tpb_rows_int8=lambda *args: calls.append(args) or 0))
    monkeypatch.setattr(native, "_stream", lambda: None)
    monkeypatch.setattr(native, "device_state", lambda device: types.SimpleNamespace(status=torch.zeros(4, dtype=torch.int32)))
    x = torch.ones(3, 32, dtype=torch.bfloat16)
    native.rows_int8(x)
    native.rows_int8(x, x[0], None, 1e-5, 0)
    native.rows_int8(x, ahead=True)
    assert all(len(args) == len(argtypes) for args in calls) and [args[-3] for args in calls] == [0, 0, 1]


class _Chain:
    """Stands in for the native module: writes down what an engine's layer asks for."""

    def __init__(self):
        self.rows, self.products = [], []

    def rows_int8(self, x, *args, ahead=False, **kwargs):
        self.rows.append(ahead)
        return x, x

    def gemm_int8(self, x, weight, bias=None, act=None, residual=None, out=None, early=False):
        self.products.append(early)
        return out


def _layer_engine(world, parallel=False):
    engine = DecoderEngine.__new__(DecoderEngine)
    engine.world, engine.parallel, engine.nq, engine.head_dim, engine.mode, engine.eps, engine.act = world, parallel, 1, 8, 1, 1e-5, None
    engine._summed = None
    engine.layers = [dict(wqkv=None, bqkv=None, ln1=(None, None), ln2=(None, None), w1=None, b1=None, wo=None, bo=None, wd=None, bd=None)]
    engine._attend = lambda i, qkv, q_rot, cat, *rest: cat[:, :8]
    engine.comm = types.SimpleNamespace(staging_view=lambda which, shape, dtype: torch.zeros(shape, dtype=dtype), all_reduce=lambda t: t * world)
    return engine


@needs_library
@pytest.mark.parametrize("parallel", [False, True])
@pytest.mark.parametrize("decode", [False, True])
@pytest.mark.parametrize("world", [1, 2])
def test_the_engine_asks_for_it_on_one_rank_only(world, decode, parallel, monkeypatch):
    from tensor_parallel_b200 import engine as module

    chain = _Chain()
    monkeypatch.setattr(module, "native", chain)
    engine = _layer_engine(world, parallel)
    x = torch.zeros(2, 8, dtype=torch.bfloat16)
    engine._int8_layer(0, x, torch.zeros(2, 24), None, torch.zeros(2, 16), torch.zeros(2, 8), 2, 1, decode)
    assert len(chain.rows) == 4 and set(chain.rows) == {world == 1}
    assert set(chain.products) <= {decode and world == 1, False} and (not decode or world > 1 or all(chain.products))


@needs_library
@pytest.mark.parametrize("parallel", [False, True])
def test_a_pass_that_ends_early_leaves_nothing_for_the_next(parallel, monkeypatch):
    """What the ranks' last sum leaves for the next norm belongs to the pass, not to the engine."""
    from tensor_parallel_b200 import engine as module

    class Chain(_Chain):
        def rows_int8(self, x, *args, residual=None, **kwargs):
            self.rows.append(residual is not None)
            return x, x

    class Two(list):  # (and the second is not there)
        def __len__(self):
            return 2

    monkeypatch.setattr(module, "native", chain := Chain())
    engine = _layer_engine(2, parallel)
    one, engine.layers = engine.layers, Two(engine.layers)
    engine.quantize, x = "int8", torch.zeros(2, 8, dtype=torch.bfloat16)
    args = (torch.zeros(2, 24), None, torch.zeros(2, 16), torch.zeros(2, 8), 2, 1, False)
    for _ in range(2):
        chain.rows.clear()
        with pytest.raises(IndexError):
            engine._layers(x, None, *args)
        assert chain.rows[0] is False and sum(chain.rows) == (0 if parallel else 1)
    chain.rows.clear()
    engine.layers = one
    engine._layers(x, None, *args)
    assert chain.rows[0] is False and not x.any()


@needs_library
def test_a_rank_alone_runs_the_tensor_kernels_of_several(monkeypatch):
    """A kernel that is launched for the first time may be loaded then, which may wait for the device: not behind a kernel that waits for a peer which the same thread has yet to
    launch.  So a rank's own passes include the operations that only several ranks take: a bias times the number of ranks, added to all rows."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from tensor_parallel_b200.ops import native

    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types_, args=(), kwargs=None):
            seen.append((func, [tuple(a.shape) for a in args if isinstance(a, torch.Tensor)]))
            return func(*args, **(kwargs or {}))

    monkeypatch.setattr(native, "LIB", types.SimpleNamespace(tpb_gemm_preload=lambda: 0, tpb_comm_preload=lambda: 0, tpb_int8_preload=lambda: 0))
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    engine = types.SimpleNamespace(comm=object(), world=2, head_split="vocab", embed_split=False, max_seq=80, device="cpu", vocab_local=32, x=torch.zeros(1, 8), quantize="int8",
                                   logits_local=torch.zeros(1, 32), pos=torch.zeros(1), ids=torch.zeros(1), prefill=lambda ids: None, _decode_body=lambda batch: None)
    with Watch():
        DecoderEngine.preload(engine)
    assert (torch.ops.aten.mul.Tensor, [(8,)]) in seen and (torch.ops.aten.add_.Tensor, [(2, 8), (8,)]) in seen
