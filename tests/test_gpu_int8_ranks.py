"""The serving engine with 8-bit projections on several ranks: the life of the buffers that the ranks' sums come in, and two GPUs."""
import copy

import pytest
import torch

import tensor_parallel_b200 as tp
from tensor_parallel_b200 import engine_spec
from tensor_parallel_b200.engine import DecoderEngine
from test_gpu_int8_engine import CLOSE, _off, _pair

pytestmark = pytest.mark.gpu


class _OneHeap:
    """Stands in for the communication of two ranks that hold the same partial sums.  As in the real one, what goes in and what comes out lies in two buffers that every call
    uses again, and what a call has left in them is spoilt as soon as it may be: the input when it has been summed, the sum when the next call begins."""

    world, rank, mc_base = 2, 0, 0

    def __init__(self, device, size):
        self._call = 0
        self.staging_in, self.staging_out = (torch.zeros(size, dtype=torch.uint8, device=device) for _ in range(2))
        self.status = torch.zeros(4, dtype=torch.int32, device=device)

    def staging_view(self, which, shape, dtype):
        buf = self.staging_in if which == "in" else self.staging_out
        count = torch.Size(shape).numel() * torch.empty((), dtype=dtype).element_size()
        assert count <= buf.numel()
        return buf[:count].view(dtype).view(shape)

    def all_reduce(self, t):
        self._call += 1
        self.staging_out.fill_(255)  # (bf16 NaN)
        out = self.staging_view("out", t.shape, t.dtype)
        torch.mul(t, 2, out=out)
        self.staging_in.fill_(255)
        return out

    def all_gather(self, t):
        return torch.stack([t, t])

    def check_status(self):
        pass


@pytest.mark.parametrize("family", ["llama", "llama_grouped", "opt", "falcon"])
def test_sums_in_buffers_that_are_used_again(family):
    """Two ranks with half of every row-parallel weight each add up to the whole model, step after step, in the one pair of buffers; on a second prompt too."""
    _, served = _pair(family)
    whole = DecoderEngine(served, max_batch=2, max_seq=96, quantize="int8", use_graph=False)
    halved = copy.deepcopy(served)
    with torch.no_grad():
        for name, p in halved.named_parameters():
            if any(part in name for part in ("o_proj", "down_proj", "out_proj", "fc2", "attention.dense", "dense_4h_to_h")):
                p.mul_(0.5)
    spec = engine_spec.describe(halved, 96)
    spec.head_split = "vocab"
    heap = _OneHeap(torch.device("cuda", 0), 2 * 50 * 512 * 2)
    split = DecoderEngine(halved, heap, max_batch=2, max_seq=96, quantize="int8", use_graph=False, spec=spec)
    for seed in (5, 6):
        ids = torch.randint(0, 1024, (2, 50), generator=torch.Generator().manual_seed(seed)).cuda()
        before = heap._call
        want, got = whole.prefill(ids), split.prefill(ids)
        assert heap._call > before and _off(got[:, :1024], want) < CLOSE / 2  # (the sum is rounded to bf16 once more than in one GEMM)
        for step in range(3):
            for e in (whole, split):
                e.ids[:2].copy_(ids[:, step])
                e.decode_step(2)
            assert _off(split.logits_local[:2], whole.logits_local[:2]) < CLOSE / 2


@pytest.mark.multigpu
@pytest.mark.parametrize("family", ["llama", "falcon"])
def test_two_gpus_follow_one(family):
    """A sequential and a parallel block, split over two GPUs that one thread drives, against the same engine on one: prompt and several steps."""
    from tensor_parallel_b200.engine import EngineGroup

    _, served = _pair(family)
    one = DecoderEngine(copy.deepcopy(served), max_batch=2, max_seq=128, quantize="int8")
    two = tp.tensor_parallel(served.cpu(), ["cuda:0", "cuda:1"])
    ids = torch.randint(0, 1024, (2, 70), generator=torch.Generator().manual_seed(7))
    got = two.prefill(ids, max_new_tokens=16, quantize="int8")
    group = two._engine
    assert isinstance(group, EngineGroup) and group.quantize == "int8"
    assert _off(got[:, :1024], one.prefill(ids.cuda())) < CLOSE / 2
    for step in range(4):
        nxt = ids[:, step]
        one.ids[:2].copy_(nxt)
        one.decode_step(2)
        for e in group.engines:
            e.ids[:2].copy_(nxt)
        group.decode_step(2)
    # (a shard of a head need not be columns of the logits: what the steps left in the caches is looked at through a second prompt behind them)
    more = ids[:, 10:20]
    assert _off(group.prefill(more, base=74)[:, :1024], one.prefill(more.cuda(), base=74)) < CLOSE / 2
    group.check_status()
