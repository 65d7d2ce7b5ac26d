"""The serving engine with 8-bit projections, against the fp32 module-level forward of the same (bf16-rounded) weights.

Tolerances: rounding a row to 8 bits is off by a step / sqrt(12) in the mean, a step being its largest value / 127.  The rows here are about normal and
up to 1400 long, so that their largest value is about 3.5 deviations and the error 0.8 % of their size, for weights and activations alike: 1.2 % for a
projection.  A model of three layers has twelve of them on its residual stream, 4 % in the root of the sum of squares; twice that is allowed."""
import copy

import pytest
import torch

import tensor_parallel_b200 as tp
from tensor_parallel_b200.engine import DecoderEngine
from tensor_parallel_b200.models.falcon import FalconConfig, FalconForCausalLM
from tensor_parallel_b200.models.llama import LlamaConfig, LlamaForCausalLM
from tensor_parallel_b200.models.opt import OPTConfig, OPTForCausalLM

pytestmark = pytest.mark.gpu
CLOSE = 0.08


def _llama(kv_heads=4, ffn=1376):
    return LlamaForCausalLM(LlamaConfig(vocab_size=1024, hidden_size=512, intermediate_size=ffn, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=kv_heads))


def _opt():
    model = OPTForCausalLM(OPTConfig(vocab_size=1024, hidden_size=512, num_hidden_layers=3, ffn_dim=1024, num_attention_heads=8, max_position_embeddings=256))
    with torch.no_grad():
        for name, p in model.named_parameters():
            if name.endswith("bias"):
                p.normal_(0.0, 0.05)
            if "layer_norm.weight" in name:
                p.add_(0.1 * torch.randn_like(p))
    return model


FAMILIES = {
    "llama": _llama, "llama_grouped": lambda: _llama(2), "llama_ragged": lambda: _llama(4, 344),  # 344: no multiple of the groups of 16 gate and up rows
    "opt": _opt, "falcon": lambda: FalconForCausalLM(FalconConfig(vocab_size=1024, hidden_size=512, n_layer=3, n_head=8, n_head_kv=2)),
}


def _pair(family):
    torch.manual_seed(0)
    model = FAMILIES[family]()
    served = copy.deepcopy(model).to(device="cuda", dtype=torch.bfloat16).eval()
    oracle = model.float().eval()
    oracle.load_state_dict({k: v.float().cpu() for k, v in served.state_dict().items()})
    return oracle, served


def _off(got, want):
    got, want = got.float().cpu(), want.float().cpu()
    return ((got - want).norm() / want.norm()).item()


@pytest.mark.parametrize("family", FAMILIES)
def test_prefill_and_decode_follow_the_model(family):
    from tensor_parallel_b200.ops import native

    oracle, served = _pair(family)
    wrapped = tp.tensor_parallel(served, ["cuda:0"])
    ids = torch.randint(0, 1024, (3, 70), generator=torch.Generator().manual_seed(1))
    logits = wrapped.prefill(ids, max_new_tokens=16, quantize="int8")
    engine = wrapped._engine
    assert engine.quantize == "int8"
    with torch.no_grad():
        want = oracle(input_ids=ids, use_cache=True)
    assert _off(logits, want.logits[:, -1]) < CLOSE
    nxt, past = want.logits[:, -1].argmax(-1), want.past_key_values
    for _ in range(4):  # the first call captures the graph, later calls replay it
        engine.ids[:3].copy_(nxt)
        engine.decode_step(3)
        with torch.no_grad():
            out = oracle(input_ids=nxt[:, None], past_key_values=past, use_cache=True)
        past = out.past_key_values
        assert _off(engine.logits_local[:3], out.logits[:, -1]) < CLOSE
        nxt = out.logits[:, -1].argmax(-1)
    torch.cuda.synchronize()
    native.device_state(torch.device("cuda", 0)).check_status()
    assert engine.graph is not None and engine.kernels_per_step <= 9 * 3 + 5


def test_few_and_many_tokens_agree():
    """A prompt as a whole and token by token: the same 8-bit rows and sums whatever kernel the number of tokens chooses; what differs is the order of the
    attention's sums and a rounding to bf16 here and there, which an 8-bit step (0.8 %) passes on at worst."""
    _, served = _pair("llama")
    engine = DecoderEngine(served, max_batch=2, max_seq=128, quantize="int8")
    ids = torch.randint(0, 1024, (2, 90), generator=torch.Generator().manual_seed(2)).cuda()
    whole = engine.prefill(ids)
    engine.prefill(ids[:, :60])
    for t in range(60, 90):
        engine.ids[:2].copy_(ids[:, t])
        engine.decode_step(2)
    assert _off(engine.logits_local[:2], whole) < CLOSE / 2
    assert int(engine.pos[0]) == 90


def test_the_engine_changes_its_form_when_asked_and_generates():
    oracle, served = _pair("llama")
    wrapped = tp.tensor_parallel(served, ["cuda:0"])
    ids = torch.randint(0, 1024, (2, 33), generator=torch.Generator().manual_seed(3))
    plain = wrapped.generate(ids, max_new_tokens=5)
    first = wrapped._engine
    assert first.quantize is None
    out = wrapped.generate(ids, max_new_tokens=5, quantize="int8")
    second = wrapped._engine
    assert second is not first and second.quantize == "int8" and out.shape == plain.shape and torch.equal(out[:, :33].cpu(), ids)
    assert torch.equal(wrapped.generate(ids, max_new_tokens=5), out) and wrapped._engine is second  # (stays what it is)
    assert torch.equal(wrapped.generate(ids, max_new_tokens=5, quantize="bf16"), plain) and wrapped._engine.quantize is None
    with pytest.raises(ValueError):
        wrapped.serving_engine(quantize="int4")
    with pytest.raises(ValueError):
        wrapped.generate(ids, max_new_tokens=2, quantize="int8", do_sample=True)


def test_weights_are_released():
    _, served = _pair("llama")
    wrapped = tp.tensor_parallel(served, ["cuda:0"])
    ids = torch.randint(0, 1024, (2, 40), generator=torch.Generator().manual_seed(4))
    logits = wrapped.prefill(ids, max_new_tokens=8, quantize="int8").clone()
    freed = wrapped.release_training_weights()
    layer = wrapped.module_shards[0].model.layers[0]
    assert layer.self_attn.o_proj.weight.numel() == 0 and layer.mlp.down_proj.weight.numel() == 0  # (the engine has all projections in 8 bits)
    assert freed > 0 and torch.equal(wrapped.prefill(ids, max_new_tokens=8), logits)
    with pytest.raises(RuntimeError, match="released"):
        wrapped.serving_engine(quantize="bf16")


class _Ranks:
    """Stands in for the communication of two ranks that hold the same partial sums: a sum is twice one's own."""

    world, rank, mc_base = 2, 0, 0

    def __init__(self, device):
        self.device, self._call = device, 0
        self.status = torch.zeros(4, dtype=torch.int32, device=device)

    def staging_view(self, which, shape, dtype):
        return torch.empty(shape, dtype=dtype, device=self.device)

    def all_reduce(self, t):
        return t * 2

    def all_gather(self, t):
        return torch.stack([t, t])

    def check_status(self):
        pass


@pytest.mark.parametrize("family", ["llama", "opt", "falcon"])
def test_the_ranks_sum_is_added_by_the_next_norm(family):
    """Two ranks with half of every row-parallel weight each add up to the whole model (halves are exact, in 8 bits too); their biases count twice, as shards that
    carry half of them do."""
    _, served = _pair(family)
    whole = DecoderEngine(served, max_batch=2, max_seq=96, quantize="int8", use_graph=False)
    halved = copy.deepcopy(served)
    with torch.no_grad():
        for name, p in halved.named_parameters():
            if any(part in name for part in ("o_proj", "down_proj", "out_proj", "fc2", "attention.dense", "dense_4h_to_h")):
                p.mul_(0.5)
    ids = torch.randint(0, 1024, (2, 50), generator=torch.Generator().manual_seed(5)).cuda()
    from tensor_parallel_b200 import engine_spec

    spec = engine_spec.describe(halved, 96)
    spec.head_split = "vocab"
    split = DecoderEngine(halved, _Ranks(torch.device("cuda", 0)), max_batch=2, max_seq=96, quantize="int8", use_graph=False, spec=spec)
    want, got = whole.prefill(ids), split.prefill(ids)
    assert _off(got[:, :1024], want) < CLOSE / 2  # (the sum is rounded to bf16 once more than in one GEMM)
    for e in (whole, split):
        e.ids[:2].copy_(ids[:, -1])
        e.decode_step(2)
    assert _off(split.logits_local[:2], whole.logits_local[:2]) < CLOSE / 2
