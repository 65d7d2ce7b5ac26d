"""Ragged serving operators on the CPU: scaled frequencies pair by pair, what the C entries refuse, prompts of other types."""
import math

import pytest
import torch

from tensor_parallel_b200.ops import functional as OF


def yarn64(dim, theta, d):
    """Frequencies and factor by the published formulas, one pair at a time."""
    original, by = d["original_max_position_embeddings"], d["factor"]
    ends = [dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (d.get("beta_fast") or 32, d.get("beta_slow") or 1)]
    if d.get("truncate", True):
        ends = [math.floor(ends[0]), math.ceil(ends[1])]
    low, high = max(ends[0], 0), min(ends[1], dim - 1)
    frequencies = []
    for i in range(dim // 2):
        f = theta ** (-2 * i / dim)
        slow = min(max((i - low) / (high - low), 0.0), 1.0)
        frequencies.append((1 - slow) * f + slow * f / by)
    if d.get("attention_factor") is not None:
        factor = d["attention_factor"]
    elif d.get("mscale") and d.get("mscale_all_dim"):
        factor = (0.1 * d["mscale"] * math.log(by) + 1) / (0.1 * d["mscale_all_dim"] * math.log(by) + 1) if by > 1 else 1.0
    else:
        factor = 0.1 * math.log(by) + 1 if by > 1 else 1.0
    return torch.tensor(frequencies, dtype=torch.float64), factor


@pytest.mark.parametrize("dim,theta,more", [
    (64, 10000.0, dict(factor=4.0)), (128, 1000000.0, dict(factor=4.0, beta_fast=24, beta_slow=2)), (64, 150000.0, dict(factor=32.0, truncate=False)),
    (64, 150000.0, dict(factor=32.0, truncate=True, beta_fast=None, beta_slow=None)), (64, 10000.0, dict(factor=40.0, mscale=1.0, mscale_all_dim=1.0)),
    (64, 10000.0, dict(factor=40.0, mscale=0.707, mscale_all_dim=1.0)), (64, 10000.0, dict(factor=40.0, mscale=0.707)), (64, 10000.0, dict(factor=40.0, mscale_all_dim=0.707)),
    (64, 10000.0, dict(factor=40.0, mscale=0.0, mscale_all_dim=0.0)), (64, 10000.0, dict(factor=1.0, mscale=0.5, mscale_all_dim=1.0)), (32, 10000.0, dict(factor=8.0, attention_factor=1.5)),
    (32, 10000.0, dict(factor=8.0, attention_factor=0.0, mscale=1.0, mscale_all_dim=0.5)), (32, 10000.0, dict(factor=8.0, attention_factor=None))])
@pytest.mark.parametrize("original", [4096, 32768])
def test_yarn_pair_by_pair(dim, theta, more, original):
    d = dict(rope_type="yarn", original_max_position_embeddings=original, **more)
    want, factor = yarn64(dim, theta, d)
    got = OF.rotary(dim, theta, scaling=d)
    # a rounding to fp32, and some in 64 bits
    assert ((got.frequencies.double() - want).abs() <= 2.0 ** -24 * 1.01 * want).all()
    assert got.factor == pytest.approx(factor, rel=1e-14) and isinstance(got.factor, float)
    assert torch.equal(OF.rotary(dim, theta, scaling=dict(d, rope_theta=theta, partial_rotary_factor=0.5, finetuned=True)).frequencies, got.frequencies)


def test_scaling_that_is_not_known_is_refused_by_name():
    yarn = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)
    for scaling, name in ((dict(yarn, short_factor=[1.0]), "short_factor"), (dict(rope_type="default", mrope_section=[16, 24, 24]), "mrope_section"),
                          (dict(type="linear", factor=2.0, mscale=1.0), "mscale"), (dict(yarn, rope_theta=500000.0), "rope_theta"), (dict(rope_type="longrope", factor=4.0), "longrope")):
        with pytest.raises(ValueError, match=name):
            OF.rotary(64, scaling=scaling)
    plain = OF.rotary(64)
    for scaling in (None, {}, dict(rope_type="default"), dict(rope_type="default", rope_theta=10000.0), dict(rope_type="default", rope_theta=None)):
        assert torch.equal(OF.rotary(64, scaling=scaling).frequencies, plain.frequencies)


def _adjust(x, out, tokens=None):
    """The C entry's answer for ``x`` and ``out``, ``[rows, vocab]`` views (on a GPU where there is one: nothing here is launched with addresses that it cannot reach)."""
    from tensor_parallel_b200.ops import native

    status = torch.zeros(4, dtype=torch.int32, device=x.device)
    a = native.AdjustLogits(logits=x.data_ptr(), out=out.data_ptr(), status=status.data_ptr(), logits_ld=x.stride(0), out_ld=out.stride(0), rows=x.shape[0], vocab=x.shape[1],
                            dtype=int(x.dtype == torch.float32), repetition_all=1.0)
    if tokens is not None:
        a.tokens, a.tokens_ld, a.width = tokens.data_ptr(), tokens.stride(0), tokens.shape[1]
    return native.LIB.tpb_adjust_logits(a, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_results_over_the_logits_are_refused_in_c(dtype):
    device = "cuda" if torch.cuda.is_available() else "cpu"
    room, tokens = torch.zeros(12, 128, dtype=dtype, device=device), torch.zeros(4, 3, dtype=torch.int64, device=device)
    x = room[:4, :64]
    err_arg = 1
    assert _adjust(x, x, tokens) == err_arg                       # in place, and tokens to come back to
    assert _adjust(x[:1], x[:1], tokens) == err_arg
    for history in (None, tokens):
        assert _adjust(x, room[1:5, :64], history) == err_arg     # a row further down
        assert _adjust(x, room[:4, 8:72], history) == err_arg     # a few columns on
        assert _adjust(x, room[:4, 72:].as_strided((4, 64), (128, 1), 72), history) == err_arg  # beyond the gap
        assert _adjust(x, room.as_strided((4, 64), (64, 1)), history) == err_arg                # another pitch
        assert _adjust(x[:1], room[:1, 63:127], history) == err_arg


def test_which_strides_the_append_kernel_takes():
    """Up to 64 GB between heads of the cache and 4 GB between rows, any number between pages; what is further apart goes by its steps."""
    from tensor_parallel_b200.ops import native

    def held(shape, strides):
        return torch.empty_strided(shape, strides, dtype=torch.bfloat16, device="meta")

    limit = native.APPEND_HEAD_STRIDE
    rows, table = held((3, 2, 64), (128, 64, 1)), torch.zeros(1, 2, dtype=torch.int32)
    near = held((2, 2, 16, 64), (2 * limit, limit - 8, 64, 1))
    assert native.paged_append_supported((near, near, table), rows, rows, rows, None)
    far = held((2, 2, 16, 64), (1024, limit, 64, 1))
    assert not native.paged_append_supported((far, near, table), rows, rows, rows, None)
    assert not native.paged_append_supported((near, far, table), rows, rows, rows, None)
    wide = held((3, 2, 64), (native.APPEND_ROW_STRIDE, 64, 1))
    rows_apart = held((3, 2, 64), (native.APPEND_ROW_STRIDE - 8, 64, 1))
    assert native.paged_append_supported((near, near, table), rows_apart, rows_apart, rows_apart, rows_apart)
    for args in ((wide, rows, rows, None), (rows, wide, rows, None), (rows, rows, wide, None), (rows, rows, rows, wide)):
        assert not native.paged_append_supported((near, near, table), *args)


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_generate_with_penalties_takes_prompts_of_either_type(kind):
    from tensor_parallel_b200.models.llama import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    model = LlamaForCausalLM(LlamaConfig(vocab_size=50, hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2)).eval()
    prompt = torch.tensor([[3, 7, 9], [11, 3, 3]])
    want = model.generate(prompt, max_new_tokens=5, repetition_penalty=1.4, presence_penalty=0.5)
    assert torch.equal(model.generate(prompt.to(kind), max_new_tokens=5, repetition_penalty=1.4, presence_penalty=0.5).long(), want)
    assert model.generate(prompt.to(kind), max_new_tokens=5, repetition_penalty=1.4).dtype == model.generate(prompt.to(kind), max_new_tokens=5).dtype


def test_the_workspace_is_within_its_documented_bound():
    from tensor_parallel_b200.ops import native

    bound = int(OF.paged_attention.__doc__.split("a workspace of up to ")[1].split(" MB")[0]) * 10 ** 6
    most = 0
    for dim in (64, 128):
        for group in (1, 2, 3, 4, 7, 8, 15, 16, 17, 31, 32, 33, 64, 65, 71, 128):
            for kv_heads in (1, 8, 64):
                for n, tokens, most_new in ((1, 1, 1), (1, 100000, 100000), (7, 64, 64), (256, 256, 1), (4096, 4096, 4096), (3, 300, 5), (50, 60, 16)):
                    for width in (1, 2, 1000, 100000):
                        most = max(most, native.LIB.tpb_paged_attention_workspace(n, tokens, width, 16, most_new, kv_heads, group, dim))
    assert 0.9 * bound < most <= bound, most
