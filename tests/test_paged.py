"""Paged cache, attention over it and adjusted logits on the CPU: the definitions against 64 bits, what is refused, and a run of them together."""
import math

import pytest
import torch

from paged_cases import BF16, attention64, batch, check_append, check_logits, numbers, within
from tensor_parallel_b200.ops import functional as OF


def cache_of(b):
    return OF.PagedCache(b["keys"], b["values"], b["table"])


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("window", [None, 1, 5, 40])
@pytest.mark.parametrize("new,past,heads,kv_heads,dim,page", [([1], [0], 2, 2, 8, 4), ([1, 3, 0, 7], [5, 0, 9, 30], 6, 2, 16, 4), ([33, 2], [0, 63], 5, 1, 24, 16),
                                                              ([0, 0], [3, 0], 2, 1, 8, 3)])
def test_attention_of_ragged_batches(new, past, heads, kv_heads, dim, page, window, dtype):
    b = batch(new, past, heads, kv_heads, dim, page, dtype, front=2, rest=3)
    out = OF.paged_attention(b["q"], cache_of(b), b["starts"], b["past"], window=window)
    want, tol = attention64(b, window=window)
    within(out, want, tol + 2.0 ** -20 * want.abs().max() * (dtype == torch.float32))
    assert out.dtype == dtype and not out[:2].any() and not out[2 + sum(new):].any()
    kept = torch.full_like(b["q"], 3.0)
    assert OF.paged_attention(b["q"], cache_of(b), b["starts"], b["past"], window=window, most_new=max(new), out=kept) is kept
    assert torch.equal(kept[2:2 + sum(new)], out[2:2 + sum(new)]) and (kept[:2] == 3).all() and (kept[2 + sum(new):] == 3).all()


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("turn", [None, (8, False, 1.0), (8, True, 1.0), (4, False, 1.25), (6, True, 0.5), (2, False, 1.0)])
def test_append_with_norms_and_rotation(turn, norms, dtype):
    b = batch([1, 3, 0, 9], [5, 0, 2, 100003], 6, 2, 8, 4, dtype, front=1, rest=2, only_new=True)
    gen = torch.Generator().manual_seed(5)
    rotary = None if turn is None else OF.Rotary(OF.rotary(turn[0], 1000.0).frequencies, turn[1], turn[2])
    q_norm, k_norm = (1 + numbers(gen, 8, dtype=dtype, scale=0.2) if norms else None for _ in range(2))
    before = b["keys"].clone(), b["values"].clone()
    q = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=rotary, q_norm=q_norm, k_norm=k_norm)
    if rotary is None and not norms:
        assert q is b["q"]
        q = torch.cat((q[:1] * 0, q[1:-2], q[-2:] * 0))
    check_append(b, q, before, rotary, q_norm, k_norm)


def test_append_into_out_and_without_queries():
    b = batch([2, 1], [3, 0], 4, 2, 8, 4, rest=2)
    turn = OF.rotary(8)
    want = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=turn)
    q = b["q"].clone()
    assert OF.paged_append(cache_of(b), q, b["k"], b["v"], b["starts"], b["past"], rotary=turn, out=q) is q
    assert torch.equal(q[:3], want[:3]) and torch.equal(q[3:], b["q"][3:]) and not want[3:].any()
    assert OF.paged_append(cache_of(b), None, b["k"], b["v"], b["starts"], b["past"], rotary=turn) is None


def test_frequencies():
    plain = OF.rotary(64, 10000.0)
    want = 10000.0 ** (-torch.arange(0, 64, 2).double() / 64)
    torch.testing.assert_close(plain.frequencies.double(), want, rtol=2.0 ** -23, atol=0)
    assert plain.factor == 1.0 and not plain.interleaved and OF.rotary(64, interleaved=True).interleaved
    torch.testing.assert_close(OF.rotary(64, scaling={"type": "linear", "factor": 4.0}).frequencies.double(), want / 4, rtol=2.0 ** -23, atol=0)
    three = OF.rotary(64, scaling={"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}).frequencies.double()
    length = 2 * math.pi / want
    assert torch.allclose(three[length < 8192 / 4], want[length < 8192 / 4], rtol=1e-6) and torch.allclose(three[length > 8192], want[length > 8192] / 8, rtol=1e-6)
    between = (length > 8192 / 4) & (length < 8192)
    smooth = (8192 / length - 1) / 3
    assert between.any() and torch.allclose(three[between], ((1 - smooth) * want / 8 + smooth * want)[between], rtol=1e-6)
    yarn = OF.rotary(64, scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})
    assert yarn.factor == pytest.approx(0.1 * math.log(4) + 1)
    ratio = yarn.frequencies.double() / want
    assert ratio[0] == pytest.approx(1, rel=1e-6) and ratio[-1] == pytest.approx(0.25, rel=1e-6) and (ratio.diff() <= 1e-6).all()
    for bad in ({"type": "dynamic", "factor": 2.0},):
        with pytest.raises(ValueError, match="dynamic"):
            OF.rotary(64, scaling=bad)
    for dim in (0, 7, -2):
        with pytest.raises(ValueError):
            OF.rotary(dim)


def test_a_run_of_steps_is_dense_attention_over_everything():
    """Prompts in chunks, then token by token, in one ragged batch: what dense attention over each whole sequence gives."""
    torch.manual_seed(3)
    heads, kv_heads, dim, page = 4, 2, 16, 4
    plan = [[5, 0, 9], [3, 7, 1], [1, 1, 1], [1, 1, 1], [0, 1, 4]]
    lengths = [sum(c) for c in zip(*plan)]
    whole = [tuple(torch.randn(n, h, dim) for h in (heads, kv_heads, kv_heads)) for n in lengths]
    pages = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(pages)).int()
    table = torch.full((3, max(pages)), -1, dtype=torch.int32)
    for s, at in enumerate((0, pages[0], pages[0] + pages[1])):
        table[s, :pages[s]] = order[at:at + pages[s]]
    cache = OF.PagedCache(torch.full((sum(pages), kv_heads, page, dim), math.nan), torch.full((sum(pages), kv_heads, page, dim), math.nan), table)
    past, got, turn = [0, 0, 0], [[], [], []], OF.rotary(dim)
    for new in plan:
        starts = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
        q, k, v = (torch.cat([whole[s][i][past[s]:past[s] + new[s]] for s in range(3)]) for i in range(3))
        lens = torch.tensor(past, dtype=torch.int32)
        q = OF.paged_append(cache, q, k, v, starts, lens, rotary=turn)
        out = OF.paged_attention(q, cache, starts, lens)
        for s in range(3):
            got[s].append(out[starts[s]:starts[s + 1]])
        past = [p + n for p, n in zip(past, new)]
    for s, (q, k, v) in enumerate(whole):
        at = torch.arange(lengths[s])[None]
        q, k = OF.apply_rope_ref(q[None], at, 10000.0), OF.apply_rope_ref(k[None], at, 10000.0)
        torch.testing.assert_close(torch.cat(got[s]), OF.attention_ref(q, k, v[None], True)[0], rtol=1e-5, atol=1e-5)


def test_refused_caches():
    b = batch([2, 1], [3, 0], 4, 2, 8, 4)
    cache = cache_of(b)
    args = (b["starts"], b["past"])
    for what, broken in dict(table=cache._replace(table=b["table"].long()), types=cache._replace(values=b["values"].float()), shapes=cache._replace(values=b["values"][1:]),
                             rows=cache._replace(table=b["table"][:1]), dims=cache._replace(keys=b["keys"][0], values=b["values"][0])).items():
        with pytest.raises(ValueError):
            OF.paged_attention(b["q"], broken, *args)
        with pytest.raises(ValueError):
            OF.paged_append(broken, b["q"], b["k"], b["v"], *args)
    for starts, past in ((b["starts"].long(), b["past"]), (b["starts"], b["past"].long()), (b["starts"][:2], b["past"]), (b["starts"][None], b["past"])):
        with pytest.raises(ValueError):
            OF.paged_attention(b["q"], cache, starts, past)
    with pytest.raises(ValueError, match="no place"):
        OF.paged_attention(b["q"], OF.PagedCache(b["keys"][:0], b["values"][:0], b["table"]), *args)
    with pytest.raises(ValueError, match="query heads"):
        OF.paged_attention(b["q"][:, :3], cache, *args)
    for bad in (dict(window=0), dict(window=-3), dict(most_new=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(out=b["q"].float()), dict(out=b["q"][:2]),
                dict(out=b["q"][:1].expand(3, 4, 8))):
        with pytest.raises(ValueError):
            OF.paged_attention(b["q"], cache, *args, **bad)
    for bad in (dict(q_norm=torch.ones(8)), dict(k_norm=torch.ones(4, dtype=BF16)), dict(rotary=OF.Rotary(torch.ones(5))), dict(rotary=OF.Rotary(torch.ones(2, dtype=torch.float64))),
                dict(rotary=OF.Rotary(torch.ones(0))), dict(out=b["q"].float())):
        with pytest.raises(ValueError):
            OF.paged_append(cache, b["q"], b["k"], b["v"], *args, **bad)
    for q, k, v in ((b["q"][:2], b["k"], b["v"]), (b["q"], b["k"][:, :1], b["v"]), (b["q"], b["k"], b["v"].float()), (b["q"][..., :4], b["k"], b["v"])):
        with pytest.raises(ValueError):
            OF.paged_append(cache, q, k, v, *args)
    with pytest.raises(ValueError, match="queries"):
        OF.paged_append(cache, None, b["k"], b["v"], *args, out=b["q"])
    q = b["q"].float().requires_grad_()
    full = OF.PagedCache(b["keys"].float(), b["values"].float(), b["table"])
    with pytest.raises(RuntimeError, match="gradient"):
        OF.paged_attention(q, full, *args)
    with torch.no_grad():
        OF.paged_attention(q, full, *args)
    with pytest.raises(RuntimeError, match="traced"):
        torch.func.vmap(lambda t: OF.paged_attention(t, full, *args))(q.detach()[None])


def test_lengths_that_do_not_fit():
    b = batch([2, 1], [3, 0], 4, 2, 8, 4)
    cache = cache_of(b)

    def both(starts, past, cache=cache):
        starts, past = (torch.tensor(t, dtype=torch.int32) for t in (starts, past))
        with pytest.raises(ValueError):
            OF.paged_attention(b["q"], cache, starts, past)
        before = cache.keys.clone()
        with pytest.raises(ValueError):
            OF.paged_append(cache, b["q"], b["k"], b["v"], starts, past)
        assert torch.equal(cache.keys.view(torch.int16), before.view(torch.int16))

    both([0, 2, 4], [3, 0])   # more rows than there are
    both([0, 2, 1], [3, 0])   # back again
    both([-1, 2, 3], [3, 0])
    both([0, 2, 3], [-1, 0])
    both([0, 2, 3], [7, 0])   # beyond the table
    for entry in (-1, 99):
        table = b["table"].clone()
        table[0, 1] = entry
        both([0, 2, 3], [3, 0], cache._replace(table=table))
    with pytest.raises(ValueError, match="most_new"):
        OF.paged_attention(b["q"], cache, b["starts"], b["past"], most_new=1)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rows,vocab,width", [(1, 1, 1), (3, 50, 20), (2, 33, 0), (4, 64, 7), (2, 127, 300)])
def test_adjusted_logits(rows, vocab, width, dtype):
    gen = torch.Generator().manual_seed(rows * vocab)
    logits = numbers(gen, rows, vocab, dtype=dtype, scale=4.0)
    tokens = torch.randint(-2, vocab + 2, (rows, width), generator=gen)
    lengths, prompts = (torch.randint(0, width + 1, (rows,), generator=gen, dtype=torch.int32) for _ in range(2))
    r, f, p = (torch.rand(rows, generator=gen) + low for low in (0.6, 0.0, -0.5))
    bias = numbers(gen, rows, vocab, dtype=torch.float32)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=gen).int()
    for args in ((logits, tokens, lengths, prompts, r, f, p, bias, allowed), (logits, tokens, None, None, 1.3, 0.2, 0.4), (logits, tokens, lengths, None, None, f, None),
                 (logits, None, None, None, None, None, None, bias[0].to(BF16), allowed[0]), (logits, tokens, None, prompts, 0.5), (logits,)):
        check_logits(OF.adjust_logits(*args), args)


def test_adjusted_logits_that_are_not_finite():
    inf, nan = math.inf, math.nan
    logits = torch.tensor([[inf, -inf, nan, 1.0, torch.finfo(torch.float32).min, 0.0]])
    tokens = torch.tensor([[0, 1, 2, 4, 5]])
    out = OF.adjust_logits(logits, tokens, repetition=2.0, presence=1.0)
    assert out[0, 0] == inf and out[0, 1] == -inf and out[0, 2].isnan() and out[0, 3] == 1 and out[0, 4] == -inf and out[0, 5] == -1
    out = OF.adjust_logits(logits, allowed=torch.zeros(1, 1, dtype=torch.int32))
    assert (out == -inf).all()  # (a grammar that allows nothing)


def test_refused_logits():
    x, t = torch.zeros(2, 40), torch.zeros(2, 3, dtype=torch.int64)
    one = torch.ones(2, dtype=torch.int32)
    for args in ((x[0],), (x.long(),), (x, t.int()), (x, t[:1]), (x, t, one.long()), (x, t, one[:1]), (x, t, None, one.long()), (x, t, None, None, 0.0), (x, t, None, None, -1.0),
                 (x, t, None, None, torch.ones(2).double()), (x, t, None, None, torch.ones(3)), (x, None, one), (x, None, None, None, 1.5), (x, None, None, None, None, None, 1.0)):
        with pytest.raises(ValueError):
            OF.adjust_logits(*args)
    for bad in (dict(bias=torch.zeros(39)), dict(bias=torch.zeros(40).half()), dict(bias=torch.zeros(1, 40)), dict(allowed=torch.zeros(1, dtype=torch.int32)), dict(allowed=torch.zeros(2, 2))):
        with pytest.raises(ValueError):
            OF.adjust_logits(x, **bad)
    with pytest.raises(RuntimeError, match="gradient"):
        OF.adjust_logits(x.clone().requires_grad_())


# -- in generate ---------------------------------------------------------------------------------


def _tiny():
    from tensor_parallel_b200.models.llama import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    return LlamaForCausalLM(LlamaConfig(vocab_size=50, hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2)).eval()


def test_generate_adjusts_its_logits():
    model, prompt = _tiny(), torch.tensor([[3, 7, 9], [11, 3, 3]])
    plain, scores = model.generate(prompt, max_new_tokens=6, output_scores=True)
    same = model.generate(prompt, max_new_tokens=6, repetition_penalty=1.0, frequency_penalty=0.0, logit_bias=torch.zeros(50))
    assert torch.equal(plain, same)
    # a large presence penalty: no token of the answer comes twice; one of the prompt may
    once = model.generate(prompt, max_new_tokens=12, presence_penalty=1e4)
    assert all(len(set(row[3:].tolist())) == 12 for row in once)
    # the repetition penalty is for the prompt too
    with torch.no_grad():
        first = model(input_ids=prompt)["logits"][:, -1].float()
    want = OF.adjust_logits(first, prompt, None, None, 1.9).argmax(-1)
    assert torch.equal(model.generate(prompt, max_new_tokens=1, repetition_penalty=1.9)[:, -1], want)
    # a bias that decides, and bits that leave one token each
    bias = torch.zeros(2, 50)
    bias[0, 17] = bias[1, 23] = 1e4
    assert model.generate(prompt, max_new_tokens=3, logit_bias=bias)[:, 3:].tolist() == [[17] * 3, [23] * 3]
    steps = iter([5, 40, 33])

    def grammar(ids):
        bits = torch.zeros(2, dtype=torch.int64)
        t = next(steps)
        bits[t // 32] = 1 << (t % 32)
        return torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).int()

    assert model.generate(prompt, max_new_tokens=3, allowed_tokens=grammar)[:, 3:].tolist() == [[5, 40, 33]] * 2
    sampled = model.generate(prompt, max_new_tokens=4, do_sample=True, allowed_tokens=torch.tensor([1 << 4, 1 << 1], dtype=torch.int32), generator=torch.Generator().manual_seed(0))
    assert set(sampled[:, 3:].flatten().tolist()) <= {4, 33}
    with pytest.raises(ValueError, match="beam"):
        model.generate(prompt, max_new_tokens=2, num_beams=2, presence_penalty=1.0)


def test_generate_of_a_wrapped_model_adjusts_too():
    import tensor_parallel_b200 as tp

    model, prompt = _tiny(), torch.tensor([[3, 7, 9]])
    want = model.generate(prompt, max_new_tokens=5, presence_penalty=3.0, repetition_penalty=1.3)
    wrapped = tp.tensor_parallel(model, ["cpu", "cpu"])
    assert torch.equal(wrapped.generate(prompt, max_new_tokens=5, presence_penalty=3.0, repetition_penalty=1.3), want)


def test_under_a_compiler():
    b = batch([2, 1], [3, 0], 4, 2, 8, 4)
    turn = OF.rotary(8)

    def step(q, k, v):
        q = OF.paged_append(cache_of(b), q * 1.0, k, v, b["starts"], b["past"], rotary=turn)
        return OF.paged_attention(q, cache_of(b), b["starts"], b["past"]) + 1.0

    want = step(b["q"], b["k"], b["v"])
    assert torch.equal(torch.compile(step, backend="eager")(b["q"], b["k"], b["v"]), want)
    x, t = torch.randn(2, 40), torch.randint(0, 40, (2, 6))
    adjust = torch.compile(lambda x: OF.adjust_logits(x, t, presence=0.5), backend="eager", fullgraph=True)
    assert torch.equal(adjust(x), OF.adjust_logits(x, t, presence=0.5))
