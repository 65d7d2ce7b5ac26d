"""Paged attention, append and adjusted logits where their kernels change form: rows that are not finite, pages that are not there, strides beyond 32 bits, sizes behind
which a launch is made another way."""
import math

import pytest
import torch

from paged_cases import BF16, attention64, batch, numbers, turned64, within
from tensor_parallel_b200.ops import functional as OF

pytestmark = pytest.mark.gpu


def native():
    from tensor_parallel_b200.ops import native

    return native


def status_of(device="cuda"):
    word = native().device_state(torch.device(device)).status
    code = int(word[0])
    word.zero_()
    return code


def cache_of(b):
    return OF.PagedCache(b["keys"], b["values"], b["table"])


def attend(b, **kw):
    before = native().launch_count
    out = OF.paged_attention(b["q"], cache_of(b), b["starts"], b["past"], **kw)
    assert native().launch_count > before
    return out


@pytest.mark.parametrize("number", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (8, 2, 128), (12, 4, 64)])
@pytest.mark.parametrize("new,past,rows", [([1], [9999], [0]), ([1, 1, 1], [50, 4000, 9], [0, 1, 2]), ([3], [12000], [1]), ([600], [8000], [0, 333, 599]), ([300, 1], [0, 70], [0, 1, 2, 3, 130, 300]),
                                           ([1, 200, 1], [900, 3000, 40], [0, 1, 70, 201])])
def test_query_rows_that_are_not_finite(new, past, rows, heads, kv_heads, dim, number):
    """A row of queries that is NaN, or infinite in an element, gives NaN wherever its keys are cut, and its neighbours what they give without it."""
    b = batch(new, past, heads, kv_heads, dim, 16, device="cuda", seed=len(new) + past[0])
    want, tol = attention64(b)
    q = b["q"].clone()
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for i, r in enumerate(rows):
        q[r, (3 * i + 1) % heads, 5 if math.isinf(number) else slice(None)] = number
        bad[r, (3 * i + 1) % heads] = True
    for most_new in (None, max(new)):
        out = attend(dict(b, q=q), most_new=most_new)
        assert out[bad].isnan().all()
        within(out[~bad], want[~bad], tol[~bad])
    assert status_of() == 0


@pytest.mark.parametrize("dim", [64, 128])
def test_values_that_a_row_does_not_see_yet(dim):
    """The largest numbers of the type in the values of later tokens of the same sequence."""
    b = batch([200], [40], 4, 2, dim, 16, device="cuda")
    want, tol = attention64(b)
    low = torch.finfo(BF16).min
    for at in range(100, 240):  # (tokens 60 and up see them)
        b["values"][b["table"][0, at // 16].long(), :, at % 16] = low
    within(attend(b)[:60], want[:60], tol[:60])
    want, tol = attention64(b, window=30)
    within(attend(b, window=30)[:60], want[:60], tol[:60])


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 128), (2, 2, 64), (4, 1, 128), (7, 1, 64)])
def test_a_page_that_only_later_rows_reach(heads, kv_heads, dim):
    """The first half of a row tile of 256 ends in front of the tile of keys with a page that is not there: its rows are right, call after call; those that reach the page are NaN."""
    group = heads // kv_heads
    tokens, half = 256 // group, -(-128 // group)
    b = batch([tokens], [256 - half], heads, kv_heads, dim, 16, device="cuda")  # (the half's last key is the last of a tile)
    want, tol = attention64(b)
    bad = dict(b, table=b["table"].clone())
    page = (256 - half + tokens - 1) // 16
    bad["table"][0, page] = -1
    outs = [attend(bad) for _ in range(20)]
    assert status_of() == 3
    within(outs[0][:128 // group], want[:128 // group], tol[:128 // group])
    assert outs[0][page * 16 - (256 - half):].isnan().all()
    for out in outs:
        assert torch.equal(out.view(torch.int16), outs[0].view(torch.int16))


# -- logits ----------------------------------------------------------------------------------------


def logits64(x, tokens, lengths, prompts, repetition, frequency, presence, bias, allowed):
    """``(want, tolerance)`` of long histories: a rounding to the type, and four in 32 bits of what goes into a result (logit, penalties, bias)."""
    want, half = x.double().clone(), 2.0 ** -8 if x.dtype == BF16 else 2.0 ** -24
    rows, vocab = x.shape
    size = want.abs()
    for r in range(rows):
        history = tokens[r, :int(lengths[r])]
        there = (history >= 0) & (history < vocab)
        seen = torch.bincount(history[there], minlength=vocab) > 0
        there[:int(prompts[r])] = False
        count = torch.bincount(history[there], minlength=vocab)
        rep, f, p = (float(t[r]) for t in (repetition, frequency, presence))
        want[r] = torch.where(seen, torch.where(want[r] > 0, want[r] / rep, want[r] * rep), want[r])
        size[r] = size[r] * max(rep, 1 / rep) + (f * count + p * (count > 0)).abs()
        want[r] -= f * count + p * (count > 0)
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    if allowed is not None:
        at = torch.arange(vocab, device=x.device)
        want[(allowed.long()[:, at // 32] >> (at % 32)) % 2 == 0] = -math.inf
    return want, half * 1.01 * want.abs().nan_to_num(posinf=0.0) + 4 * 2.0 ** -24 * size


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rows,vocab,width", [(3, 1000, 2048), (3, 1000, 2049), (2, 5003, 4097), (5, 300, 9000), (40, 65027, 9000), (128, 19000, 4096), (128, 19001, 4097), (1, 3000001, 5000),
                                              (300, 8200, 300), (2, 1300000, 1)])
@pytest.mark.parametrize("form", ["whole rows", "odd rows", "shared"])
def test_adjusted_logits_of_long_histories(rows, vocab, width, dtype, form):
    """Histories of several rounds of a block (2048 tokens, behind a stream 4096), and rows and vocabularies that go by two kernels."""
    gen = torch.Generator(device="cuda").manual_seed(rows + vocab + width)
    room = 4 * torch.randn(rows, vocab + 3, device="cuda", generator=gen)
    x = room.to(dtype)[:, 3:] if form == "odd rows" else room[:, :vocab].to(dtype)
    tokens = torch.randint(-2, vocab + 2, (rows, width), device="cuda", generator=gen)
    tokens[:, 1::2] %= 7  # the same ones again and again, in every round
    tokens[:, 2::5] = vocab - 1
    lengths, prompts = (torch.randint(0, width + 1, (rows,), device="cuda", generator=gen, dtype=torch.int32) for _ in range(2))
    lengths[0], prompts[0] = width, 0
    lengths[-1], prompts[-1] = width, width // 2
    r, f, p = (torch.rand(rows, device="cuda", generator=gen) + low for low in (0.6, 0.0, -0.5))
    bias = None if form == "odd rows" else torch.randn(*(() if form == "shared" else (rows,)), vocab, device="cuda", generator=gen).to(BF16 if form == "shared" else torch.float32)
    allowed = None if form == "shared" else torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), device="cuda", generator=gen, dtype=torch.int64).int()
    args = (x, tokens, lengths, prompts, r, f, p, bias, allowed)
    want, tol = logits64(*args)
    for _ in range(3):
        got = OF.adjust_logits(*args)
        off = (got.double() - want).abs()
        bad = ~((off <= tol) | (got.double() == want))
        assert not bad.any(), f"{int(bad.sum())} off, first at {bad.nonzero()[0].tolist()}: {got[bad][0].item()} for {want[bad][0].item()} +- {tol[bad][0].item():.3g}"
    assert status_of() == 0


def _adjust(x, out, tokens=None, bias=None):
    status = native().device_state(x.device).status
    a = native().AdjustLogits(logits=x.data_ptr(), out=out.data_ptr(), status=status.data_ptr(), logits_ld=x.stride(0), out_ld=out.stride(0), rows=x.shape[0], vocab=x.shape[1],
                              dtype=int(x.dtype == torch.float32), repetition_all=1.25, presence_all=0.5)
    if tokens is not None:
        a.tokens, a.tokens_ld, a.width = tokens.data_ptr(), tokens.stride(0), tokens.shape[1]
    if bias is not None:
        a.bias, a.bias_dtype = bias.data_ptr(), 1
    native().check(native().LIB.tpb_adjust_logits(a, torch.cuda.current_stream().cuda_stream), "tpb_adjust_logits")


@pytest.mark.parametrize("rows,vocab", [(3, 1000), (40, 65000)])
def test_where_the_c_entry_writes_results(rows, vocab):
    gen = torch.Generator().manual_seed(2)
    room = numbers(gen, rows, 2 * vocab + 8, dtype=torch.float32, scale=4.0).cuda()
    bias, tokens = numbers(gen, vocab, dtype=torch.float32).cuda(), torch.randint(0, vocab, (rows, 50), generator=gen).cuda()
    x, beside = room[:, :vocab], room[:, vocab + 4:2 * vocab + 4]
    given, edges = x.clone(), room[:, vocab:vocab + 4].clone()
    # in the gaps between the rows, with a history
    _adjust(x, beside, tokens, bias)
    torch.cuda.synchronize()
    assert torch.equal(beside, OF.adjust_logits(given, tokens, None, None, 1.25, None, 0.5, bias=bias))
    assert torch.equal(x, given) and torch.equal(room[:, vocab:vocab + 4], edges)
    # in place, without one
    _adjust(x, x, None, bias)
    torch.cuda.synchronize()
    assert torch.equal(x, given + bias)


# -- append ----------------------------------------------------------------------------------------


def ragged(tokens, most, seed):
    """Numbers of new tokens that add up to ``tokens``, up to ``most`` each, some of them none."""
    gen = torch.Generator().manual_seed(seed)
    new = []
    while tokens:
        new.append(min(tokens, int(torch.randint(0, most + 1, (), generator=gen))))
        tokens -= new[-1]
    return new


@pytest.mark.parametrize("tokens", [591, 592, 1183, 1184, 1185, 4735, 4736, 4739])
@pytest.mark.parametrize("heads,kv_heads,dim,turn,norms", [(8, 2, 64, None, True), (6, 2, 128, (128, False), True), (5, 1, 64, (32, True), False), (4, 4, 32, (20, False), True), (3, 1, 256, (256, True), False)])
def test_append_of_several_tokens_to_a_block(tokens, heads, kv_heads, dim, turn, norms):
    """A token's rows over several blocks, one, two and eight tokens to a block, the last block's fewer, sequences that begin and end inside of blocks, rows of no sequence."""
    front, rest = 3, 6
    new = ragged(tokens - front - rest, 211, tokens + dim)
    gen = torch.Generator().manual_seed(dim)
    past = torch.randint(0, 400, (len(new),), generator=gen).tolist()
    past[1] = 100003
    b = batch(new, past, heads, kv_heads, dim, 16, device="cuda", seed=tokens, front=front, rest=rest, junk=0.5, only_new=True)
    assert b["q"].shape[0] == tokens
    rotary = None if turn is None else OF.Rotary(OF.rotary(turn[0], device="cuda").frequencies, turn[1], 1.25)
    norm = (1 + numbers(gen, dim, scale=0.2)).cuda() if norms else None
    before = b["keys"].clone(), b["values"].clone()
    for given in (None, torch.full_like(b["q"], 3.0)):
        q = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=rotary, q_norm=norm, k_norm=norm, out=given)
        outside = torch.cat((q[:front], q[tokens - rest:]))
        assert (outside == (0 if given is None else 3)).all()
        check_append_at_once(b, q[front:tokens - rest], before, rotary, norm)
        if given is not None:
            assert torch.equal(q[front:tokens - rest], first)
        first = q[front:tokens - rest]
    assert status_of() == 0


def check_append_at_once(b, q, before, rotary, norm, eps=1e-6):
    """As ``check_append``, all tokens at a time: ``q`` holds those of the sequences."""
    starts, past, page = b["starts"].long(), b["past"].long(), b["keys"].shape[2]
    first, last = int(starts[0]), int(starts[-1])
    of = torch.repeat_interleave(torch.arange(len(past), device=q.device), starts[1:] - starts[:-1])
    at = past[of] + torch.arange(first, last, device=q.device) - starts[of]
    want, tol = turned64(b["q"][first:last], norm, eps, at, rotary)
    within(q, want, tol, "queries")
    pages, slots = b["table"][of, at // page].long(), at % page
    want, tol = turned64(b["k"][first:last], norm, eps, at, rotary)
    within(b["keys"][pages, :, slots], want, tol, "keys")
    assert torch.equal(b["values"][pages, :, slots], b["v"][first:last])
    for now, then in zip((b["keys"], b["values"]), before):
        then = then.clone()
        then[pages, :, slots] = now[pages, :, slots]
        assert torch.equal(now.view(torch.int16), then.view(torch.int16))


def test_a_cache_with_heads_outside_of_pages_beyond_32_bits():
    """``[kv_heads, pages, page_size, head_dim]`` with 4 GB between heads, values behind the keys of each."""
    if torch.cuda.get_device_properties(0).total_memory < 20 << 30:
        pytest.skip("needs 5 GB")
    small = batch([1, 70], [130, 40], 8, 2, 64, 16, device="cuda", junk=0.0)
    pages, apart = small["keys"].shape[0], 2 ** 31 + 64 * 8
    room = torch.zeros(apart + 2 * small["keys"].numel(), dtype=BF16, device="cuda")
    far = dict(small)
    for name, at in (("keys", 0), ("values", pages * 16 * 64)):
        far[name] = room.as_strided(small["keys"].shape, (16 * 64, apart, 64, 1), at)
        far[name].copy_(small[name])
    want, tol = attention64(small)
    within(attend(far), want, tol)
    turn = OF.rotary(64, device="cuda")
    before = far["keys"].clone(), far["values"].clone()
    launches = native().launch_count
    q = OF.paged_append(cache_of(far), far["q"], far["k"], far["v"], far["starts"], far["past"], rotary=turn)
    assert native().launch_count == launches + 1
    check_append_at_once(far, q, before, turn, None)


# -- launches --------------------------------------------------------------------------------------


def launches_of(call):
    """Kernels that ``launch_count`` adds for a call, and those that a profile of it shows."""
    call()
    torch.cuda.synchronize()
    before = native().launch_count
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as seen:
        call()
        torch.cuda.synchronize()
    return native().launch_count - before, sum(e.count for e in seen.key_averages() if "tpb::" in e.key)


@pytest.mark.parametrize("new,past,heads,most_new,kernels", [([1], [100], 4, 1, 1), ([1], [5000], 4, 1, 2), ([1, 1], [5000, 3], 4, None, 2), ([70], [5], 4, 70, 2), ([70, 1], [5, 900], 4, None, 3),
                                                             ([1, 1], [30, 40], 71, 1, 2)])
@pytest.mark.parametrize("directly", [True, False])
def test_launches_of_the_attention(new, past, heads, most_new, kernels, directly):
    b = batch(new, past, heads, 1, 64, 16, device="cuda")
    scale = 1.0 if directly else 1  # (a whole number goes on in Python)
    counted, seen = launches_of(lambda: OF.paged_attention(b["q"], cache_of(b), b["starts"], b["past"], scale=scale, most_new=most_new))
    assert counted == kernels and seen in (0, kernels)  # (0: no profiler on this machine)


@pytest.mark.parametrize("rows,vocab,width,kernels", [(2, 1000, 9, 1), (128, 19000, 0, 1), (128, 19000, 9, 2)])
@pytest.mark.parametrize("penalty", [1.25, 1])
def test_launches_of_adjusted_logits(rows, vocab, width, kernels, penalty):
    x, tokens = torch.zeros(rows, vocab, device="cuda"), torch.zeros(rows, width, dtype=torch.int64, device="cuda")
    counted, seen = launches_of(lambda: OF.adjust_logits(x, tokens, repetition=penalty))  # (a whole number goes on in Python)
    assert counted == kernels and seen in (0, kernels)


# -- long contexts, nothing new, graphs and streams ------------------------------------------------


@pytest.mark.parametrize("heads,kv_heads,dim,page,new,past,window", [(4, 2, 64, 16, 1, 1000003, None), (8, 1, 128, 64, 1, 700001, None), (2, 2, 64, 256, 300, 200000, None), (2, 1, 128, 16, 70, 300000, 100000),
                                                                     (8, 1, 64, 16, 1, 2000000, 2999)])
def test_attention_of_a_million_keys(heads, kv_heads, dim, page, new, past, window):
    """Pages of a few, again and again (a table may name a page as often as it likes)."""
    gen = torch.Generator().manual_seed(1)
    total, pages, group = past + new, 97, heads // kv_heads
    b = dict(keys=numbers(gen, pages, kv_heads, page, dim).cuda(), values=numbers(gen, pages, kv_heads, page, dim).cuda(), table=torch.randint(0, pages, (1, -(-total // page)), generator=gen).int().cuda(),
             starts=torch.tensor([0, new], dtype=torch.int32).cuda(), past=torch.tensor([past], dtype=torch.int32).cuda(), q=numbers(gen, new, heads, dim, scale=1.5).cuda())
    low = 0 if window is None else max(0, past - window + 1) // page * page
    k, v = (b[name][b["table"][0, low // page:].long(), 0].reshape(-1, dim)[:total - low].double() for name in ("keys", "values"))
    q = b["q"][:, :group].double()
    scores = torch.einsum("tgd,jd->gtj", q, k) / math.sqrt(dim)
    size = (torch.einsum("tgd,jd->gtj", q.abs(), k.abs()) / math.sqrt(dim)).amax(-1).t()[..., None]
    far = torch.arange(past, total, device="cuda")[:, None] - torch.arange(low, total, device="cuda")[None]
    p = torch.softmax(scores.masked_fill((far < 0) | (far >= (window or 1 << 40)), -math.inf), -1)
    want, a = torch.einsum("gtj,jd->tgd", p, v), torch.einsum("gtj,jd->tgd", p, v.abs())
    # as attention64: probabilities and results to bf16, scores and sums in 32 bits
    tol = (2.0 ** -8 + 2 * (dim + 4) * 2.0 ** -24 * size + len(k) * 2.0 ** -24) * a * 1.02 + 2.0 ** -8 * want.abs() * 1.02
    for most_new in (None, new):
        within(attend(b, window=window, most_new=most_new)[:, :group], want, tol)
    assert status_of() == 0


def test_no_new_tokens_at_all():
    b = batch([0, 0, 0], [900, 5, 0], 4, 2, 64, 16, device="cuda", rest=5, front=2)
    for most_new in (0, None):
        assert not attend(b, most_new=most_new).any()
        out = torch.full_like(b["q"], 2.0)
        attend(b, most_new=most_new, out=out)
        assert (out == 2).all()
    before = b["keys"].clone()
    q = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=OF.rotary(64, device="cuda"))
    assert not q.any() and torch.equal(b["keys"].view(torch.int16), before.view(torch.int16)) and status_of() == 0


def test_captured_logits_of_two_kernels_at_once():
    """Two graphs, each of a stream and its seen entries, replayed on two streams while histories change."""
    rows, vocab, width = 130, 19001, 5000
    gen = torch.Generator(device="cuda").manual_seed(4)

    def make():
        x, tokens = torch.randn(rows, vocab, device="cuda", generator=gen), torch.randint(-3, vocab + 3, (rows, width), device="cuda", generator=gen)
        tokens[:, ::2] %= 11
        lengths, prompts = (torch.randint(0, width + 1, (rows,), device="cuda", generator=gen, dtype=torch.int32) for _ in range(2))
        args = [x, tokens, lengths, prompts, *(torch.rand(rows, device="cuda", generator=gen) + 0.6 for _ in range(3))]
        OF.adjust_logits(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = OF.adjust_logits(*args)
        return args, graph, out, torch.cuda.Stream()

    both = [make(), make()]
    for _ in range(3):
        for args, *_ in both:
            args[0].normal_(generator=gen)
            args[1].copy_(args[1].roll(7, 1))
            args[2].copy_((args[2] + 613) % (width + 1))
        torch.cuda.synchronize()
        for _ in range(4):
            for _, graph, _, stream in both:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for args, _, out, _ in both:
            want, tol = logits64(*args, None, None)
            within(out, want, tol)
    assert status_of() == 0
