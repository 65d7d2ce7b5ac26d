"""Kernels of a paged cache and of adjusted logits against 64 bits, and what they are handed at the edges."""
import math

import pytest
import torch
import torch.fx.experimental.proxy_tensor
import torch.utils.flop_counter

from paged_cases import BF16, append64, attention64, batch, check_append, check_logits, numbers, within
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


# -- attention -----------------------------------------------------------------------------------


@pytest.mark.parametrize("new,past", [([1], [0]), ([1], [63]), ([1], [64]), ([1, 1, 1], [5, 200, 1000]), ([2, 0, 5, 1], [15, 7, 16, 700]), ([16], [48]), ([17, 3], [0, 130]),
                                      ([33, 1, 70], [100, 0, 59]), ([129], [0]), ([300, 1, 257], [0, 513, 40])])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 128, 16), (8, 2, 64, 16), (7, 1, 128, 64), (16, 1, 64, 32), (6, 3, 64, 128), (5, 5, 128, 256)])
def test_attention(new, past, heads, kv_heads, dim, page):
    b = batch(new, past, heads, kv_heads, dim, page, device="cuda", seed=len(new) + heads, rest=3)
    out = attend(b)
    want, tol = attention64(b)
    within(out, want, tol)
    out = attend(b, most_new=max(new))
    within(out, want, tol)
    assert status_of() == 0


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 200, 5000])
@pytest.mark.parametrize("new,past", [([1, 1], [500, 63]), ([6, 1], [130, 700]), ([200, 3, 1], [77, 0, 300])])
def test_attention_with_a_window(new, past, window):
    b = batch(new, past, 8, 2, 64, 16, device="cuda", seed=window)
    # pages that every token has left behind may be another's by now
    for s, p in enumerate(past):
        gone = max(0, p - window + 1) // 16
        b["table"][s, :gone] = -5
    clean = batch(new, past, 8, 2, 64, 16, device="cuda", seed=window)
    want, tol = attention64(clean, window=window)
    within(attend(b, window=window), want, tol)
    within(attend(b, window=window, most_new=max(new)), want, tol)
    assert status_of() == 0


@pytest.mark.parametrize("heads,kv_heads,dim", [(71, 1, 64), (12, 12, 64), (40, 8, 128), (64, 2, 128)])
def test_attention_of_a_long_context(heads, kv_heads, dim):
    """One sequence over the whole GPU, cut into many pieces."""
    b = batch([1], [9999], heads, kv_heads, dim, 16, device="cuda")
    want, tol = attention64(b)
    within(attend(b, most_new=1), want, tol)
    within(attend(b), want, tol)


def test_attention_of_many_sequences():
    gen = torch.Generator().manual_seed(9)
    new = torch.randint(0, 3, (700,), generator=gen).tolist()
    past = torch.randint(0, 90, (700,), generator=gen).tolist()
    b = batch(new, past, 4, 2, 64, 16, device="cuda", seed=4, front=2, rest=5)
    want, tol = attention64(b)
    within(attend(b, most_new=2), want, tol)
    within(attend(b), want, tol)
    assert status_of() == 0


def test_attention_scale_and_peaked_scores():
    b = batch([3, 1], [400, 90], 8, 2, 128, 32, device="cuda")
    for scale in (1e-6, 0.3, 2.0):
        want, tol = attention64(b, scale=scale)
        within(attend(b, scale=scale), want, tol)


def test_attention_of_strided_views():
    b = batch([2, 40, 1], [37, 0, 300], 8, 2, 64, 16, device="cuda", junk=0.0)
    want, tol = attention64(b)
    pages = b["keys"].shape[0]
    # heads inside of slots, keys beside values, layers of one tensor
    inside = torch.zeros(pages, 2, 16, 2, 2, 64, dtype=BF16, device="cuda")
    inside[:, 0, :, :, 1], inside[:, 1, :, :, 1] = b["keys"].transpose(1, 2), b["values"].transpose(1, 2)
    held = dict(b, keys=inside[:, 0, :, :, 1].transpose(1, 2), values=inside[:, 1, :, :, 1].transpose(1, 2))
    assert not held["keys"].is_contiguous()
    within(attend(held), want, tol)
    # queries inside of a projection, and rows that no vector load can take
    wide = torch.zeros(43, 24, 64, dtype=BF16, device="cuda")
    wide[:, 3:11] = b["q"]
    within(attend(dict(b, q=wide[:, 3:11])), want, tol)
    odd = torch.zeros(43 * 8 * 64 + 1, dtype=BF16, device="cuda")[1:].view(43, 8, 64)
    odd.copy_(b["q"])
    within(attend(dict(b, q=odd)), want, tol)
    # results between other rows, lengths and table as parts of larger tensors
    room = torch.full((43, 16, 64), 7.0, dtype=BF16, device="cuda")
    table = torch.full((3, 100), -1, dtype=torch.int32, device="cuda")
    table[:, 1:1 + b["table"].shape[1]] = b["table"]
    past = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    past[:, 1] = b["past"]
    view = dict(b, table=table[:, 1:1 + b["table"].shape[1]], past=past[:, 1])
    attend(view, out=room[:, 4:12])
    within(room[:, 4:12], want, tol)
    assert (room[:, :4] == 7).all() and (room[:, 12:] == 7).all()
    # in place of the queries
    q = b["q"].clone()
    assert attend(dict(b, q=q), out=q) is q
    within(q, want, tol)


@pytest.mark.parametrize("most_new", [1, None])
def test_attention_leaves_rows_outside_alone(most_new):
    b = batch([1, 1], [100, 3], 4, 4, 128, 16, device="cuda", front=1, rest=6)
    out = torch.full_like(b["q"], 5.0)
    attend(b, out=out, most_new=most_new)
    want, tol = attention64(b)
    within(out[1:3], want[1:3], tol[1:3])
    assert (out[0] == 5).all() and (out[3:] == 5).all()
    assert not attend(b, most_new=most_new)[[0, 3, 4, 5, 6, 7, 8]].any()


def test_no_sequences_and_no_tokens():
    b = batch([1, 1], [5, 9], 4, 4, 64, 16, device="cuda")
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    empty = OF.PagedCache(b["keys"], b["values"], b["table"][:0])
    assert not OF.paged_attention(b["q"], empty, none, none[:0]).any()
    q = OF.paged_append(empty, b["q"], b["k"], b["v"], none, none[:0], rotary=OF.rotary(64, device="cuda"))
    assert q.shape == b["q"].shape and not q.any()
    assert OF.paged_attention(b["q"][:0], cache_of(b), torch.zeros(3, dtype=torch.int32, device="cuda"), b["past"]).shape == (0, 4, 64)
    assert not OF.paged_attention(b["q"], cache_of(b), torch.zeros(3, dtype=torch.int32, device="cuda"), b["past"]).any()
    assert status_of() == 0


def test_values_that_are_not_finite_stay_with_their_sequence():
    """Slots of no sequence hold NaN in all these batches; infinities in one sequence's own keys and values reach its rows alone."""
    b = batch([1, 1, 1], [90, 90, 90], 4, 4, 64, 16, device="cuda")
    want, tol = attention64(b)
    b["values"][b["table"][1, 0].long(), :, 3] = math.inf
    b["keys"][b["table"][2, 1].long(), :, 3] = math.nan
    out = attend(b)
    within(out[:1], want[:1], tol[:1])
    assert (out[1] == math.inf).all() and out[2].isnan().all()


def test_attention_at_offsets_beyond_32_bits():
    pages, page, heads, dim = 17000, 64, 16, 128  # 2.2e9 elements of keys
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 10 GB")
    small = batch([1, 70], [130, 40], 16, heads, dim, page, device="cuda")
    keys, values = (torch.empty(pages, heads, page, dim, dtype=BF16, device="cuda") for _ in range(2))
    moved = small["table"].clone()
    for s, j in ((s, j) for s in range(2) for j in range(moved.shape[1]) if int(moved[s, j]) >= 0):
        moved[s, j] = pages - 1 - int(small["table"][s, j])
        keys[int(moved[s, j])], values[int(moved[s, j])] = small["keys"][int(small["table"][s, j])], small["values"][int(small["table"][s, j])]
    want, tol = attention64(small)
    big = dict(small, keys=keys, values=values, table=moved)
    within(attend(big), want, tol)
    within(attend(big, most_new=70), want, tol)
    turn = OF.rotary(dim, device="cuda")
    q, tq, stored = append64(big, turn)
    within(OF.paged_append(cache_of(big), big["q"], big["k"], big["v"], big["starts"], big["past"], rotary=turn), q, tq)
    for at, slot, k, tk, v in stored:
        within(keys[at, :, slot], k, tk)
        assert torch.equal(values[at, :, slot], v)


# -- lengths and pages that do not fit ---------------------------------------------------------------


@pytest.mark.parametrize("most_new", [None, 2])
@pytest.mark.parametrize("what", ["rows", "back", "negative", "past", "room", "page", "pages"])
def test_attention_of_lengths_that_do_not_fit(what, most_new):
    b = batch([1, 2, 1], [100, 40, 7], 4, 2, 64, 16, device="cuda")
    want, tol = attention64(b)
    bad = {k: t.clone() for k, t in b.items()}
    if what == "rows":
        bad["starts"][3] = 9
    elif what == "back":
        bad["starts"][2] = 0
    elif what == "negative":
        bad["starts"][0] = -4
    elif what == "past":
        bad["past"][1] = -3
    elif what == "room":
        bad["past"][1] = 2 ** 31 - 2
    elif what == "page":
        bad["table"][1, 0] = bad["keys"].shape[0]
    else:
        bad["table"][1, 2] = -2 ** 31
    assert status_of() == 0
    out = attend(bad, most_new=most_new)
    assert status_of() == 3
    if what in ("past", "room", "page", "pages"):
        rows = [1, 2]
    else:
        rows = {"rows": [3], "back": [0, 1, 2, 3], "negative": [0]}[what]
    for r in range(4):
        if r in rows:
            assert what == "back" or out[r].isnan().all()
        else:
            within(out[r], want[r], tol[r])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,past,row0", [([200], [700], 0), ([1, 300, 1], [90, 100, 400], 1), ([1, 600], [3000, 2000], 1)])
def test_attention_of_chunks_whose_pages_are_not_there(new, past, row0, dim):
    b = batch(new, past, 4, 2, dim, 16, device="cuda")
    want, tol = attention64(b)
    chunk = max(range(len(new)), key=lambda s: new[s])
    bad = dict(b, table=b["table"].clone())
    bad["table"][chunk, 5] = 10 ** 9
    out = attend(bad)
    assert status_of() == 3 and out[row0:row0 + new[chunk]].isnan().all()
    others = [r for r in range(sum(new)) if not row0 <= r < row0 + new[chunk]]
    within(out[others], want[others], tol[others])
    bad = dict(b, past=b["past"].clone())
    bad["past"][chunk] = 2 ** 30
    out = attend(bad)
    assert status_of() == 3 and out[row0:row0 + new[chunk]].isnan().all()
    within(out[others], want[others], tol[others])


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (14, 2), (71, 1), (8, 8)])
def test_chunks_by_boxes_and_by_rows(heads, kv_heads):
    """Query rows of whole tokens come by boxes, those of 7 or 71 heads and broadcast ones by rows."""
    b = batch([130, 257, 1, 40], [300, 0, 60, 1000], heads, kv_heads, 128, 32, device="cuda", rest=5)
    want, tol = attention64(b)
    within(attend(b), want, tol)
    one = b["q"][:, :1].expand(-1, heads, -1)
    want, tol = attention64(dict(b, q=one.contiguous()))
    within(OF.paged_attention(one, cache_of(b), b["starts"], b["past"]), want, tol)
    q = b["q"].clone()
    want, tol = attention64(b)
    assert attend(dict(b, q=q), out=q) is q
    used = int(b["starts"][-1])
    within(q[:used], want[:used], tol[:used])
    assert torch.equal(q[used:], b["q"][used:])


def test_attention_of_more_new_tokens_than_said():
    b = batch([1, 5, 2], [100, 40, 7], 4, 2, 64, 16, device="cuda")
    want, tol = attention64(b)
    out = attend(b, most_new=2)
    assert status_of() == 3 and out[1:6].isnan().all()
    within(out[[0, 6, 7]], want[[0, 6, 7]], tol[[0, 6, 7]])


@pytest.mark.parametrize("what", ["rows", "back", "past", "room", "page"])
def test_append_of_lengths_that_do_not_fit(what):
    b = batch([1, 2, 1], [100, 40, 7], 4, 2, 64, 16, device="cuda")
    before = {k: t.clone() for k, t in b.items()}
    if what == "rows":
        b["starts"][3] = 9
    elif what == "back":
        b["starts"][2] = 0
    elif what == "past":
        b["past"][1] = -3
    elif what == "room":
        b["past"][1] = 2 ** 31 - 2
    else:
        b["table"][1, 2] = b["keys"].shape[0]
    OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=OF.rotary(64, device="cuda"))
    assert status_of() == 3
    # nothing but slots that the batch names has changed: those of its sequences, and where rows 0 to 4 have become the last one's, the four behind its keys
    slots = [place[:2] for place in append64(before)[2]]
    if what == "back":
        slots = [(int(b["table"][2, 0]), 7 + i) for i in range(4)]
    rest = before["values"].clone()
    for page, slot in slots:
        rest[page, :, slot] = b["values"][page, :, slot]
    assert torch.equal(b["values"].view(torch.int16), rest.view(torch.int16))
    if what != "back":
        assert torch.equal(b["values"][slots[0][0], :, slots[0][1]], b["v"][0])


# -- append --------------------------------------------------------------------------------------


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 32, 128, 16), (8, 2, 64, 32), (7, 1, 256, 64), (71, 1, 64, 16), (5, 3, 80, 1), (4, 4, 96, 8), (2, 1, 8, 4)])
@pytest.mark.parametrize("turn", [None, (1.0, False, 1.0), (1.0, True, 1.3), (0.25, False, 0.8), (0.25, True, 1.0), (0.5, False, 1.0)])
@pytest.mark.parametrize("norms", [False, True])
def test_append(heads, kv_heads, dim, page, turn, norms):
    b = batch([1, 3, 0, 40, 1], [255, 0, 9, 17, 131071], heads, kv_heads, dim, page, device="cuda", front=1, rest=2, junk=0.5, only_new=True)
    gen = torch.Generator().manual_seed(5)
    part = 0 if turn is None else max(2, int(dim * turn[0]) // 2 * 2)
    rotary = None if turn is None else OF.Rotary(OF.rotary(part, 10000.0, device="cuda").frequencies, turn[1], turn[2])
    q_norm, k_norm = ((1 + numbers(gen, dim, scale=0.2)).cuda() if norms else None for _ in range(2))
    before = b["keys"].clone(), b["values"].clone()
    launches = native().launch_count
    q = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=rotary, q_norm=q_norm, k_norm=k_norm, eps=1e-5)
    assert native().launch_count == launches + 1
    if rotary is None and not norms:
        assert q is b["q"]
        q = torch.cat((q[:1] * 0, q[1:-2], q[-2:] * 0))
    check_append(b, q, before, rotary, q_norm, k_norm, 1e-5)
    assert status_of() == 0


def test_append_of_one_norm_in_place_and_of_many_tokens():
    b = batch([700, 123, 1], [0, 50, 300], 8, 2, 128, 64, device="cuda", rest=2)
    turn = OF.rotary(128, device="cuda")
    norm = (1 + 0.1 * torch.randn(128)).to(BF16).cuda()
    before = b["keys"].clone(), b["values"].clone()
    q, given = b["q"].clone(), b["q"].clone()
    assert OF.paged_append(cache_of(b), q, b["k"], b["v"], b["starts"], b["past"], rotary=turn, k_norm=norm, out=q) is q
    assert torch.equal(q[-2:], given[-2:])
    check_append(b, torch.cat((q[:-2], q[-2:] * 0)), before, turn, None, norm)
    q = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], q_norm=norm)
    check_append(b, q, before, None, norm, None)
    assert OF.paged_append(cache_of(b), None, b["k"], b["v"], b["starts"], b["past"], rotary=turn, k_norm=norm) is None


def test_append_of_views():
    b = batch([3, 1, 20], [14, 77, 0], 6, 2, 64, 16, device="cuda", junk=0.0)
    turn = OF.rotary(32, device="cuda")
    qkv = torch.randn(24, 10, 64, device="cuda").to(BF16)
    b["q"], b["k"], b["v"] = qkv.split([6, 2, 2], dim=1)
    both = torch.zeros(b["keys"].shape[0], 16, 2, 2, 64, dtype=BF16, device="cuda")  # slots of heads, keys beside values
    b["keys"], b["values"] = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    before = b["keys"].clone(), b["values"].clone()
    q = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=turn)
    check_append(b, q, before, turn)
    b["k"], b["v"] = b["k"][:, :1].expand(24, 2, 64), torch.randn(24, 64, 2, device="cuda").to(BF16).transpose(1, 2)  # broadcast, and columns of rows
    q = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=turn)
    check_append(b, q, before, turn)


def test_other_types_go_by_their_steps():
    b = batch([3, 1], [14, 77], 4, 2, 32, 16, dtype=torch.float32, device="cuda")
    want, tol = attention64(b)
    within(OF.paged_attention(b["q"], cache_of(b), b["starts"], b["past"]), want, tol + 1e-5)
    before = b["keys"].clone(), b["values"].clone()
    turn = OF.rotary(32, device="cuda")
    check_append(b, OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=turn), before, turn)


# -- logits --------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("rows,vocab,width", [(1, 1, 1), (3, 1000, 20), (2, 1025, 300), (5, 9001, 0), (2, 50257, 64), (700, 37, 9)])
def test_adjusted_logits(rows, vocab, width, dtype):
    gen = torch.Generator().manual_seed(rows * vocab)
    logits = numbers(gen, rows, vocab, dtype=dtype, scale=4.0)
    tokens = torch.randint(-2, vocab + 2, (rows, width), generator=gen)
    tokens[:, width // 2:] = tokens[:, width // 2:] % 7
    lengths, prompts = (torch.randint(0, width + 1, (rows,), generator=gen, dtype=torch.int32) for _ in range(2))
    r, f, p = (torch.rand(rows, generator=gen) + low for low in (0.6, 0.0, -0.5))
    bias = numbers(gen, rows, vocab, dtype=torch.float32)
    allowed = torch.randint(-2 ** 31, 2 ** 31, (rows, (vocab + 31) // 32), generator=gen).int()
    for args in ((logits, tokens, lengths, prompts, r, f, p, bias, allowed), (logits, tokens, None, None, 1.3, 0.2, 0.4),
                 (logits, None, None, None, None, None, None, bias[0].to(BF16), allowed[0]), (logits,)):
        launches = native().launch_count
        got = OF.adjust_logits(*(t.cuda() if isinstance(t, torch.Tensor) else t for t in args))
        assert native().launch_count == launches + 1
        check_logits(got.cpu(), args)
    assert status_of() == 0


def test_adjusted_logits_of_views_and_odd_lengths():
    gen = torch.Generator().manual_seed(1)
    three = numbers(gen, 4, 3, 999, dtype=torch.float32).cuda()
    tokens = torch.randint(0, 999, (4, 50), generator=gen).cuda()
    args = (three[:, -1], tokens[:, 5:45], None, None, 1.2)
    check_logits(OF.adjust_logits(*args).cpu(), tuple(t.cpu() if isinstance(t, torch.Tensor) else t for t in args))
    for view in (three[:, 1, 1:], three[:, 0, ::2], three[:1, 0].expand(4, 999)):
        check_logits(OF.adjust_logits(view, tokens, presence=0.5).cpu(), (view.cpu(), tokens.cpu(), None, None, None, None, 0.5))
    lengths = torch.tensor([-3, 60, 0, 50], dtype=torch.int32, device="cuda")
    out = OF.adjust_logits(three[:, 0], tokens, lengths, frequency=0.25)
    assert status_of() == 3
    check_logits(out.cpu(), (three[:, 0].cpu(), tokens.cpu(), lengths.cpu(), None, None, 0.25))


# -- graphs, streams, a run of them together ---------------------------------------------------------


def test_a_captured_step_follows_its_lengths():
    """One graph of append and attention, replayed while the batch grows, and a second one on another stream at the same time."""
    heads, kv_heads, dim, page, n, room = 8, 2, 64, 16, 4, 400
    turn = OF.rotary(dim, device="cuda")

    def make(seed):
        gen = torch.Generator().manual_seed(seed)
        pages = n * room // page
        b = dict(keys=torch.zeros(pages, kv_heads, page, dim, dtype=BF16).cuda(), values=torch.zeros(pages, kv_heads, page, dim, dtype=BF16).cuda(),
                 table=torch.randperm(pages, generator=gen).int().view(n, -1).cuda(), starts=torch.zeros(n + 1, dtype=torch.int32).cuda(), past=torch.zeros(n, dtype=torch.int32).cuda(),
                 q=numbers(gen, 40, heads, dim).cuda(), k=numbers(gen, 40, kv_heads, dim).cuda(), v=numbers(gen, 40, kv_heads, dim).cuda())
        b["turned"], b["out"] = torch.zeros_like(b["q"]), torch.zeros_like(b["q"])

        def step():
            OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=turn, out=b["turned"])
            OF.paged_attention(b["turned"], cache_of(b), b["starts"], b["past"], out=b["out"])

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        return b, graph, gen, torch.cuda.Stream()

    both = [make(1), make(2)]
    past = [0] * n
    for new in ([20, 1, 0, 13], [1, 1, 1, 1], [7, 30, 1, 2], [1, 0, 1, 1], [1, 1, 1, 37]):
        for b, graph, gen, stream in both:
            b["starts"].copy_(torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()]))
            b["past"].copy_(torch.tensor(past))
            for name in "qkv":
                b[name].copy_(numbers(gen, *b[name].shape))
            b["out"].fill_(9)
        torch.cuda.synchronize()
        for _ in range(3):
            for b, graph, gen, stream in both:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for b, *_ in both:
            want, tol = attention64(dict(b, q=b["turned"]))
            used = sum(new)
            within(b["out"][:used], want[:used], tol[:used])
            assert (b["out"][used:] == 9).all()
        past = [p + m for p, m in zip(past, new)]
    assert status_of() == 0


def test_calls_on_two_streams_at_once():
    batches = [batch([1] * 5 + [30], [3000, 100, 2000, 5, 700, 900], 8, 2, 128, 16, device="cuda", seed=s) for s in range(2)]
    wants = [attention64(b) for b in batches]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(attend(batches[i]))
    torch.cuda.synchronize()
    for got, (want, tol) in zip(outs, wants):
        for o in got:
            within(o, want, tol)
            assert torch.equal(o, got[0])  # (no result depends on timing)


def test_a_step_of_a_served_batch():
    """Append, attention, projection to logits, their adjustment and the pick, for a batch of chunks and single tokens, against the same steps in 64 bits."""
    b = batch([1, 60, 1, 7], [300, 0, 17, 90], 8, 2, 64, 16, device="cuda", seed=8)
    gen = torch.Generator().manual_seed(3)
    turn, norm = OF.rotary(64, 10000.0, device="cuda"), (1 + numbers(gen, 64, scale=0.1)).cuda()
    head = numbers(gen, 1000, 512, scale=0.2).cuda()
    q = OF.paged_append(cache_of(b), b["q"], b["k"], b["v"], b["starts"], b["past"], rotary=turn, q_norm=norm, k_norm=norm)
    out = OF.paged_attention(q, cache_of(b), b["starts"], b["past"])
    want, tol = attention64(dict(b, q=q))
    within(out, want, tol)
    last = out[b["starts"][1:].long() - 1].flatten(1)
    logits = OF.linear(last, head)
    tokens = torch.randint(0, 1000, (4, 300), generator=gen).cuda()
    allowed = torch.randint(-2 ** 31, 2 ** 31, (4, 32), generator=gen).int().cuda()
    lengths = b["past"].clone()
    args = (logits, tokens, lengths, None, 1.2, 0.1, 0.3, None, allowed)
    got = OF.adjust_logits(*args)
    check_logits(got.cpu(), tuple(t.cpu() if isinstance(t, torch.Tensor) else t for t in args))
    picks = got.argmax(-1)
    assert all(int(allowed[r, t // 32]) >> (t % 32) & 1 for r, t in enumerate(picks.tolist()))


def test_what_is_compiled_or_traced():
    b = batch([1, 3], [30, 5], 4, 2, 64, 16, device="cuda")
    want, tol = attention64(b)
    with pytest.raises(RuntimeError, match="traced"):
        torch.fx.experimental.proxy_tensor.make_fx(lambda q: OF.paged_attention(q, cache_of(b), b["starts"], b["past"]))(b["q"])
    with torch.utils.flop_counter.FlopCounterMode(display=False):
        within(attend(b), want, tol)
    within(torch.compile(lambda q: OF.paged_attention(q * 1.0, cache_of(b), b["starts"], b["past"]) * 1.0, backend="eager")(b["q"]), want, tol)


def test_negative_views_and_numbers_that_are_not_ordinary():
    b = batch([1, 80], [30, 5], 4, 2, 64, 16, device="cuda", junk=0.0)
    want, tol = attention64(b)
    within(attend(dict(b, q=torch._neg_view(-b["q"]))), want, tol)
    within(OF.paged_attention(b["q"], OF.PagedCache(torch._neg_view(-b["keys"]), torch._neg_view(-b["values"]), b["table"]), b["starts"], b["past"]), want, tol)
    within(attend(b, scale=1 / 8, window=2 ** 40, most_new=2 ** 40), want, tol)
    x, t = torch.randn(3, 100, device="cuda"), torch.randint(0, 100, (3, 9), device="cuda")
    assert torch.equal(OF.adjust_logits(torch._neg_view(-x), t, None, None, 2), OF.adjust_logits(x, t, None, None, 2.0))


def test_falcon_heads_and_bad_lengths_without_the_kernel_for_few_rows():
    """71 query heads of one KV head are more rows than the kernel for few takes."""
    b = batch([1, 1, 2, 1], [100, 40, 7, 300], 71, 1, 64, 16, device="cuda", front=1, rest=2)
    want, tol = attention64(b)
    within(attend(b, most_new=2), want, tol)
    assert status_of() == 0
    b["past"][1] = -5
    out = attend(b, most_new=2)
    assert status_of() == 3 and out[2].isnan().all()
    within(out[[0, 1, 3, 4, 5, 6, 7]], want[[0, 1, 3, 4, 5, 6, 7]], tol[[0, 1, 3, 4, 5, 6, 7]])


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (8, 2, 64), (64, 2, 128), (20, 1, 64), (64, 1, 64)])
@pytest.mark.parametrize("new,past,window", [([1] * 40 + [70], [900 + 37 * i for i in range(40)] + [0], None), ([1, 600], [0, 900], None), ([300, 1, 1, 128], [0, 2000, 5, 128], None),
                                             ([1] * 400 + [65] * 3, [i % 50 for i in range(403)], 33), ([1, 0, 2], [300, 0, 70], None)])
def test_decoding_sequences_beside_chunks(new, past, window, heads, kv_heads, dim):
    """The SMs that either launch gets follow from the lengths: almost all for one, almost all for the other, all."""
    b = batch(new, past, heads, kv_heads, dim, 16, device="cuda", rest=2)
    want, tol = attention64(b, window=window)
    out = attend(b, window=window)
    within(out, want, tol)
    assert torch.equal(out, attend(b, window=window)) and status_of() == 0


def test_bad_lengths_beside_a_chunk():
    b = batch([1, 200, 2, 1], [100, 40, 7, 300], 8, 2, 128, 16, device="cuda")
    want, tol = attention64(b)
    for s, rows in ((0, slice(0, 1)), (1, slice(1, 201)), (2, slice(201, 203))):
        past = b["past"].clone()
        past[s] = -5
        out = attend(dict(b, past=past))
        assert status_of() == 3 and out[rows].isnan().all()
        keep = torch.ones(len(out), dtype=torch.bool)
        keep[rows] = False
        within(out[keep], want[keep], tol[keep])


@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (8, 2), (64, 2), (12, 2)])
@pytest.mark.parametrize("dim", [64, 128])
def test_results_of_chunks_go_to_their_rows_only(heads, kv_heads, dim):
    b = batch([260, 131, 160], [0, 70, 1000], heads, kv_heads, dim, 32, device="cuda", front=3, rest=5)
    want, tol = attention64(b)
    room = torch.full((len(b["q"]) + 2, heads + 3, dim + 16), 7.0, dtype=BF16, device="cuda")
    out = room[1:-1, 2:-1, 8:-8]
    attend(b, out=out)
    within(out[3:-5], want[3:-5], tol[3:-5])
    out[3:-5].fill_(7.0)  # (rows outside of all sequences are left as they were where the caller gives the result's place)
    assert (room == 7.0).all()
