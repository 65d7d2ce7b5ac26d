"""Operators of serving sequences of different lengths: what they are measured on.

One step of such a batch appends the keys and values of its new tokens to a paged cache, with the norms of queries and keys and the position
rotation applied on the way (``append``), lets the new tokens attend to the pages of their sequences (``attend``), and adjusts the logits of
every sequence by what it has said already, its biases and the tokens its grammar allows (``logits``).  Heads and widths are those of the
model configurations in ``tensor_parallel_b200/models`` (7B: 32 heads of 128; Falcon-40B: 128 query and 8 KV heads of 64; GPT-J: 16 heads of
256, a quarter of each rotated in interleaved pairs), batch sizes and lengths those of the benchmark (8 x 2048) and ragged ones around them.

``exact`` restates every operator in 64-bit PyTorch, with none of this package's code.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
EPS = 1e-6


def _text(numbers):
    """A case holds plain values: lengths as a text, a word for each sequence."""
    return " ".join(str(n) for n in numbers)


def _numbers(text):
    return [int(word) for word in text.split()]


def listed():
    prompts = _text([2048, 1999, 2501, 1024, 2200, 1777, 2050, 2785])
    return [
        # one sequence's new token: all latency
        dict(name="append_token", kind="append", new="1", past="255", heads=32, kv_heads=32, dim=128, page=16, rotary=128, interleaved=False,
             norms=False, scaled=False),
        # a decode step of 64 sequences in the middle of their answers, with norms of queries and keys
        dict(name="append_decode", kind="append", new=_text([1] * 64), past=_text(37 + 61 * i for i in range(64)), heads=32, kv_heads=8, dim=128, page=16,
             rotary=128, interleaved=False, norms=True, scaled=False),
        # a ragged chunk of GPT-J: interleaved pairs, a quarter of the head, behind a prefix
        dict(name="append_partial", kind="append", new="333 1 410 257", past="0 999 128 77", heads=16, kv_heads=16, dim=256, page=32, rotary=64,
             interleaved=True, norms=False, scaled=False),
        # prompts of eight sequences, frequencies stretched for a long context, far positions
        dict(name="append_prompt", kind="append", new=prompts, past="0 0 30000 0 0 100000 0 0", heads=32,
             kv_heads=8, dim=128, page=64, rotary=128, interleaved=False, norms=True, scaled=True),
        # one sequence's new token, a short context: all latency
        dict(name="attend_token", kind="attend", new="1", past="255", heads=32, kv_heads=32, dim=128, page=16, window=0),
        # the decode step of the benchmark, 8 x 2048
        dict(name="attend_decode", kind="attend", new=_text([1] * 8), past=_text([2048] * 8), heads=32, kv_heads=32, dim=128, page=16, window=0),
        # a decode step of sequences of very different lengths, 16 query heads to a KV head
        dict(name="attend_ragged", kind="attend", new=_text([1] * 48), past=_text([97 + 3 * i * i for i in range(47)] + [30011]), heads=128, kv_heads=8, dim=64, page=64,
             window=0),
        # a chunk of a long prompt over what is cached of it
        dict(name="attend_chunk", kind="attend", new="512", past="32000", heads=32, kv_heads=8, dim=128, page=16, window=0),
        # decoding sequences and a chunk of a prompt in one step, with a sliding window
        dict(name="attend_mixed", kind="attend", new=_text([1] * 15 + [777] + [1] * 16), past=_text(411 + 199 * i for i in range(32)), heads=32, kv_heads=8, dim=128,
             page=32, window=4096),
        # prompts of eight sequences
        dict(name="attend_prompt", kind="attend", new=prompts, past="0 0 512 0 0 1000 0 0", heads=32,
             kv_heads=32, dim=128, page=64, window=0),
        # a decode step of the benchmark's batch: penalties
        dict(name="logits_step", kind="logits", rows=8, vocab=32000, width=2304, dtype="bf16", penalties=True, bias="none", mask=False),
        # a large batch over a large vocabulary: penalties, a bias for all and a grammar's mask for each
        dict(name="logits_batch", kind="logits", rows=128, vocab=65024, width=1000, dtype="fp32", penalties=True, bias="shared", mask=True),
    ]


def _spread(rng, low, high, step=1):
    """A whole number in [low, high], even over the logarithm, a multiple of ``step``."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(value / step)) * step))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "logits"])
    if kind == "logits":
        penalties = rng.random() < 0.75
        vocab = _spread(rng, 1000, 260000, rng.choice([1, 8, 64]))
        rows = _spread(rng, 1, max(1, min(256, 128 * 65024 // vocab)))
        return dict(kind=kind, rows=rows, vocab=vocab, width=_spread(rng, 16, 4096), dtype=rng.choice(["bf16", "fp32"]), penalties=penalties,
                    bias=rng.choice(["none", "shared", "rows"]) if vocab * rows < 4000000 else "none", mask=not penalties or rng.random() < 0.5)
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (64, 8), (128, 8), (28, 4), (16, 16), (12, 12), (71, 1), (5, 1), (40, 40), (48, 16)])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        dim = rng.choice([64, 128, 128, 256])
        n = _spread(rng, 1, 64)
        most = max(1, 16384 * 48 * 128 // ((heads + 2 * kv_heads) * dim) // n)
        longest = _spread(rng, 1, min(4096, most))
        rotary = rng.choice([dim, dim, dim // 2, dim // 4, 0])
        return dict(kind=kind, new=_text(rng.randint(1, longest) for _ in range(n)),
                    past=_text(rng.randint(0, _spread(rng, 1, 100000 if n < 9 else 4000)) for _ in range(n)),
                    heads=heads, kv_heads=kv_heads, dim=dim, page=page, rotary=rotary, interleaved=rng.random() < 0.4, norms=rng.random() < 0.5,
                    scaled=rng.random() < 0.5)
    dim = rng.choice([64, 128, 128])
    form = rng.choice(["decode", "decode", "few", "chunks", "mixed"])
    n = _spread(rng, 1, 96)
    reach = _spread(rng, 16, max(64, min(32768, 6000000 // (n * kv_heads * dim // 64))))
    past = [rng.randint(0, reach) for _ in range(n)]
    if form == "decode":
        new = [1] * n
    elif form == "few":
        new = [rng.randint(1, 6) for _ in range(n)]
    else:
        room = 2048 * 16000 * 32 * 128 // (heads * dim) // 8  # (query, key) pairs of a head
        new = []
        for p in past:
            most = max(1, int(math.sqrt(p * p + 2 * room / n) - p) // 2)
            new.append(_spread(rng, 1, min(2048, most)) if form == "chunks" or rng.random() < 0.2 else 1)
    return dict(kind=kind, new=_text(new), past=_text(past), heads=heads, kv_heads=kv_heads, dim=dim, page=page, window=rng.choice([0, 0, 0, _spread(rng, 16, 4096)]))


def _starts(new):
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return starts


def _frequencies(rotary, scaled):
    """Radians per position: the usual powers of 10000, or of 500000 with the slow ones eight times slower and a ramp between (for long contexts)."""
    theta = 500000.0 if scaled else 10000.0
    f = theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))
    if scaled:
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / 3).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    return f.float().cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["kind"] == "logits":
        rows, vocab, width = case["rows"], case["vocab"], case["width"]
        logits = (3 * normal(rows, vocab)).to(torch.float32 if case["dtype"] == "fp32" else BF16)
        state = dict(kind="logits", logits=logits, tokens=None, lengths=None, prompts=None, repetition=None, frequency=None, presence=None, bias=None, allowed=None)

        def per_row(low, high):
            return low + (high - low) * torch.rand(rows, device="cuda", generator=gen)

        if case["penalties"]:
            # text repeats itself: most tokens are among a few hundred
            state["tokens"] = (torch.rand(rows, width, device="cuda", generator=gen) ** 3 * vocab).long().clamp_(0, vocab - 1)
            state["lengths"] = torch.randint(width // 2, width + 1, (rows,), device="cuda", generator=gen, dtype=torch.int32)
            state["prompts"] = (state["lengths"] * torch.rand(rows, device="cuda", generator=gen)).int()
            state["repetition"], state["frequency"], state["presence"] = per_row(1.0, 1.5), per_row(0.0, 0.5), per_row(0.0, 0.5)
        if case["bias"] != "none":
            shape = (vocab,) if case["bias"] == "shared" else (rows, vocab)
            state["bias"] = normal(*shape) * (torch.rand(*shape, device="cuda", generator=gen) < 0.01)
        if case["mask"]:
            words = (vocab + 31) // 32
            state["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, words), device="cuda", generator=gen, dtype=torch.int64).int()
        return state

    new, past, page, dim = _numbers(case["new"]), _numbers(case["past"]), case["page"], case["dim"]
    starts = _starts(new)
    need = [(p + n + page - 1) // page for p, n in zip(past, new)]
    if case["kind"] == "append":
        # (only the pages that the new tokens reach are there: a sequence's earlier ones are another sequence's in this cache)
        held = sorted({(s, at // page) for s, (p, n) in enumerate(zip(past, new)) for at in (*range(p, p + n, page), p + n - 1)})
    else:
        held = [(s, j) for s in range(len(new)) for j in range(need[s])]
    order = torch.randperm(len(held) + 3, device="cuda", generator=gen)[:len(held)]
    table = torch.zeros(len(new), max(need), dtype=torch.int32)
    at = torch.tensor(held, dtype=torch.long)
    table[at[:, 0], at[:, 1]] = order.int().cpu()
    state = dict(kind=case["kind"], keys=normal(len(held) + 3, case["kv_heads"], page, dim).to(BF16), values=normal(len(held) + 3, case["kv_heads"], page, dim).to(BF16),
                 table=table.cuda(), starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), past=torch.tensor(past, dtype=torch.int32, device="cuda"),
                 spans=list(zip(starts, new, past)), most_new=max(new))
    if case["kind"] == "append":
        # one projection's rows: queries, keys and values side by side
        qkv = normal(starts[-1], case["heads"] + 2 * case["kv_heads"], dim).mul_(torch.exp(0.3 * normal(starts[-1], 1, 1))).to(BF16)
        state["q"], state["k"], state["v"] = qkv.split([case["heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        state["frequencies"] = _frequencies(case["rotary"], case["scaled"]) if case["rotary"] else None
        state["interleaved"], state["factor"] = case["interleaved"], 1.1 if case["scaled"] else 1.0
        state["q_norm"], state["k_norm"] = ((1 + 0.1 * normal(dim)).to(BF16) if case["norms"] else None for _ in range(2))
    else:
        state["q"] = (1.5 * normal(starts[-1], case["heads"], dim)).to(BF16)
        state["window"] = case["window"] or None
    return state


def run(state):
    if own:
        from tensor_parallel_b200.ops import functional as OF

        if state["kind"] == "logits":
            return OF.adjust_logits(state["logits"], state["tokens"], state["lengths"], state["prompts"], state["repetition"], state["frequency"],
                                    state["presence"], bias=state["bias"], allowed=state["allowed"])
        cache = OF.PagedCache(state["keys"], state["values"], state["table"])
        if state["kind"] == "append":
            rotary = None if state["frequencies"] is None else OF.Rotary(state["frequencies"], state["interleaved"], state["factor"])
            q = OF.paged_append(cache, state["q"], state["k"], state["v"], state["starts"], state["past"], rotary=rotary, q_norm=state["q_norm"],
                                k_norm=state["k_norm"], eps=EPS)
            return q, state["keys"], state["values"]
        return OF.paged_attention(state["q"], cache, state["starts"], state["past"], window=state["window"], most_new=state["most_new"])
    if state["kind"] == "logits":
        return _plain_logits(state)
    return _plain_append(state) if state["kind"] == "append" else _plain_attend(state)


# -- plain forms ---------------------------------------------------------------------------------


def _plain_rows(x, weight, positions, state):
    h = x.float()
    if weight is not None:
        h = h * torch.rsqrt((h * h).sum(-1, keepdim=True) / h.shape[-1] + EPS) * weight.float()
    f = state["frequencies"]
    if f is not None:
        turn = positions.double()[:, None] * f.double()  # (far positions: 32 bits hold their angles to a few hundredths)
        c, s = ((t(turn) * state["factor"]).float()[:, None] for t in (torch.cos, torch.sin))
        half = f.shape[0]
        h = h.clone()
        if state["interleaved"]:
            a, b = h[..., 0:2 * half:2].clone(), h[..., 1:2 * half:2].clone()
            h[..., 0:2 * half:2], h[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
        else:
            a, b = h[..., :half].clone(), h[..., half:2 * half].clone()
            h[..., :half], h[..., half:2 * half] = a * c - b * s, b * c + a * s
    return h.to(x.dtype)


def _plain_append(state):
    counts = state["starts"][1:] - state["starts"][:-1]
    tokens = state["q"].shape[0]
    of = torch.repeat_interleave(torch.arange(counts.shape[0], device="cuda"), counts, output_size=tokens)
    positions = state["past"][of] + torch.arange(tokens, device="cuda") - state["starts"][of]
    page = state["keys"].shape[2]
    pages, slots = state["table"][of, positions // page].long(), positions % page
    state["keys"][pages, :, slots] = _plain_rows(state["k"], state["k_norm"], positions, state)
    state["values"][pages, :, slots] = state["v"]
    return _plain_rows(state["q"], state["q_norm"], positions, state), state["keys"], state["values"]


def _plain_attend(state):
    q, keys = state["q"], state["keys"]
    heads, dim = q.shape[1:]
    kv_heads, page = keys.shape[1:3]
    out = torch.empty_like(q)
    for s, (start, new, past) in enumerate(state["spans"]):
        total = past + new
        first = max(0, past - state["window"] + 1) // page * page if state["window"] else 0
        pages = state["table"][s, first // page:(total + page - 1) // page].long()
        k, v = (t[pages].transpose(0, 1).reshape(kv_heads, -1, dim)[:, :total - first].float() for t in (keys, state["values"]))
        rows = q[start:start + new].float().view(new, kv_heads, heads // kv_heads, dim).permute(1, 2, 0, 3).reshape(kv_heads, -1, dim)
        scores = torch.matmul(rows, k.transpose(1, 2)).mul_(1 / math.sqrt(dim)).view(kv_heads, -1, new, total - first)
        at, key = torch.arange(past, total, device="cuda")[:, None], torch.arange(first, total, device="cuda")[None]
        hidden = key > at
        if state["window"]:
            hidden = hidden | (key <= at - state["window"])
        if new > 1 or state["window"]:
            scores = scores.masked_fill_(hidden, float("-inf"))
        scores = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        scores = scores.div_(scores.sum(-1, keepdim=True))
        o = torch.matmul(scores.view(kv_heads, -1, total - first), v)
        out[start:start + new] = o.view(kv_heads, -1, new, dim).permute(2, 0, 1, 3).reshape(new, heads, dim).to(q.dtype)
    return out


def _plain_logits(state):
    x = state["logits"].float()
    if state["tokens"] is not None:
        at = torch.arange(state["tokens"].shape[1], device="cuda")[None]
        there, said = at < state["lengths"][:, None], at >= state["prompts"][:, None]
        counts = torch.zeros_like(x)
        seen = torch.zeros_like(x).scatter_add_(1, state["tokens"], there.float())
        counts.scatter_add_(1, state["tokens"], (there & said).float())
        r = state["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - state["frequency"][:, None] * counts - state["presence"][:, None] * (counts > 0)
    if state["bias"] is not None:
        x = x + state["bias"]
    if state["allowed"] is not None:
        bits = state["allowed"][:, :, None] >> torch.arange(32, dtype=torch.int32, device="cuda") & 1
        x = x.masked_fill(bits.flatten(1)[:, :x.shape[1]] == 0, float("-inf"))
    return x.to(state["logits"].dtype)


# -- 64 bits -------------------------------------------------------------------------------------


def _exact_rows(x, weight, first, s):
    """Rows of one sequence, the first at position ``first``: complex products for the rotation."""
    h = x.double()
    if weight is not None:
        h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * weight.double()
    if s["frequencies"] is None:
        return h
    f = s["frequencies"].double()
    half = f.shape[0]
    turns = torch.polar(torch.full((len(h), half), float(s["factor"]), dtype=torch.float64, device="cuda"),
                        torch.outer(torch.arange(first, first + len(h), dtype=torch.float64, device="cuda"), f))
    part = h[..., :2 * half].unflatten(-1, (half, 2) if s["interleaved"] else (2, half))
    pairs = part if s["interleaved"] else part.transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turns[:, None])
    turned = (turned if s["interleaved"] else turned.transpose(-1, -2)).flatten(-2)
    return torch.cat((turned, h[..., 2 * half:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "logits":
        x = s["logits"].double()
        if s["tokens"] is not None:
            vocab = x.shape[1]
            for row in range(x.shape[0]):
                length, prompt = int(s["lengths"][row]), int(s["prompts"][row])
                history = s["tokens"][row, :length]
                r, f, p = (float(s[name][row]) for name in ("repetition", "frequency", "presence"))
                known = history.unique()
                x[row, known] = torch.where(x[row, known] > 0, x[row, known] / r, x[row, known] * r)
                said = torch.bincount(history[prompt:], minlength=vocab)
                x[row] -= f * said + p * (said > 0)
        if s["bias"] is not None:
            x = x + s["bias"].double()
        if s["allowed"] is not None:
            column = torch.arange(x.shape[1], device="cuda")
            open_ = (s["allowed"].long()[:, column // 32] >> (column % 32)) % 2 == 1
            x[~open_] = -math.inf
        return x
    page = case["page"]
    if s["kind"] == "append":
        keys, values = s["keys"].double(), s["values"].double()
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for i, (start, new, past) in enumerate(s["spans"]):
            rows = slice(start, start + new)
            out[rows] = _exact_rows(s["q"][rows], s["q_norm"], past, s)
            k, v = _exact_rows(s["k"][rows], s["k_norm"], past, s), s["v"][rows].double()
            for j in range(past // page, (past + new - 1) // page + 1):
                low, high = max(past, j * page), min(past + new, (j + 1) * page)
                into = int(s["table"][i, j])
                keys[into, :, low - j * page:high - j * page] = k[low - past:high - past].transpose(0, 1)
                values[into, :, low - j * page:high - j * page] = v[low - past:high - past].transpose(0, 1)
        return out, keys, values
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    for i, (start, new, past) in enumerate(s["spans"]):
        pages = s["table"][i, :(past + new + page - 1) // page].long()
        q = s["q"][start:start + new].double()
        for h in range(case["kv_heads"]):
            k, v = (s[name][pages, h].reshape(-1, case["dim"])[:past + new].double() for name in ("keys", "values"))
            scores = torch.einsum("tgd,jd->tgj", q[:, h * group:(h + 1) * group], k) / math.sqrt(case["dim"])
            far = torch.arange(past, past + new, device="cuda")[:, None] - torch.arange(past + new, device="cuda")[None]  # how far back a key lies
            seen = (far >= 0) & ((far < s["window"]) if s["window"] else True)
            out[start:start + new, h * group:(h + 1) * group] = torch.softmax(scores.masked_fill(~seen[:, None], -math.inf), -1) @ v
    return out


def work(case):
    if case["kind"] == "logits":
        n = case["rows"] * case["vocab"]
        moved = n * 2 * (4 if case["dtype"] == "fp32" else 2)
        if case["penalties"]:
            moved += case["rows"] * (8 * case["width"] * 3 // 4 + 20)  # (three quarters of the width, on average)
        if case["bias"] != "none":
            moved += 4 * (n if case["bias"] == "rows" else case["vocab"])
        if case["mask"]:
            moved += n // 8
        return {"bytes": moved, "flops": 6 * n}
    new, past, dim = _numbers(case["new"]), _numbers(case["past"]), case["dim"]
    tokens, heads, kv_heads = sum(new), case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        values = tokens * (heads + 2 * kv_heads) * dim
        turned = tokens * (heads + kv_heads)
        return {"bytes": 4 * values + 12 * len(new), "flops": turned * (3 * case["rotary"] + (4 * dim if case["norms"] else 0))}
    reach = case["window"] or 10 ** 9
    read = sum(min(p + n, reach + n - 1) for n, p in zip(new, past))
    pairs = sum(min(p + i + 1, reach) for n, p in zip(new, past) for i in range(n))
    return {"bytes": 4 * tokens * heads * dim + 4 * read * kv_heads * dim, "flops": 4 * dim * heads * pairs}
