"""Ragged batches over paged caches for the tests, and what their operators come to in 64 bits, token by token."""
import math

import torch

BF16 = torch.bfloat16


def numbers(gen, *shape, dtype=BF16, scale=1.0):
    return (torch.randn(*shape, generator=gen, dtype=torch.float32) * scale).to(dtype)


def batch(new, past, heads, kv_heads, dim, page, dtype=BF16, device="cpu", seed=0, spare=3, rest=0, front=0, junk=float("nan"), width=None, unused=-7, only_new=False):
    """A batch in which every slot that belongs to no sequence holds ``junk`` and every table entry beyond a sequence's pages ``unused``; ``front`` and ``rest`` rows of the
    queries are in front of the first sequence and behind the last.  ``only_new``: one page stands for all that no new token reaches."""
    gen = torch.Generator().manual_seed(seed)
    n = len(new)
    need = [-(-(p + m) // page) for p, m in zip(past, new)]
    begin = [min(p // page, j) if only_new else 0 for p, j in zip(past, need)]
    pages = sum(need) - sum(begin) + spare
    order = torch.randperm(pages, generator=gen)
    table = torch.full((n, width or max([1, *need])), unused, dtype=torch.int32)
    keys = torch.full((pages, kv_heads, page, dim), junk, dtype=dtype)
    values = torch.full((pages, kv_heads, page, dim), junk, dtype=dtype)
    at = 0
    for s in range(n):
        table[s, :begin[s]] = order[-1]
        table[s, begin[s]:need[s]] = order[at:at + need[s] - begin[s]].int()
        at += need[s] - begin[s]
        for j in range(begin[s], need[s]):
            held = min(page, past[s] + new[s] - j * page)
            keys[table[s, j], :, :held] = numbers(gen, kv_heads, held, dim, dtype=dtype)
            values[table[s, j], :, :held] = numbers(gen, kv_heads, held, dim, dtype=dtype)
    starts = [front]
    for m in new:
        starts.append(starts[-1] + m)
    tokens = starts[-1] + rest
    q = numbers(gen, tokens, heads, dim, dtype=dtype, scale=1.5)
    k, v = (numbers(gen, tokens, kv_heads, dim, dtype=dtype) for _ in range(2))
    made = dict(keys=keys, values=values, table=table, starts=torch.tensor(starts, dtype=torch.int32), past=torch.tensor(past, dtype=torch.int32), q=q, k=k, v=v)
    return {name: t.to(device) for name, t in made.items()}


def sequence(b, s, name):
    """Keys or values of a whole sequence, ``[tokens, kv_heads, dim]`` in 64 bits."""
    page = b["keys"].shape[2]
    total = int(b["past"][s]) + int(b["starts"][s + 1]) - int(b["starts"][s])
    pages = b["table"][s, :-(-total // page)].long()
    return b[name][pages].double().transpose(1, 2).flatten(0, 1)[:total]


def attention64(b, scale=None, window=None):
    """``(out, tolerance)``, zeros in rows outside all sequences.  The tolerance counts the roundings: a probability to bf16 (2^-8 of it, so 2^-8 of sum p |v|), the result to
    bf16 (2^-8), and the score's in 32 bits (head_dim + 4 of 2^-24 of sum |q k|, twice in the exponent of p: its own and the row's)."""
    q = b["q"].double()
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    heads, dim = q.shape[1:]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    for s in range(len(b["past"])):
        start, end, past = int(b["starts"][s]), int(b["starts"][s + 1]), int(b["past"][s])
        if end == start:
            continue
        k, v = (sequence(b, s, name).repeat_interleave(heads // b["keys"].shape[1], 1) for name in ("keys", "values"))
        rows = q[start:end]
        scores = torch.einsum("thd,jhd->htj", rows, k) * scale
        size = torch.einsum("thd,jhd->htj", rows.abs(), k.abs()).amax(-1) * scale
        far = torch.arange(past, past + end - start, device=q.device)[:, None] - torch.arange(len(k), device=q.device)[None]
        p = torch.softmax(scores.masked_fill((far < 0) | (far >= (window or 1 << 40)), -math.inf), -1)
        o, a = torch.einsum("htj,jhd->thd", p, v), torch.einsum("htj,jhd->thd", p, v.abs())
        out[start:end] = o
        slack = 2 * (dim + 4) * 2.0 ** -24 * size.t()[..., None] + len(k) * 2.0 ** -24
        half = 2.0 ** -8 if b["q"].dtype == BF16 else 2.0 ** -24
        tol[start:end] = (half + slack) * a * 1.02 + half * o.abs() * 1.02 + 1e-30
    return out, tol


def turned64(x, weight, eps, positions, rotary):
    """``(rows, tolerance)`` of ``[tokens, heads, dim]`` normed and rotated: a rounding to the type, and 2^-20 of the pair's size for those in 32 bits."""
    h = x.double()
    if weight is not None:
        h = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double()
    y, size = h.clone(), h.abs()
    if rotary is not None:
        f, interleaved, factor = rotary
        half = len(f)
        angle = positions.double()[:, None] * f.double()[None]
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            c, s = torch.cos(angle[:, i])[:, None] * factor, torch.sin(angle[:, i])[:, None] * factor
            y[..., a], y[..., b] = h[..., a] * c - h[..., b] * s, h[..., b] * c + h[..., a] * s
            size[..., a] = size[..., b] = (h[..., a].abs() + h[..., b].abs()) * factor
    half_step = 2.0 ** -8 if x.dtype == BF16 else 2.0 ** -24
    return y, half_step * 1.01 * y.abs() + 2.0 ** -20 * size + 1e-38


def append64(b, rotary=None, q_norm=None, k_norm=None, eps=1e-6):
    """``(queries, their tolerance, [(page, slot, key row, its tolerance, value row)])``."""
    q, tq = torch.zeros(b["q"].shape, dtype=torch.float64, device=b["q"].device), torch.zeros(b["q"].shape, dtype=torch.float64, device=b["q"].device)
    stored, page = [], b["keys"].shape[2]
    for s in range(len(b["past"])):
        start, end, past = int(b["starts"][s]), int(b["starts"][s + 1]), int(b["past"][s])
        if end == start:
            continue
        at = torch.arange(past, past + end - start, device=b["q"].device)
        q[start:end], tq[start:end] = turned64(b["q"][start:end], q_norm, eps, at, rotary)
        k, tk = turned64(b["k"][start:end], k_norm, eps, at, rotary)
        for i in range(end - start):
            stored.append((int(b["table"][s, (past + i) // page]), (past + i) % page, k[i], tk[i], b["v"][start + i]))
    return q, tq, stored


def within(got, want, tol, what=""):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {got[bad][0].item()} for {want[bad][0].item()} +- {tol[bad][0].item():.3g}"


def check_append(b, got_q, before, rotary=None, q_norm=None, k_norm=None, eps=1e-6):
    """``got_q`` and the cache in ``b`` against 64 bits; ``before``: copies of keys and values from before the call, whose other slots have to be as they were."""
    q, tq, stored = append64(b, rotary, q_norm, k_norm, eps)
    within(got_q, q, tq, "queries")
    keys, values = (t.clone() for t in before)
    for page, slot, k, tk, v in stored:
        within(b["keys"][page, :, slot], k, tk, "keys")
        assert torch.equal(b["values"][page, :, slot], v)
        keys[page, :, slot], values[page, :, slot] = b["keys"][page, :, slot], v
    for now, want in ((b["keys"], keys), (b["values"], values)):
        assert torch.equal(now.contiguous().view(torch.int8), want.contiguous().view(torch.int8))


def logits64(logits, tokens=None, lengths=None, prompts=None, repetition=None, frequency=None, presence=None, bias=None, allowed=None):
    x = logits.double().clone()
    rows, vocab = x.shape
    pick = lambda t, r, neutral: neutral if t is None else float(t[r]) if isinstance(t, torch.Tensor) else float(t)
    for r in range(rows):
        if tokens is not None:
            length = tokens.shape[1] if lengths is None else min(max(int(lengths[r]), 0), tokens.shape[1])
            prompt = 0 if prompts is None else max(int(prompts[r]), 0)
            said = {}
            for i, t in enumerate(tokens[r, :length].tolist()):
                if 0 <= t < vocab:
                    said[t] = said.get(t, 0) + (i >= prompt)
            for t, count in said.items():
                v, rep = x[r, t], pick(repetition, r, 1.0)
                v = v / rep if v > 0 else v * rep
                x[r, t] = v - (pick(frequency, r, 0.0) * count + pick(presence, r, 0.0)) if count else v
        if bias is not None:
            x[r] += (bias if bias.ndim == 1 else bias[r]).double()
        if allowed is not None:
            words = allowed if allowed.ndim == 1 else allowed[r]
            bits = [int(words[t]) >> i & 1 for t in range(len(words)) for i in range(32)][:vocab]
            x[r, torch.tensor(bits) == 0] = -math.inf
    return x


def check_logits(got, args):
    want = logits64(*args)
    assert got.dtype == args[0].dtype and got.shape == want.shape
    # a rounding to the type of a result, and four in 32 bits of what goes into it (logit, penalties and bias below 2^7 here)
    tol = (2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24) * want.abs().nan_to_num(posinf=0.0) * 1.01 + 4 * 2.0 ** -24 * 2 ** 7
    same = (got.double() == want) | (got.isnan() & want.isnan())
    assert (same | ((got.double() - want).abs() <= tol)).all()
    assert torch.equal(got.isinf(), want.isinf())
