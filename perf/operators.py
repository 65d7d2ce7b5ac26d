"""Operators of 8-bit serving: what they are measured on.

Three operators make up a decoder layer with 8-bit integer weights and activations (W8A8): the RMSNorm in front of a projection with the
residual's addition and its result in 8 bits, the rows of an activation (or of a weight) in 8 bits, and the matrix product of 8-bit
integers with a scale per token and per output channel.  Widths are those of the model configurations in ``tensor_parallel_b200/models``
(7B: 4096 / 11008, 13B: 5120), batch sizes and lengths those of the benchmark (8 x 2048) and of ragged prompts.

The 8-bit results are whole numbers, which the matrix product takes as they are; they are returned as those numbers, next to the scales.  They are
exact: ``v * (127 / max |v|)`` has two roundings in 32 bits, and the statistics of an RMSNorm are common to a row and cancel out of it.

``exact`` restates every operator in 64-bit PyTorch, with none of this package's code.
"""
import math

import torch

own = False

BF16 = torch.bfloat16
EPS = 1e-5
LEAST = 1e-30  # least maximum of a row: a row of zeros has a scale too


def listed():
    return [
        # the norm of a decode step of one sequence: all latency
        dict(name="norm_token", kind="norm", rows=1, cols=4096, dtype="bf16", residual=False),
        # the norm of a prompt pass, 4 x 2048 tokens, with the sum of the ranks' partial results added
        dict(name="norm_prompt", kind="norm", rows=8192, cols=4096, dtype="bf16", residual=True),
        # a residual stream in 32 bits, 13B width, an odd number of rows
        dict(name="norm_wide_stream", kind="norm", rows=1999, cols=5120, dtype="fp32", residual=True),
        # MLP activations of a decode step, batch 8
        dict(name="rows_decode", kind="rows", rows=8, cols=11008, dtype="bf16"),
        # MLP activations of a prompt pass
        dict(name="rows_prompt", kind="rows", rows=8192, cols=11008, dtype="bf16"),
        # rows of an odd width: no row but the first starts on a vector's boundary
        dict(name="rows_odd", kind="rows", rows=1999, cols=2731, dtype="bf16"),
        # output projection of one sequence's decode step
        dict(name="product_token", kind="product", tokens=1, features=4096, k=4096, act="none", bias=False, residual=True),
        # gate and up projection of a decode step, batch 8
        dict(name="product_decode", kind="product", tokens=8, features=22016, k=4096, act="swiglu16", bias=False, residual=False),
        # down projection of a short prompt
        dict(name="product_short", kind="product", tokens=100, features=4096, k=11008, act="none", bias=False, residual=True),
        # odd sizes on every side, with bias and activation
        dict(name="product_odd", kind="product", tokens=257, features=2999, k=1001, act="gelu", bias=True, residual=False),
        # q, k and v of a ragged prompt pass, 4 x 1000 tokens
        dict(name="product_prompt", kind="product", tokens=4000, features=12288, k=4096, act="none", bias=True, residual=False),
        # gate and up projection of a prompt pass, 4 x 2048 tokens
        dict(name="product_gated", kind="product", tokens=8192, features=22016, k=4096, act="swiglu16", bias=False, residual=False),
    ]


def _spread(rng, low, high, step=1):
    """A whole number in [low, high], even over the logarithm, a multiple of ``step``."""
    value = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(value / step)) * step))


def draw(rng):
    kind = rng.choice(["norm", "rows", "product", "product", "product"])
    if kind != "product":
        cols = _spread(rng, 64, 20480, rng.choice([1, 8, 64]))
        rows = _spread(rng, 1, min(8192, 8192 * 11008 // cols))
        case = dict(kind=kind, rows=rows, cols=cols, dtype=rng.choice(["bf16", "bf16", "fp32"]))
        if kind == "norm":
            case["residual"] = rng.random() < 0.5
        return case
    tokens = _spread(rng, 1, rng.choice([64, 512, 8192]))
    k = _spread(rng, 64, 16384, rng.choice([1, 8, 64]))
    act = rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu", "swiglu16"])
    features = _spread(rng, 64, min(32768, 8192 * 22016 * 4096 // (tokens * k)), 32 if act == "swiglu16" else rng.choice([1, 8, 64]))
    return dict(kind=kind, tokens=tokens, features=features, k=k, act=act, bias=rng.random() < 0.5, residual=act != "swiglu16" and rng.random() < 0.5)


def _type(case):
    return torch.float32 if case["dtype"] == "fp32" else BF16


def _activations(gen, rows, cols, dtype):
    """Hidden states: about normal, every row of its own magnitude, and a few channels that are much larger than the others."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    channel = 1 + 19 * (torch.rand(cols, device="cuda", generator=gen) < 0.005)
    row = torch.exp(0.5 * torch.randn(rows, 1, device="cuda", generator=gen))
    return x.mul_(channel).mul_(row).to(dtype)


def _eight_bits(x):
    """(whole numbers, scales) of the rows of ``x``, which lie a multiple of 16 bytes apart as in the framework."""
    rows, cols = x.shape
    most = x.abs().amax(1, keepdim=True)
    q = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device="cuda")[:, :cols]
    q.copy_(torch.round(x * (127 / most)))
    return q, (most[:, 0] / 127).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["kind"] != "product":
        dtype = _type(case)
        state = dict(kind=case["kind"], x=_activations(gen, case["rows"], case["cols"], dtype))
        if case["kind"] == "norm":
            state["weight"] = (1 + 0.1 * torch.randn(case["cols"], device="cuda", generator=gen)).to(dtype)
            state["residual"] = _activations(gen, case["rows"], case["cols"], dtype) if case["residual"] else None
        return state
    tokens, features, k = case["tokens"], case["features"], case["k"]
    x, sx = _eight_bits(_activations(gen, tokens, k, torch.float32))
    w, sw = _eight_bits(torch.randn(features, k, device="cuda", generator=gen) / math.sqrt(k))
    cols = features // 2 if case["act"] == "swiglu16" else features
    return dict(
        kind="product", x=x, sx=sx, w=w, sw=sw, act=None if case["act"] == "none" else case["act"],
        bias=(0.1 * torch.randn(features, device="cuda", generator=gen)).to(BF16) if case["bias"] else None,
        residual=torch.randn(tokens, cols, device="cuda", generator=gen).to(BF16) if case["residual"] else None)


def run(state):
    if own:
        from tensor_parallel_b200.ops import functional as OF

        if state["kind"] == "rows":
            return tuple(OF.quantize_int8(state["x"]))
        if state["kind"] == "norm":
            rows, summed = OF.rms_norm_int8(state["x"], state["weight"], EPS, residual=state["residual"])
            return (*rows, summed)
        return OF.linear_int8(OF.Int8Rows(state["x"], state["sx"]), OF.Int8Rows(state["w"], state["sw"]), state["bias"], act=state["act"],
                              residual=state["residual"])
    if state["kind"] == "rows":
        return _plain_rows(state["x"].float())
    if state["kind"] == "norm":
        return _plain_norm(state["x"], state["weight"], state["residual"])
    return _plain_product(state)


# -- plain forms ---------------------------------------------------------------------------------


def _plain_rows(v, factor=None):
    most = v.abs().amax(1, keepdim=True).clamp_min(LEAST)
    q = torch.round(v * (torch.full_like(most, 127.0) / most)).to(torch.int8)
    scale = most[:, 0] / 127
    return q, scale if factor is None else scale * factor


def _plain_norm(x, weight, residual):
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).sum(1) / hf.shape[1] + EPS)
    return (*_plain_rows(hf * weight.float(), rstd), h)


def _plain_act(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "swiglu16":  # 16 gate columns, then their 16 up columns
        pairs = v.view(v.shape[0], -1, 2, 16)
        gate, up = pairs[:, :, 0], pairs[:, :, 1]
        return (gate / (1 + torch.exp(-gate)) * up).reshape(v.shape[0], -1)
    return v


def _plain_product(state):
    # (the products are whole numbers; sums of more than 2^24 lose their last bits in 32, far below the rounding of the result)
    v = torch.matmul(state["x"].float(), state["w"].float().t())
    v = v * state["sx"][:, None] * state["sw"][None, :]
    if state["bias"] is not None:
        v = v + state["bias"].float()
    v = _plain_act(v, state["act"])
    if state["residual"] is not None:
        v = v + state["residual"].float()
    return v.to(BF16)


# -- 64 bits -------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "product":
        out = torch.empty(s["x"].shape[0], s["w"].shape[0], dtype=torch.float64, device="cuda")
        w = s["w"].double()
        for at in range(0, out.shape[0], 2048):  # (a part of the tokens at a time, for their memory)
            out[at:at + 2048] = torch.einsum("tk,fk->tf", s["x"][at:at + 2048].double(), w)
        del w
        out.mul_(s["sw"].double()).mul_(s["sx"].double()[:, None])
        if s["bias"] is not None:
            out.add_(s["bias"].double())
        act = s["act"]
        if act == "swiglu16":
            halves = out.unflatten(1, (-1, 32))
            out = (halves[..., :16] * torch.sigmoid(halves[..., :16]) * halves[..., 16:]).flatten(1)
        elif act == "silu":
            out = out * torch.sigmoid(out)
        elif act == "relu":
            out = torch.relu(out)
        elif act is not None:
            out = torch.nn.functional.gelu(out, approximate="tanh" if act == "gelu_tanh" else "none")
        return out if s["residual"] is None else out + s["residual"].double()
    x = s["x"]
    if s["kind"] == "norm":
        # the sum is held in the type of its parts, and the norm is taken of what is held
        h = x if s["residual"] is None else (x.double() + s["residual"].double()).to(x.dtype)
        hd = h.double()
        v, rms = hd * s["weight"].double(), torch.sqrt(hd.square().mean(1) + EPS)
    else:
        v, rms = x.double(), torch.ones(x.shape[0], dtype=torch.float64, device="cuda")
    most = v.abs().max(1).values.clamp(min=LEAST)
    rows = (torch.round(v / most[:, None] * 127).to(torch.int8), most / rms / 127)
    return rows if s["kind"] == "rows" else (*rows, h.double())


def work(case):
    if case["kind"] == "product":
        t, f, k = case["tokens"], case["features"], case["k"]
        cols = f // 2 if case["act"] == "swiglu16" else f
        moved = t * k + f * k + 4 * t + 4 * f + 2 * t * cols * (2 if case["residual"] else 1) + (2 * f if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * t * f * k}
    n, size = case["rows"] * case["cols"], 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "rows":
        return {"bytes": n * (size + 1) + 4 * case["rows"], "flops": 4 * n}
    # with a residual both are read, and their sum is written
    return {"bytes": n * (size * (3 if case["residual"] else 1) + 1) + 4 * case["rows"] + size * case["cols"], "flops": 7 * n}
