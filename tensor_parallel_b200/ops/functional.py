"""Operator front-end used by the self-contained models.

Every operator has a plain PyTorch definition (the numerical reference, and the CPU path) and,
for CUDA tensors, a hand-written sm_100a kernel from ``tensor_parallel_b200.ops.native``.
Dispatch rule: CUDA bf16/fp16/fp32 tensors go to the native kernel when the shape is
supported; if the native library cannot be loaded on a CUDA machine the call raises, unless
``TENSOR_PARALLEL_USE_NATIVE`` asks for stock PyTorch operators.
"""
from __future__ import annotations

import math
import os
from typing import NamedTuple, Optional, Tuple

import torch
import torch.nn.functional as F

_FORCE_TORCH = bool(os.environ.get("TENSOR_PARALLEL_USE_NATIVE"))
_native_module = None


def _native(x: torch.Tensor):
    """The native module if ``x`` should run on hand-written kernels, else ``None``: on other devices, and where operators are being captured (``make_fx``,
    fake tensors), since a kernel leaves nothing in the graph."""
    global _native_module
    if not x.is_cuda or _FORCE_TORCH:
        return None
    if _native_module is None:  # (an import statement per call costs as much as all other checks)
        from tensor_parallel_b200.ops import native  # raises if the library is missing on a GPU box

        _native_module = native
    return _native_module if _compiling() or not _native_module.captured() else None


# -- reference definitions ---------------------------------------------------------------------


def rms_norm_ref(x, weight, eps: float):
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return (y * weight.float()).to(x.dtype) if weight is not None else y.to(x.dtype)


def layer_norm_ref(x, weight, bias, eps: float):
    return F.layer_norm(x.float(), x.shape[-1:], None if weight is None else weight.float(), None if bias is None else bias.float(), eps).to(x.dtype)


def rope_tables(positions: torch.Tensor, rotary_dim: int, theta: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos / sin of shape ``[..., rotary_dim/2]`` in fp32 for integer ``positions``."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, rotary_dim, 2, device=positions.device, dtype=torch.float32) / rotary_dim))
    angles = positions.to(torch.float32)[..., None] * inv_freq
    return angles.cos(), angles.sin()


def apply_rope_ref(x, positions, theta: float, rotary_dim: Optional[int] = None, interleaved: bool = False):
    """Rotary embedding on ``x[B, S, H, D]`` with ``positions[B, S]``.  ``interleaved`` pairs
    ``(2i, 2i+1)`` (GPT-J / CodeGen); otherwise ``(i, i + rotary_dim/2)`` (Llama / NeoX / Falcon)."""
    d = x.shape[-1]
    rotary_dim = d if rotary_dim is None else rotary_dim
    cos, sin = rope_tables(positions, rotary_dim, theta)
    cos, sin = cos[:, :, None, :], sin[:, :, None, :]
    rot, keep = x[..., :rotary_dim].float(), x[..., rotary_dim:]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = rot[..., : rotary_dim // 2], rot[..., rotary_dim // 2 :]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((out.to(x.dtype), keep), dim=-1)


def attention_ref(q, k, v, causal: bool, bias=None, scale: Optional[float] = None):
    """``q[B,Sq,Hq,D]``, ``k/v[B,Sk,Hkv,D]`` -> ``[B,Sq,Hq,D]``.  With ``causal`` query *i* sees keys
    ``<= i + (Sk - Sq)`` (so a cached decode step sees the whole cache).  ``bias`` is added to the
    scores and broadcasts against ``[B,Hq,Sq,Sk]``.  Softmax in fp32."""
    b, sq, hq, d = q.shape
    sk, hkv = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    qf = q.float().permute(0, 2, 1, 3)
    kf = k.float().permute(0, 2, 1, 3)
    vf = v.float().permute(0, 2, 1, 3)
    if hkv != hq:
        kf = kf.repeat_interleave(hq // hkv, dim=1)
        vf = vf.repeat_interleave(hq // hkv, dim=1)
    scores = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    if bias is not None:
        scores = scores + bias.float()
    if causal:
        i = torch.arange(sq, device=q.device)[:, None] + (sk - sq)
        j = torch.arange(sk, device=q.device)[None, :]
        scores = scores.masked_fill(j > i, float("-inf"))
    probs = torch.softmax(scores, dim=-1)
    return torch.matmul(probs, vf).permute(0, 2, 1, 3).to(q.dtype)


def gelu_ref(x, approximate: str = "none"):
    return F.gelu(x, approximate=approximate)


def swiglu_ref(gate, up):
    return F.silu(gate) * up


def geglu_ref(gate, up, approximate: str = "tanh"):
    return F.gelu(gate, approximate=approximate) * up


def relative_bias_ref(embedding, buckets, queries: int, keys: int):
    i = torch.arange(queries, device=buckets.device)[:, None]
    j = torch.arange(keys, device=buckets.device)[None, :]
    return embedding(buckets[j - i + queries - 1]).permute(2, 0, 1)[None]


def relative_bias_table_grad_ref(grad, buckets, rows: int):
    """Gradient of a ``[rows, heads]`` table from that of its bias, ``[1, heads, queries, keys]``; differentiable itself."""
    heads, queries, keys = grad.shape[1:]
    i = torch.arange(queries, device=buckets.device)[:, None]
    j = torch.arange(keys, device=buckets.device)[None, :]
    pairs = grad[0].permute(1, 2, 0).reshape(queries * keys, heads).float()
    return torch.zeros(rows, heads, dtype=torch.float32, device=grad.device).index_add(0, buckets[j - i + queries - 1].reshape(-1), pairs)


class Int8Rows(NamedTuple):
    """Rows in 8-bit integers with a scale each: ``values`` int8 ``[..., cols]``, ``scales`` fp32 ``[...]``; row ``r`` stands for
    ``values[r] * scales[r]``.  An activation has a row per token, a weight a row per output channel.  Rows made here lie a multiple of 16 bytes apart,
    as the matrix product reads them; what lies between is not written."""

    values: torch.Tensor
    scales: torch.Tensor

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return (self.values.float() * self.scales[..., None]).to(dtype)


INT8_LEAST = 1e-30  # least maximum of a row, so that a row of zeros has a finite factor
INT8_MAX_K = 131071  # longest contraction whose sum stays below 2^31 whatever the integers are


def _int8_rows_ref(v: torch.Tensor, factor: Optional[torch.Tensor] = None) -> Int8Rows:
    most = v.abs().amax(-1, keepdim=True).clamp_min(INT8_LEAST)
    full = torch.full_like(most, 127.0)  # (with a plain number, PyTorch multiplies by a rounded reciprocal)
    values = torch.round(v * (full / most))
    scales = (most / full)[..., 0]
    finite = torch.isfinite(most)
    scales = torch.where(finite[..., 0], scales if factor is None else scales * factor, torch.full_like(scales, float("nan")))
    return Int8Rows(torch.where(finite, values, torch.zeros_like(values)).to(torch.int8), scales)


def quantize_int8_ref(x) -> Int8Rows:
    return _int8_rows_ref(x.float())


def _add_ref(x, residual):
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def _in_range(rstd):
    """NaN for the 1 / deviation of a row whose sum of squares passes the range of fp32 (a value above 2^64 is enough), which would come out as zero."""
    return torch.where(rstd > 0, rstd, torch.full_like(rstd, float("nan")))


def rms_norm_int8_ref(x, weight, eps: float, residual=None) -> Tuple[Int8Rows, torch.Tensor]:
    h = _add_ref(x, residual)
    hf = h.float()
    rstd = _in_range(torch.rsqrt(hf.pow(2).mean(-1) + eps))
    return _int8_rows_ref(hf if weight is None else hf * weight.to(x.dtype).float(), rstd), h


def layer_norm_int8_ref(x, weight, bias, eps: float, residual=None) -> Tuple[Int8Rows, torch.Tensor]:
    h = _add_ref(x, residual)
    hf = h.float()
    w, b = (None if t is None else t.to(x.dtype).float() for t in (weight, bias))
    values, scales = _int8_rows_ref(F.layer_norm(hf, h.shape[-1:], w, b, eps))
    rstd = torch.rsqrt((hf - hf.mean(-1, keepdim=True)).pow(2).mean(-1) + eps)
    return Int8Rows(values, torch.where(_in_range(rstd).isnan(), rstd.new_full((), float("nan")), scales)), h


def linear_int8_ref(x: Int8Rows, weight: Int8Rows, bias=None, act: Optional[str] = None, residual=None):
    # (64 bits hold the sums of products exactly)
    v = torch.matmul(x.values.double(), weight.values.double().t()).float() * x.scales[..., None] * weight.scales
    if bias is not None:
        v = v + bias.float()
    if act == "swiglu16":
        pairs = v.unflatten(-1, (-1, 2, 16))
        v = (F.silu(pairs[..., 0, :]) * pairs[..., 1, :]).flatten(-2)
    elif act is not None:
        v = {"relu": F.relu, "silu": F.silu, "gelu": F.gelu, "gelu_tanh": lambda t: F.gelu(t, approximate="tanh")}[act](v)
    if residual is not None:
        v = v + residual.float()
    return v.to(torch.bfloat16)


class PagedCache(NamedTuple):
    """Keys and values of sequences of different lengths, ``[pages, kv_heads, page_size, head_dim]`` each, and the pages of every sequence, int32
    ``[sequences, most pages of one]``: key ``j`` of sequence ``s`` is slot ``j % page_size`` of page ``table[s, j // page_size]``.  Pages may be in any order and
    belong to several sequences (a common prefix); entries beyond a sequence's keys are not read.  Keys and values may be strided views (the layers
    of one tensor, keys and values side by side, heads inside of slots)."""

    keys: torch.Tensor
    values: torch.Tensor
    table: torch.Tensor


class Rotary(NamedTuple):
    """A position rotation: the pairs of the first ``2 * len(frequencies)`` elements of a head are turned by ``position * frequencies[i]`` radians and multiplied
    by ``factor``.  Pairs are ``(2i, 2i + 1)`` if ``interleaved`` (GPT-J / CodeGen), else ``(i, i + len(frequencies))`` (Llama / NeoX / Falcon)."""

    frequencies: torch.Tensor  # fp32 [rotary_dim / 2]
    interleaved: bool = False
    factor: float = 1.0


# What a dictionary of scaled frequencies may name, by its kind.
_SCALING_KEYS = {"default": (), "linear": ("factor",), "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_max_position_embeddings"),
                 "yarn": ("factor", "original_max_position_embeddings", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim")}


def rotary(rotary_dim: int, theta: float = 10000.0, interleaved: bool = False, scaling: Optional[dict] = None, device=None) -> Rotary:
    """The usual frequencies ``theta ** (-2i / rotary_dim)``, for contexts longer than a model was trained on scaled as ``scaling`` says (the dictionary of
    a Hugging Face configuration): ``"linear"`` (all slower by ``factor``), ``"llama3"`` (slow ones slower by ``factor``, a ramp between) or ``"yarn"`` (a ramp over the
    pairs, from whole pairs unless ``truncate`` is false, and a factor on cosine and sine: ``attention_factor``, or by ``mscale`` and ``mscale_all_dim`` where both
    are there).  A ``rope_theta`` in it has to be ``theta``, a ``partial_rotary_factor`` is what ``rotary_dim`` says already and ``finetuned`` changes no number; what else it names is refused."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"a rotation takes an even number of elements, got {rotary_dim}")
    f = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    kind, factor = "default", 1.0
    if scaling:
        kind = scaling.get("rope_type", scaling.get("type", "default"))
        if kind not in _SCALING_KEYS:
            raise ValueError(f"scaling of rotary frequencies: 'linear', 'llama3' or 'yarn', got {kind!r}")
        strange = sorted(set(scaling) - {"rope_type", "type", "rope_theta", "partial_rotary_factor", "finetuned", *_SCALING_KEYS[kind]})
        if strange:
            raise ValueError(f"scaling of rotary frequencies: {kind!r} does not know {', '.join(map(repr, strange))}")
        if scaling.get("rope_theta") not in (None, theta):
            raise ValueError(f"scaling of rotary frequencies: it says rope_theta={scaling['rope_theta']}, theta is {theta}")
    if kind == "linear":
        f = f / scaling["factor"]
    elif kind == "llama3":
        low, high = scaling["low_freq_factor"], scaling["high_freq_factor"]
        turns = scaling["original_max_position_embeddings"] * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        f = f * keep + f / scaling["factor"] * (1 - keep)
    elif kind == "yarn":
        by = scaling["factor"]

        def pair(turns):  # the pair that makes so many turns over the original context
            return rotary_dim * math.log(scaling["original_max_position_embeddings"] / (turns * 2 * math.pi)) / (2 * math.log(theta))

        def temperature(weight):
            return 0.1 * weight * math.log(by) + 1.0 if by > 1 else 1.0

        low, high = pair(scaling.get("beta_fast") or 32), pair(scaling.get("beta_slow") or 1)
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        slow = ((torch.arange(rotary_dim // 2, dtype=torch.float64) - low) / (high - low if high != low else 0.001)).clamp(0, 1)
        f = f * (1 - slow) + f / by * slow
        factor = scaling.get("attention_factor")
        if factor is None:
            whole, part = scaling.get("mscale"), scaling.get("mscale_all_dim")
            factor = temperature(whole) / temperature(part) if whole and part else temperature(1.0)
    return Rotary(f.float().to(device), interleaved, float(factor))


def _spans(what: str, cache: PagedCache, tokens: int, starts, past, most_new: Optional[int] = None):
    """``(start, new, past)`` of every sequence, from the device; what the kernels answer with NaN and a status is an error here."""
    bounds, cached = starts.tolist(), past.tolist()
    room = cache.table.shape[1] * cache.keys.shape[2]
    spans = []
    for s, p in enumerate(cached):
        a, e = bounds[s], bounds[s + 1]
        if not 0 <= a <= e <= tokens or p < 0 or (e > a and p + e - a > room) or (most_new is not None and e - a > most_new):
            raise ValueError(f"{what}: sequence {s} has rows {a} to {e} of {tokens} behind {p} cached keys; its table has room for {room}"
                             + ("" if most_new is None else f", most_new is {most_new}"))
        spans.append((a, e - a, p))
    return spans


def _pages_of(what: str, cache: PagedCache, s: int, first: int, last: int):
    pages = cache.table[s, first:last + 1].long()
    if pages.numel() and not 0 <= int(pages.min()) <= int(pages.max()) < cache.keys.shape[0]:
        raise ValueError(f"{what}: pages {pages.tolist()} of sequence {s} are not all among the {cache.keys.shape[0]} of the cache")
    return pages


def _normed_and_turned(x, weight, eps: float, positions, turn: Optional[Rotary]):
    h = x.float()
    if weight is not None:
        h = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + eps) * weight.float()
    if turn is not None:
        half = turn.frequencies.shape[0]
        angles = positions.double()[:, None] * turn.frequencies.double()  # (in 32 bits, far positions are off by hundredths of a radian)
        c, s = ((fn(angles) * turn.factor).float()[:, None] for fn in (torch.cos, torch.sin))
        rot, keep = h[..., :2 * half], h[..., 2 * half:]
        if turn.interleaved:
            a, b = rot[..., 0::2], rot[..., 1::2]
            rot = torch.stack((a * c - b * s, b * c + a * s), dim=-1).flatten(-2)
        else:
            a, b = rot[..., :half], rot[..., half:]
            rot = torch.cat((a * c - b * s, b * c + a * s), dim=-1)
        h = torch.cat((rot, keep), dim=-1)
    return h.to(x.dtype)


def paged_append_ref(cache: PagedCache, q, k, v, starts, past, rotary=None, q_norm=None, k_norm=None, eps: float = 1e-6, out=None):
    spans = _spans("paged_append", cache, k.shape[0], starts, past)
    page = cache.keys.shape[2]
    places = [_pages_of("paged_append", cache, s, p // page, (p + new - 1) // page) if new else None for s, (_, new, p) in enumerate(spans)]
    given = out
    if q is not None and (rotary is not None or q_norm is not None or out is not None):
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device) if out is None else out
    for (start, new, p), pages in zip(spans, places):
        if not new:
            continue
        at = torch.arange(p, p + new, device=k.device)
        rows = slice(start, start + new)
        into = pages[at // page - p // page]
        cache.keys[into, :, at % page] = _normed_and_turned(k[rows], k_norm, eps, at, rotary)
        cache.values[into, :, at % page] = v[rows]
        if out is not None:
            out[rows] = _normed_and_turned(q[rows], q_norm, eps, at, rotary)
    return q if out is None and given is None else out


def paged_attention_ref(q, cache: PagedCache, starts, past, scale: Optional[float] = None, window: Optional[int] = None, most_new: Optional[int] = None, out=None):
    spans = _spans("paged_attention", cache, q.shape[0], starts, past, most_new)
    page = cache.keys.shape[2]
    result = torch.zeros(q.shape, dtype=q.dtype, device=q.device) if out is None else out
    for s, (start, new, p) in enumerate(spans):
        if not new:
            continue
        total = p + new
        first = 0 if window is None else max(0, p - window + 1)  # the first key that a token sees
        pages = _pages_of("paged_attention", cache, s, first // page, (total - 1) // page)
        k, v = (t[pages].transpose(1, 2).flatten(0, 1)[first - first // page * page:][:total - first] for t in (cache.keys, cache.values))
        at, key = torch.arange(p, total, device=q.device)[:, None], torch.arange(first, total, device=q.device)[None]
        hidden = key > at if window is None else (key > at) | (key <= at - window)
        bias = torch.zeros(new, total - first, device=q.device).masked_fill_(hidden, float("-inf"))
        result[start:start + new] = attention_ref(q[None, start:start + new], k[None], v[None], False, bias, scale)[0]
    return result


def adjust_logits_ref(logits, tokens=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None, bias=None, allowed=None):
    x = logits.float()
    rows, vocab = logits.shape

    def per_row(value, neutral):
        return neutral if value is None else value[:, None] if isinstance(value, torch.Tensor) else value

    if tokens is not None:
        at = torch.arange(tokens.shape[1], device=tokens.device)[None]
        there = (tokens >= 0) & (tokens < vocab)
        if lengths is not None:
            there = there & (at < lengths[:, None])
        said = there if prompt_lengths is None else there & (at >= prompt_lengths[:, None])
        index = tokens.clamp(0, max(vocab - 1, 0))
        seen = torch.zeros(rows, vocab, dtype=torch.int32, device=logits.device).scatter_add(1, index, there.int()) > 0
        count = torch.zeros(rows, vocab, dtype=torch.int32, device=logits.device).scatter_add(1, index, said.int())
        r = per_row(repetition, 1.0)
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = torch.where(count > 0, x - (per_row(frequency, 0.0) * count.float() + per_row(presence, 0.0)), x)
    if bias is not None:
        x = x + bias.float()
    if allowed is not None:
        token = torch.arange(vocab, device=logits.device)
        bits = allowed[..., token // 32] >> (token % 32).int() & 1
        x = x.masked_fill(bits == 0, float("-inf"))
    return x.to(logits.dtype)


# -- dispatching front-end ---------------------------------------------------------------------


def linear(x, weight, bias=None):
    nat = _native(x)
    if nat is not None and nat.gemm_supported(x, weight):
        return nat.linear(x, weight, bias)
    return F.linear(x, weight, bias)


def linears(x, weights):
    """Several projections of ``x`` by one autograd node, or None where each has to be its own."""
    nat = _native(x)
    return nat.linears(x, weights) if nat is not None and nat.linears_supported(x, weights) else None


def rms_norm(x, weight, eps: float = 1e-6):
    nat = _native(x)
    if nat is not None and nat.norm_supported(x):
        return nat.rms_norm(x, weight, eps)
    return rms_norm_ref(x, weight, eps)


def layer_norm(x, weight, bias, eps: float = 1e-5):
    nat = _native(x)
    if nat is not None and nat.norm_supported(x):
        return nat.layer_norm(x, weight, bias, eps)
    return layer_norm_ref(x, weight, bias, eps)


def apply_rope(x, positions, theta: float = 10000.0, rotary_dim: Optional[int] = None, interleaved: bool = False):
    nat = _native(x)
    if nat is not None and nat.rope_supported(x):
        return nat.rope(x, positions, theta, rotary_dim, interleaved)
    return apply_rope_ref(x, positions, theta, rotary_dim, interleaved)


def attention(q, k, v, causal: bool, bias=None, scale: Optional[float] = None):
    nat = _native(q)
    if nat is not None and nat.attention_supported(q, k, v, bias):
        return nat.attention(q, k, v, causal, bias, scale)
    return attention_ref(q, k, v, causal, bias, scale)


def _only_looks_rows_up(embedding: torch.nn.Module) -> bool:
    """False for an embedding whose call does more than look rows of its weight up: another class, a ``forward`` put on the instance
    (offloading libraries), hooks of its own or of all modules, renormalisation, sparse or scaled gradients, a weight that is
    a tensor subclass."""
    every = torch.nn.modules.module
    hooks = (embedding._forward_hooks, embedding._forward_pre_hooks, embedding._backward_hooks, embedding._backward_pre_hooks, every._global_forward_hooks,
             every._global_forward_pre_hooks, every._global_backward_hooks, every._global_backward_pre_hooks)
    return (type(embedding) is torch.nn.Embedding and "forward" not in vars(embedding) and type(embedding.weight) in (torch.nn.Parameter, torch.Tensor)
            and embedding.max_norm is None and embedding.padding_idx is None and not embedding.sparse and not embedding.scale_grad_by_freq and not any(hooks))


_compiling = torch.compiler.is_dynamo_compiling
_AHEAD_OF_DISPATCH = torch._C.DispatchKey.PreDispatch


def transformed(t: torch.Tensor) -> bool:
    """True where an autograd function over raw pointers would drop out of what is going on around it: a functorch transform (vmap,
    grad, jvp), a batch of gradients (``is_grads_batched``), a forward-mode tangent, a dispatch mode (fake tensors, ``make_fx``, ahead of dispatch
    too), tracing or compilation."""
    functorch = torch._C._functorch
    return (functorch.peek_interpreter_stack() is not None or functorch.is_functorch_wrapped_tensor(t) or functorch.is_legacy_batchedtensor(t)
            or torch._C._len_torch_dispatch_stack() > 0 or torch._C._dispatch_tls_is_dispatch_key_included(_AHEAD_OF_DISPATCH)
            or torch.jit.is_tracing() or torch.compiler.is_compiling() or torch.autograd.forward_ad.unpack_dual(t).tangent is not None)


def relative_bias(embedding: torch.nn.Module, buckets, queries: int, keys: int):
    """Score bias ``[1, heads, queries, keys]`` of a learned table over position buckets; ``buckets`` holds the bucket of each distance
    ``key - query``, from ``-(queries - 1)`` up, in ``queries + keys - 1`` entries.  An embedding that does more than look rows up is
    called as the module it is."""
    direct = (_only_looks_rows_up(embedding) and not transformed(embedding.weight) and buckets.device == embedding.weight.device
              and buckets.dtype in (torch.int64, torch.int32) and buckets.ndim == 1 and buckets.shape[0] >= queries + keys - 1)
    nat = _native(embedding.weight) if direct else None
    if nat is not None and nat.relative_bias_supported(embedding.weight, queries, keys):
        return nat.relative_bias(embedding.weight, buckets, queries, keys)
    return relative_bias_ref(embedding, buckets, queries, keys)


def relative_buckets(first: int, count: int, device, bidirectional: bool, buckets: int, max_distance: int):
    """Relative-position buckets of the distances ``first``, ``first + 1``, ... by one kernel, or None where the caller has to take the steps over
    tensors (other devices than the current one, functorch transforms, tracing, dispatch modes, ranges that the kernel does not cover)."""
    exact, device = buckets // (4 if bidirectional else 2), torch.device(device)
    if (device.type != "cuda" or _FORCE_TORCH or not 0 < count <= 2 ** 31 or type(buckets) is not int or type(max_distance) is not int
            or not 0 < exact < max_distance < 2 ** 31 or torch._C._functorch.peek_interpreter_stack() is not None
            or torch._C._len_torch_dispatch_stack() > 0 or torch._C._dispatch_tls_is_dispatch_key_included(_AHEAD_OF_DISPATCH)
            or torch.jit.is_tracing() or torch.compiler.is_compiling() or device.index not in (None, torch.cuda.current_device())):
        return None
    from tensor_parallel_b200.ops import native

    return native.relative_buckets(first, count, device, bidirectional, buckets, max_distance)


def gelu(x, approximate: str = "none"):
    nat = _native(x)
    if nat is not None and nat.elementwise_supported(x):
        return nat.gelu(x, approximate)
    return gelu_ref(x, approximate)


def relu(x):
    nat = _native(x)
    if nat is not None and nat.elementwise_supported(x):
        return nat.relu(x)
    return F.relu(x)


def swiglu(gate, up):
    nat = _native(gate)
    if nat is not None and nat.elementwise_supported(gate):
        return nat.swiglu(gate, up)
    return swiglu_ref(gate, up)


def geglu(gate, up, approximate: str = "tanh"):
    nat = _native(gate)
    if nat is not None and nat.elementwise_supported(gate):
        return nat.geglu(gate, up, approximate)
    return geglu_ref(gate, up, approximate)


# -- 8-bit integers (serving) --------------------------------------------------------------------


def _not_taken(*args):
    return None


# The ordinary calls, as the native module takes them once it is loaded: its results, or None for a call that needs a check's words or a copy.  Not while a compiler
# traces the front end, which would stop there: it gets the steps.
quantize_int8_directly = norm_int8_directly = linear_int8_directly = _not_taken
paged_append_directly = paged_attention_directly = adjust_logits_directly = _not_taken


def _serving_only(what: str, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad()")
    if any(t is not None and t.is_floating_point() and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no derivative, in forward mode neither")


def _check_rows(what: str, x, weight=None, bias=None, residual=None):
    if x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{what} takes bf16 or fp32 rows, got {x.dtype}")
    if x.ndim < 1 or x.shape[-1] == 0:
        raise ValueError(f"{what} takes rows of at least one column, got {tuple(x.shape)}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (t.shape != x.shape[-1:] or t.device != x.device):
            raise ValueError(f"{what}: {name} {tuple(t.shape)} on {t.device} does not fit rows {tuple(x.shape)} on {x.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"{what}: the residual has to be like x ({tuple(x.shape)}, {x.dtype}, {x.device}), got {tuple(residual.shape)}, {residual.dtype}, {residual.device}")
    _serving_only(what, x, weight, bias, residual)


def quantize_int8(x) -> Int8Rows:
    """The rows of ``x`` (bf16 or fp32, ``[..., cols]``) in 8 bits: ``rint(x * (127 / max |x|))`` and ``max |x| / 127``, ties to even.  For an activation
    in front of :func:`linear_int8`, and for its weight (a row per output channel).  A row with a value that is not finite gets the scale NaN.
    Serving only: there is no gradient."""
    if not _compiling():
        out = quantize_int8_directly(x)
        if out is not None:
            return out
    nat = None if _compiling() else _native(x)
    _check_rows("quantize_int8", x)
    return quantize_int8_ref(x) if nat is None or transformed(x) else nat.quantize_int8(x)


def rms_norm_int8(x, weight, eps: float = 1e-6, residual=None) -> Tuple[Int8Rows, torch.Tensor]:
    """``(rows, h)``: ``h = x + residual``, rounded to the type of ``x`` (``x`` itself without a residual), and its RMSNorm in 8 bits, as
    :func:`quantize_int8` gives them.  ``weight`` may be None.  A row whose sum of squares passes the range of fp32 (a value above 2^64 is enough) gets
    the scale NaN."""
    if not _compiling():
        out = norm_int8_directly(x, weight, None, eps, 0, residual)
        if out is not None:
            return out
    nat = None if _compiling() else _native(x)
    _check_rows("rms_norm_int8", x, weight, residual=residual)
    return rms_norm_int8_ref(x, weight, eps, residual) if nat is None or transformed(x) else nat.norm_int8(x, weight, None, eps, 0, residual)


def layer_norm_int8(x, weight, bias, eps: float = 1e-5, residual=None) -> Tuple[Int8Rows, torch.Tensor]:
    """Like :func:`rms_norm_int8`, with a LayerNorm; ``weight`` and ``bias`` may be None.  A row gets the scale NaN where the sum of its values, or of the
    squares of its deviations, passes the range of fp32."""
    if not _compiling():
        out = norm_int8_directly(x, weight, bias, eps, 1, residual)
        if out is not None:
            return out
    nat = None if _compiling() else _native(x)
    _check_rows("layer_norm_int8", x, weight, bias, residual)
    return layer_norm_int8_ref(x, weight, bias, eps, residual) if nat is None or transformed(x) else nat.norm_int8(x, weight, bias, eps, 1, residual)


INT8_ACTS = (None, "relu", "gelu", "gelu_tanh", "silu", "swiglu16")


def _check_linear_int8(x, weight, bias, act, residual):
    for name, rows in (("x", x), ("weight", weight)):
        v, s = rows
        if v.dtype != torch.int8 or s.dtype != torch.float32 or s.shape != v.shape[:-1] or s.device != v.device:
            raise ValueError(f"linear_int8: {name} takes int8 values with one fp32 scale per row, got {v.dtype} {tuple(v.shape)} and {s.dtype} {tuple(s.shape)}")
    xv, wv = x[0], weight[0]
    if xv.ndim < 2 or wv.ndim != 2 or xv.shape[-1] != wv.shape[1] or xv.device != wv.device:
        raise ValueError(f"linear_int8: rows {tuple(xv.shape)} on {xv.device} and a weight {tuple(wv.shape)} on {wv.device} do not contract")
    features, k = wv.shape
    if not 0 < k <= INT8_MAX_K or features == 0:
        raise ValueError(f"linear_int8 contracts 1 to {INT8_MAX_K} columns into at least one feature, got a weight {tuple(wv.shape)}")
    if act not in INT8_ACTS:
        raise ValueError(f"linear_int8: unknown activation {act!r}")
    if act == "swiglu16" and (features % 32 or residual is not None):
        raise ValueError("linear_int8: swiglu16 takes weight rows in groups of 16 gate and 16 up rows, and no residual")
    if bias is not None and (bias.shape != (features,) or bias.dtype != torch.bfloat16 or bias.device != xv.device):
        raise ValueError(f"linear_int8: the bias has to be bf16 [{features}] on {xv.device}, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
    if residual is not None and (residual.shape != (*xv.shape[:-1], features) or residual.dtype != torch.bfloat16 or residual.device != xv.device):
        raise ValueError(f"linear_int8: the residual has to be bf16 {(*xv.shape[:-1], features)} on {xv.device}, got {residual.dtype} {tuple(residual.shape)} on {residual.device}")
    _serving_only("linear_int8", x[1], weight[1], bias, residual)


def linear_int8(x: Int8Rows, weight: Int8Rows, bias=None, act: Optional[str] = None, residual=None):
    """``act(x @ weight.T + bias) + residual`` in bf16, for rows and a weight in 8 bits (:class:`Int8Rows`, ``[..., k]`` and ``[features, k]``): the sums of
    products are exact integers, scales, bias, activation and residual are fp32.  ``act``: None, ``"relu"``, ``"gelu"``, ``"gelu_tanh"``, ``"silu"``, or
    ``"swiglu16"`` for a weight whose rows alternate in groups of 16 gate and 16 up rows (``silu(gate) * up``, half as many columns).  Serving only:
    there is no gradient."""
    if not _compiling():
        out = linear_int8_directly(x, weight, bias, act, residual)
        if out is not None:
            return out
    nat = None if _compiling() else _native(x[0])
    _check_linear_int8(x, weight, bias, act, residual)
    if nat is None or transformed(x[0]) or transformed(x[1]):
        return linear_int8_ref(Int8Rows(*x), Int8Rows(*weight), bias, act, residual)
    return nat.linear_int8(x, weight, bias, act, residual)


# -- sequences of different lengths (serving) ------------------------------------------------------


def _not_captured(what: str):
    """A kernel would leave nothing in a captured graph, and the steps depend on lengths that are on the device."""
    if (torch._C._functorch.peek_interpreter_stack() is not None or torch.jit.is_tracing()
            or torch._C._dispatch_tls_is_dispatch_key_included(_AHEAD_OF_DISPATCH) or _capturing_modes()):
        raise RuntimeError(f"{what} reads lengths on the device: it cannot be traced, captured as operators or transformed (CUDA graphs are fine)")


def _capturing_modes() -> bool:
    modes = torch._C._TorchDispatchModeKey
    return torch._C._len_torch_dispatch_stack() > 0 and any(torch._C._get_dispatch_mode(key) is not None for key in (modes.PROXY, modes.FAKE, modes.FUNCTIONAL))


def _check_paged(what: str, cache, starts, past, rows):
    """``rows``: name -> ``[tokens, heads, head_dim]``."""
    keys, values, table = cache
    if keys.ndim != 4 or values.shape != keys.shape or values.dtype != keys.dtype or not keys.is_floating_point():
        raise ValueError(f"{what}: keys and values have to be [pages, kv_heads, page_size, head_dim] of one type, got {keys.dtype} {tuple(keys.shape)} and "
                         f"{values.dtype} {tuple(values.shape)}")
    for name, t, shape in (("the table", table, (None, None)), ("starts", starts, (None,)), ("past", past, (None,))):
        if t.dtype != torch.int32 or t.ndim != len(shape):
            raise ValueError(f"{what}: {name} has to be int32 with {len(shape)} dimension{'s' * (len(shape) > 1)}, got {t.dtype} {tuple(t.shape)}")
    n = past.shape[0]
    if starts.shape[0] != n + 1 or table.shape[0] != n:
        raise ValueError(f"{what}: {n} cached lengths go with {n + 1} starts and {n} rows of the table, got {starts.shape[0]} and {table.shape[0]}")
    tokens = None
    for name, t in rows.items():
        if t is None:
            continue
        if t.ndim != 3 or t.dtype != keys.dtype or t.shape[2] != keys.shape[3] or (tokens is not None and t.shape[0] != tokens):
            raise ValueError(f"{what}: {name} has to be [tokens, heads, {keys.shape[3]}] in {keys.dtype}, got {t.dtype} {tuple(t.shape)}")
        tokens = t.shape[0]
    for t in (values, table, starts, past, *rows.values()):
        if t is not None and t.device != keys.device:
            raise ValueError(f"{what}: all tensors have to be on {keys.device}, got one on {t.device}")
    if tokens and n and (0 in keys.shape or table.shape[1] == 0):
        raise ValueError(f"{what}: a cache of {tuple(keys.shape)} with a table of {tuple(table.shape)} has no place for {tokens} tokens")


def _check_out(what: str, out, like):
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{what}: out has to be like q ({tuple(like.shape)}, {like.dtype}, {like.device}, no element twice), got {tuple(out.shape)}, {out.dtype}, {out.device}")


def paged_append(cache: PagedCache, q, k, v, starts, past, rotary: Optional[Rotary] = None, q_norm=None, k_norm=None, eps: float = 1e-6, out=None):
    """Writes the new keys and values of a ragged batch to a paged cache and returns its queries; keys and queries are normed and rotated on the way.

    ``k`` and ``v`` are ``[tokens, kv_heads, head_dim]`` and ``q`` ``[tokens, heads, head_dim]`` (strided views of one projection are fine; ``q`` may be None): rows
    ``starts[s]`` to ``starts[s + 1]`` belong to sequence ``s``, and follow its ``past[s]`` keys in the cache (int32, ``[sequences + 1]`` and ``[sequences]``).  ``q_norm`` and
    ``k_norm``, ``[head_dim]``, ask for an RMSNorm of each head, ``rotary`` for the rotation by the token's position (its index in the sequence) behind it.
    Angles are exact at any position; results are rounded once.

    The queries come in a tensor of their own, in ``out`` (which may be ``q``), or as they are where nothing is done to them.  Rows in front of the first
    sequence and behind the last (a batch padded to a captured size) are not stored; ``out`` keeps what it has there, and a new tensor holds zeros.
    The CUDA kernel takes bf16, heads of up to 256 elements in eights and pages of a power of two; other calls go by their steps, which read the lengths on the host (no CUDA graph).

    A sequence whose rows, table or pages do not fit is not stored: the CUDA kernel records status 3 (see ``native.device_state``), the steps over
    tensors raise.  Two tokens for one slot (sequences that share the page that they write to) leave either.  Serving only: there is no gradient."""
    if _compiling():
        torch._dynamo.graph_break()
    done = paged_append_directly(cache, q, k, v, starts, past, rotary, q_norm, k_norm, eps, out)
    if done is not None:
        return done[0]
    _check_paged("paged_append", cache, starts, past, dict(q=q, k=k, v=v))
    d, kv_heads = cache[0].shape[3], cache[0].shape[1]
    if k.shape[1] != kv_heads or v.shape[1] != kv_heads:
        raise ValueError(f"paged_append: the cache has {kv_heads} heads, got keys {tuple(k.shape)} and values {tuple(v.shape)}")
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None and (t.shape != (d,) or t.dtype != k.dtype or t.device != k.device):
            raise ValueError(f"paged_append: {name} has to be {k.dtype} [{d}] on {k.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if rotary is not None:
        f = rotary[0]
        if f.dtype != torch.float32 or f.ndim != 1 or f.device != k.device or not 0 < 2 * f.shape[0] <= d:
            raise ValueError(f"paged_append: frequencies have to be fp32 on {k.device}, 1 to {d // 2} of them, got {f.dtype} {tuple(f.shape)} on {f.device}")
    if out is not None:
        if q is None:
            raise ValueError("paged_append: out is for queries, and there are none")
        _check_out("paged_append", out, q)
    _serving_only("paged_append", cache[0], cache[1], q, k, v, q_norm, k_norm, out)
    _not_captured("paged_append")
    nat = _native(k)
    if nat is not None and nat.paged_append_supported(cache, q, k, v, out):
        return nat.paged_append(cache, q, k, v, starts, past, rotary, q_norm, k_norm, eps, out)
    return paged_append_ref(PagedCache(*cache), q, k, v, starts, past, None if rotary is None else Rotary(*rotary), q_norm, k_norm, eps, out)


def paged_attention(q, cache: PagedCache, starts, past, scale: Optional[float] = None, window: Optional[int] = None, most_new: Optional[int] = None, out=None):
    """Causal attention of the new tokens of a ragged batch over a paged cache that holds their own keys and values already (:func:`paged_append`).

    ``q`` is ``[tokens, heads, head_dim]``; ``starts`` and ``past`` as for :func:`paged_append`, ``past`` not counting the new tokens: row ``starts[s] + i`` sees keys ``0`` to
    ``past[s] + i`` of sequence ``s``, or the last ``window`` of them.  One token of each sequence is a decode step, a whole prompt is a prefill, and
    sequences of both kinds may be in one batch.  ``most_new`` says how many new tokens any sequence has at most, where the caller knows (the launches
    are chosen by it; without it those for prompts are made too).  A call has a workspace of up to 51 MB.  What lies in the cache outside of a sequence's keys has no influence, whatever it is, and pages that have left every token's window are not
    read; a sequence's own keys and values have to be finite (one that is not may reach any of its new tokens).  A row of queries with scores that are not finite gives NaN.

    The CUDA kernels take bf16, heads of 64 or 128 elements and pages of a power of two from 16 up; other calls go by their steps, which read the lengths on the host (no CUDA graph).

    The result is a new tensor, zero in rows outside all sequences, or ``out`` (which may be ``q``), left as it is there.  A sequence whose rows or table
    do not fit, or with more than ``most_new`` new tokens, gives NaN, as rows do that reach a page outside the cache (and some of those in front of them in its sequence), and the CUDA kernel records status 3
    (see ``native.device_state``); the steps over tensors raise.  Serving only: there is no gradient."""
    if _compiling():
        torch._dynamo.graph_break()
    done = paged_attention_directly(q, cache, starts, past, scale, window, most_new, out)
    if done is not None:
        return done
    _check_paged("paged_attention", cache, starts, past, dict(q=q))
    if q.shape[1] == 0 or cache[0].shape[1] == 0 or q.shape[1] % cache[0].shape[1]:
        raise ValueError(f"paged_attention: {q.shape[1]} query heads are no multiple of {cache[0].shape[1]} in the cache")
    if window is not None and window < 1:
        raise ValueError(f"paged_attention: a window holds at least the token itself, got {window}")
    if most_new is not None and most_new < 0:
        raise ValueError(f"paged_attention: most_new={most_new}")
    if scale is not None and not 0 < scale < math.inf:
        raise ValueError(f"paged_attention: the scale has to be positive, got {scale}")
    if out is not None:
        _check_out("paged_attention", out, q)
    _serving_only("paged_attention", q, cache[0], cache[1], out)
    _not_captured("paged_attention")
    nat = _native(q)
    if nat is not None and nat.paged_attention_supported(q, cache, out):
        return nat.paged_attention(q, cache, starts, past, scale, window, most_new, out)
    return paged_attention_ref(q, PagedCache(*cache), starts, past, scale, window, most_new, out)


def _check_adjust(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed):
    what = "adjust_logits"
    if logits.ndim != 2 or not logits.is_floating_point():
        raise ValueError(f"{what} takes logits [rows, vocabulary], got {logits.dtype} {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if tokens is None and any(t is not None for t in (lengths, prompt_lengths, repetition, frequency, presence)):
        raise ValueError(f"{what}: lengths and penalties are for the tokens that a sequence has had, and none are given")
    if tokens is not None and (tokens.dtype != torch.int64 or tokens.ndim != 2 or tokens.shape[0] != rows):
        raise ValueError(f"{what}: tokens have to be int64 [{rows}, width], got {tokens.dtype} {tuple(tokens.shape)}")
    for name, t in (("lengths", lengths), ("prompt_lengths", prompt_lengths)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (rows,)):
            raise ValueError(f"{what}: {name} have to be int32 [{rows}], got {t.dtype} {tuple(t.shape)}")
    for name, t in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
        if isinstance(t, torch.Tensor):
            if t.dtype != torch.float32 or t.shape != (rows,):
                raise ValueError(f"{what}: {name} has to be a number or fp32 [{rows}], got {t.dtype} {tuple(t.shape)}")
        elif name == "repetition" and t is not None and not t > 0:
            raise ValueError(f"{what}: logits are divided by repetition, which has to be positive, got {t}")
    if bias is not None and (bias.shape not in ((vocab,), (rows, vocab)) or bias.dtype not in (torch.bfloat16, torch.float32)):
        raise ValueError(f"{what}: the bias has to be bf16 or fp32 [{vocab}] or [{rows}, {vocab}], got {bias.dtype} {tuple(bias.shape)}")
    words = (vocab + 31) // 32
    if allowed is not None and (allowed.shape not in ((words,), (rows, words)) or allowed.dtype != torch.int32):
        raise ValueError(f"{what}: allowed tokens are bits of int32 [{words}] or [{rows}, {words}], got {allowed.dtype} {tuple(allowed.shape)}")
    for t in (tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed):
        if isinstance(t, torch.Tensor) and t.device != logits.device:
            raise ValueError(f"{what}: all tensors have to be on {logits.device}, got one on {t.device}")
    _serving_only(what, *(t if isinstance(t, torch.Tensor) else None for t in (logits, repetition, frequency, presence, bias)))


def adjust_logits(logits, tokens=None, lengths=None, prompt_lengths=None, repetition=None, frequency=None, presence=None, bias=None, allowed=None):
    """Logits ``[rows, vocabulary]`` as they go into the pick of a token, in their own type (32 bits on the way), in this order:

    * penalties for the tokens that a row has had, the first ``lengths[row]`` (None: all) of ``tokens[row]`` (int64 ``[rows, width]``; ids outside the vocabulary do not
      count): a positive logit is divided by ``repetition`` and another multiplied by it; for those behind the first ``prompt_lengths[row]`` (None: 0), how often
      one was said times ``frequency``, and ``presence`` once, are subtracted.  Each is None, a number, or fp32 ``[rows]``.
    * ``bias``, fp32 or bf16, ``[vocabulary]`` or ``[rows, vocabulary]``, is added;
    * tokens that ``allowed`` does not name become ``-inf``: bit ``i`` of word ``w`` stands for token ``32 w + i`` (int32 ``[words]`` or ``[rows, words]``).

    Lengths beyond the width count as the width, below zero as zero (the CUDA kernel records status 3).  Serving only: there is no gradient."""
    if not _compiling():
        done = adjust_logits_directly(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed)
        if done is not None:
            return done
        nat = _native(logits)
        _check_adjust(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed)
        if nat is not None and nat.adjust_logits_supported(logits) and not transformed(logits):
            return nat.adjust_logits(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed)
    else:
        _check_adjust(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed)
    return adjust_logits_ref(logits, tokens, lengths, prompt_lengths, repetition, frequency, presence, bias, allowed)


def cross_entropy(logits, labels, ignore_index: int = -100):
    return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), labels.reshape(-1), ignore_index=ignore_index)
