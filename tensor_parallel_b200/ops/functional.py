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


def cross_entropy(logits, labels, ignore_index: int = -100):
    return F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), labels.reshape(-1), ignore_index=ignore_index)
