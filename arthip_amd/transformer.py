"""Transformer operators over libarthip.so: the block of an image or video network.

``rope_axes`` (rotary positions with several axes), ``attention`` (capped scores,
distance bias, windows, prefixes, documents, ragged caches) and ``gated_norm`` (the
norms around a gated residual) mirror the C entry points of the same names, which
include/arthip.h describes. Inference only.

Tensors are torch tensors on one GPU (torch is used only as device-memory plumbing)
and keep their strides: only the innermost dimension has to be contiguous. Work goes
to torch's current stream, or to ``stream`` (a raw handle); results that a call makes
itself belong to that stream. Arguments that do not fit raise :class:`EngineError`
before anything is launched. Numbers may be tensors or arrays of one value, which are
read at each call (from a tensor on the GPU with a synchronization).
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .engine import EngineError

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_NORMS = {None: 0, "none": 0, "rms": 1, "layer": 2}
_GATES = {None: 0, "none": 0, "sigmoid": 1, "tanh": 2, "silu": 3}


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise EngineError(text)


def _float(name: str, x) -> float:
    try:
        return float(x)
    except (TypeError, ValueError, RuntimeError):
        raise EngineError(f"{name} must be a number") from None


def _int(name: str, x) -> int:
    try:
        n = int(x)
        if n == x and -2 ** 31 <= n < 2 ** 31:
            return n
    except (TypeError, ValueError, OverflowError, RuntimeError):
        pass
    raise EngineError(f"{name} must be a whole number of 32 bits")


def _bool(name: str, x) -> bool:
    try:
        return bool(x)
    except (TypeError, ValueError, RuntimeError):
        raise EngineError(f"{name} must be a truth value") from None


def _pair(name: str, x) -> tuple:
    try:
        pair = tuple(x)
    except TypeError:
        pair = ()
    _need(len(pair) == 2, f"{name} must be a pair")
    return pair


# What a call's shapes, strides, types and options come to (checked arguments with all
# pointers empty), so that the next call of the same kind only fills in pointers: a call
# takes some 8 us instead of 18. Nothing in it depends on a tensor's address or contents:
# options become plain numbers before they are part of a key.
_plans: dict = {}
_PLANS = 512


def _keep(key, plan):
    if len(_plans) >= _PLANS:
        _plans.clear()
    _plans[key] = plan
    return plan


def _sig(t):
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise EngineError(f"a {type(t).__name__} where a tensor on a GPU belongs")
    return t.shape, t.stride(), t.dtype, t.device


def _call(fn, args, device, stream) -> None:
    """Enqueues on the tensors' device, on its current stream or the one given."""
    index = device.index
    if stream is None:
        stream = torch._C._cuda_getCurrentRawStream(index)
    if index == torch._C._cuda_getDevice():
        rc = fn(ctypes.byref(args), stream)
    else:
        with torch.cuda.device(index):
            rc = fn(ctypes.byref(args), stream)
    if rc != 0:
        raise EngineError(_lib.last_error() or f"{fn.__name__} failed")


def _like(t, stream):
    """A contiguous tensor of t's shape and type that belongs to the call's stream."""
    if stream is None and t.is_contiguous():
        return torch.empty_like(t)  # half the time of torch.empty
    return _empty(t.shape, t.dtype, t.device, stream)


def _empty(shape, dtype, device, stream):
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    # An external stream of the handle 0 would be one of torch's own streams, not the default one,
    # and the memory could be given out again there while the call still writes to it.
    on = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    with torch.cuda.stream(on):
        return torch.empty(shape, dtype=dtype, device=device)


def _check(name: str, t, device, dtype, dim: int | None = None) -> None:
    _need(t is not None and t.is_cuda, f"{name} must be a tensor on a GPU")
    _need(t.device == device, f"{name} is on another device")
    _need(t.dtype == dtype, f"{name} must be {dtype}, is {t.dtype}")
    _need(dim is None or t.dim() == dim, f"{name} must have {dim} dimensions")


def _sizes(name: str, t) -> None:
    """The C structs hold sizes in 32 bits, and ctypes would cut off the rest."""
    _need(max(t.shape, default=0) < 2 ** 31, f"{name} has too many entries")


def _inner(name: str, t) -> None:
    _need(t.stride(-1) == 1 or t.shape[-1] <= 1, f"{name}: the innermost dimension must be contiguous")


# -- rotary positions ---------------------------------------------------------------

class RopePlan:
    """The frequencies of a rotary embedding, packed for the kernel and kept on the GPU.

    ``sections`` gives the turned pairs of each axis (time, height, width, ...); their
    sum n turns 2 n values of a head. Pair f turns by position * theta ** (-f / n), f
    counted over all axes, or with ``per_axis`` over its own axis' pairs. ``order``
    "blocks" gives an axis its pairs in a row, "cycle" deals them out one axis after
    the other. ``scale`` multiplies an axis' positions. ``pairs`` turns neighbours (2f,
    2f + 1) rather than (f, f + n). ``freqs`` (radians a position) replaces theta."""

    def __init__(self, sections, *, theta: float = 10000.0, per_axis: bool = False,
                 pairs: bool = False, order: str = "blocks", scale=None, freqs=None,
                 device="cuda"):
        sections = [int(s) for s in sections]
        _need(len(sections) > 0 and min(sections) >= 0 and sum(sections) > 0,
              "RopePlan: sections must be counts of pairs")
        _need(order in ("blocks", "cycle"), "RopePlan: order is 'blocks' or 'cycle'")
        _need(theta > 0, "RopePlan: theta must be positive")
        n = sum(sections)
        scale = [1.0] * len(sections) if scale is None else [float(s) for s in scale]
        _need(len(scale) == len(sections), "RopePlan: one scale an axis")
        if order == "blocks":
            axis = [a for a, s in enumerate(sections) for _ in range(s)]
        else:
            axis = [a for turn in range(max(sections)) for a, s in enumerate(sections) if turn < s]
        if freqs is None:
            freqs, seen = [], [0] * len(sections)
            for f, a in enumerate(axis):
                freqs.append(theta ** (-(seen[a] / sections[a] if per_axis else f / n)))
                seen[a] += 1
        _need(len(freqs) == n, "RopePlan: one frequency a pair")
        self.n, self.n_axes, self.pairs = n, len(sections), bool(pairs)
        self.axis = tuple(axis)
        self.freqs = tuple(float(f) * scale[a] for f, a in zip(freqs, axis))
        lib = _lib.lib()
        host = torch.empty(lib.arthip_rope_packed_bytes(n), dtype=torch.uint8)
        rc = lib.arthip_rope_pack((ctypes.c_double * n)(*self.freqs), (ctypes.c_int32 * n)(*axis), n,
                                  self.n_axes, host.data_ptr(), host.numel())
        if rc != 0:
            raise EngineError(_lib.last_error() or "arthip_rope_pack failed")
        self.packed = host.to(device)


def rope_axes(q, k, pos, plan: RopePlan, *, q_out=None, k_out=None, inverse: bool = False,
              stream=None):
    """Queries [B, L, Hq, D] and keys [B, L, Hk, D] (either may be None) turned by int32
    positions [axes, B, L] (or [axes, L], the same for every batch item). Returns
    (q_out, k_out), new contiguous tensors unless given; q_out=q turns in place."""
    inverse = _bool("rope_axes: inverse", inverse)
    key = ("rope", _sig(q), _sig(k), _sig(pos), _sig(q_out), _sig(k_out), plan.n, plan.n_axes, plan.pairs,
           plan.packed.device, inverse)
    template = _plans.get(key) or _keep(key, _rope_plan(q, k, pos, plan, q_out, k_out, inverse))
    a = _lib.RopeArgs.from_buffer_copy(template)
    device = pos.device
    if q is not None:
        if q_out is None:
            q_out = _like(q, stream)
        a.q, a.q_out = q.data_ptr(), q_out.data_ptr()
    if k is not None:
        if k_out is None:
            k_out = _like(k, stream)
        a.k, a.k_out = k.data_ptr(), k_out.data_ptr()
    a.pos, a.packed = pos.data_ptr(), plan.packed.data_ptr()
    _call(_lib.lib().arthip_rope_axes, a, device, stream)
    return q_out, k_out


def _contiguous(shape) -> tuple:
    strides, n = [], 1
    for size in reversed(shape):
        strides.append(n)
        n *= max(size, 1)
    return tuple(reversed(strides))


def _rope_plan(q, k, pos, plan, q_out, k_out, inverse) -> bytes:
    x = q if q is not None else k
    _need(x is not None and x.is_cuda, "rope_axes: q or k must be a tensor on a GPU")
    _need(x.dtype in _TYPES, f"rope_axes: unsupported type {x.dtype}")
    _need(x.dim() == 4, "rope_axes: q and k must have 4 dimensions")
    batch, tokens, _, dim = x.shape
    _check("pos", pos, x.device, torch.int32)
    _need(tuple(pos.shape) in ((plan.n_axes, batch, tokens), (plan.n_axes, tokens)),
          "rope_axes: pos must be [axes, B, L] or [axes, L]")
    _need(plan.packed.device == x.device, "rope_axes: the plan is on another device")
    a = _lib.RopeArgs()
    for name, t, out in (("q", q, q_out), ("k", k, k_out)):
        if t is None:
            _need(out is None, f"rope_axes: {name}_out without {name}")
            continue
        _check(name, t, x.device, x.dtype, 4)
        _sizes(name, t)
        _need(t.shape[0] == batch and t.shape[1] == tokens and t.shape[3] == dim,
              "rope_axes: q and k must agree in batch, tokens and head_dim")
        _inner(name, t)
        if out is not None:
            _check(name + "_out", out, x.device, x.dtype, 4)
            _need(out.shape == t.shape, f"rope_axes: {name}_out must have {name}'s shape")
            _inner(name + "_out", out)
        setattr(a, name + "_heads", t.shape[2])
        setattr(a, name + "_stride", t.stride()[:3])
        setattr(a, name + "_out_stride", (_contiguous(t.shape) if out is None else out.stride())[:3])
    st = pos.stride()
    a.pos_stride = st if pos.dim() == 3 else (st[0], 0, st[1])
    a.n_freq, a.dtype, a.pairs, a.inverse = plan.n, _TYPES[x.dtype], plan.pairs, inverse
    a.batch, a.tokens, a.head_dim = batch, tokens, dim
    return bytes(a)


# -- attention ------------------------------------------------------------------------

def attention(q, k, v, *, scale: float | None = None, cap: float = 0.0, causal: bool = False,
              window=(None, None), q_start=None, kv_len=None, prefix=None, docs=None, codes=None,
              slopes=None, table=None, table_zero: int = 0, out=None, return_lse: bool = False,
              workspace=None, stream=None):
    """softmax(score + mask) V of queries [B, Lq, Hq, D] over keys and values
    [B, Lk, Hk, D]; see arthip_attention. ``causal`` is window[1] = 0; ``window`` counts
    the keys to the left and right of a query's own position (None: no limit).
    q_start, kv_len and prefix are int32 [B]; docs and codes are pairs of int32 tensors
    (queries', keys'), [B, L] or [L]; slopes is fp32 [Hq], table fp32 [Hq, n]. Returns
    out, or (out, lse) with lse fp32 [B, Hq, Lq]. Without ``workspace`` (uint8) a call
    that needs one makes it."""
    scale = None if scale is None else _float("attention: scale", scale)
    cap, table_zero = _float("attention: cap", cap), _int("attention: table_zero", table_zero)
    causal = _bool("attention: causal", causal)
    window = tuple(None if w is None else _int("attention: a window's side", w)
                   for w in _pair("attention: window", window))
    for name, x in (("docs", docs), ("codes", codes)):
        _need(not isinstance(x, torch.Tensor), f"attention: {name} must be a pair of tensors")
    docs = None if docs is None else _pair("attention: docs", docs)
    codes = None if codes is None else _pair("attention: codes", codes)
    doc_q, doc_k = docs or (None, None)
    code_q, code_k = codes or (None, None)
    key = ("attention", _sig(q), _sig(k), _sig(v), scale, cap, causal, window, _sig(out), return_lse)
    plain = (q_start is None and kv_len is None and prefix is None and docs is None and codes is None
             and slopes is None and table is None)
    if not plain:
        more = (q_start, kv_len, prefix, doc_q, doc_k, code_q, code_k, slopes, table)
        key += tuple(_sig(t) for t in more) + (table_zero,)
    plan = _plans.get(key)
    if plan is None:
        plan = _keep(key, _attention_plan(q, k, v, scale, cap, causal, window, q_start, kv_len, prefix, docs,
                                          codes, slopes, table, table_zero, out))
    template, need = plan
    a = _lib.AttentionArgs.from_buffer_copy(template)
    device = q.device
    if out is None:
        out = _like(q, stream)
    a.q, a.k, a.v, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    lse = None
    if return_lse:
        lse = _empty((q.shape[0], q.shape[2], q.shape[1]), torch.float32, device, stream)
        a.lse = lse.data_ptr()
    if not plain:
        for name, t in zip(("q_start", "kv_len", "prefix", "doc_q", "doc_k", "code_q", "code_k", "slopes",
                            "table"), more):
            if t is not None:
                setattr(a, name, t.data_ptr())
    if workspace is None and need > 0:
        workspace = _empty((need,), torch.uint8, device, stream)
    elif workspace is not None:
        _need(isinstance(workspace, torch.Tensor), "workspace must be a tensor on a GPU")
        _check("workspace", workspace, device, torch.uint8, 1)
        _inner("workspace", workspace)
    if workspace is not None:
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    _call(_lib.lib().arthip_attention, a, device, stream)
    return (out, lse) if return_lse else out


def _attention_plan(q, k, v, scale, cap, causal, window, q_start, kv_len, prefix, docs, codes, slopes, table,
                    table_zero, out):
    """(checked arguments without pointers, bytes of workspace)."""
    _need(q is not None and q.is_cuda, "attention: q must be a tensor on a GPU")
    _need(q.dtype in (torch.float16, torch.bfloat16), f"attention: unsupported type {q.dtype}")
    device = q.device
    for name, t in (("q", q), ("k", k), ("v", v)):
        _check(name, t, device, q.dtype, 4)
        _sizes(name, t)
        _inner(name, t)
    batch, q_tokens, q_heads, dim = q.shape
    k_tokens, k_heads = k.shape[1], k.shape[2]
    _need(tuple(k.shape) == (batch, k_tokens, k_heads, dim) and k.shape == v.shape,
          "attention: k and v must be [B, Lk, Hk, D] of q's batch and head_dim")
    _need(k_heads > 0 and q_heads % k_heads == 0, "attention: q_heads must be a multiple of k_heads")
    a = _lib.AttentionArgs()
    for name, t in (("q_start", q_start), ("kv_len", kv_len), ("prefix", prefix)):
        if t is not None:
            _check(name, t, device, torch.int32)
            _need(tuple(t.shape) == (batch,) and t.is_contiguous(),
                  f"attention: {name} must be contiguous [B]")
    for name, pair in (("doc", docs), ("code", codes)):
        if pair is None:
            continue
        _need(pair[0] is not None and pair[1] is not None,
              f"attention: {name}s is a pair of tensors (queries', keys')")
        for side, t, tokens in (("q", pair[0], q_tokens), ("k", pair[1], k_tokens)):
            _check(f"{name}_{side}", t, device, torch.int32)
            _need(tuple(t.shape) in ((batch, tokens), (tokens,)),
                  f"attention: {name}_{side} must be [B, L] or [L]")
            _inner(f"{name}_{side}", t)
            setattr(a, f"{name}_{side}", 16)  # any address: which arrays there are decides the workspace
            setattr(a, f"{name}_{side}_stride", t.stride(0) if t.dim() == 2 else 0)
    if slopes is not None:
        _check("slopes", slopes, device, torch.float32)
        _need(tuple(slopes.shape) == (q_heads,) and slopes.is_contiguous(),
              "attention: slopes must be contiguous [Hq]")
    if table is not None:
        _check("table", table, device, torch.float32, 2)
        _sizes("table", table)
        _need(table.shape[0] == q_heads and table.is_contiguous(),
              "attention: table must be contiguous [Hq, n]")
        _need(table.shape[1] > 0, "attention: table without entries")
        a.table_len, a.table_zero = table.shape[1], table_zero
    left, right = window
    _need(not causal or right in (None, 0), "attention: causal and a window to the right")
    for side in (left, right):
        _need(side is None or side >= 0, "attention: a window counts keys")
    a.left = -1 if left is None else left
    a.right = 0 if causal else -1 if right is None else right
    for name, t in (("prefix", prefix), ("slopes", slopes), ("table", table)):
        if t is not None:
            setattr(a, name, 16)
    a.scale = 1.0 / math.sqrt(dim) if scale is None else scale
    a.cap = cap
    a.q_stride, a.k_stride, a.v_stride = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    a.dtype, a.batch, a.q_tokens, a.k_tokens = _TYPES[q.dtype], batch, q_tokens, k_tokens
    a.q_heads, a.k_heads, a.head_dim = q_heads, k_heads, dim
    if out is not None:
        _check("out", out, device, q.dtype, 4)
        _need(out.shape == q.shape, "attention: out must have q's shape")
        _inner("out", out)
    a.out_stride = (_contiguous(q.shape) if out is None else out.stride())[:3]
    return bytes(a), _lib.lib().arthip_attention_workspace(ctypes.byref(a))


# -- norms around a block ----------------------------------------------------------------

def _spread(name: str, t, shape, device, dtype):
    """Batch and token stride of a tensor that broadcasts to [B, L, C]."""
    _check(name, t, device, dtype)
    dims = tuple(t.shape)
    _need(1 <= len(dims) <= 3 and dims[-1] == shape[-1]
          and all(n in (1, m) for n, m in zip(dims[::-1], shape[::-1])),
          f"gated_norm: {name} must broadcast to [B, L, C]")
    _inner(name, t)
    strides = (0,) * (3 - len(dims)) + tuple(st if n > 1 else 0 for n, st in zip(dims, t.stride()))
    return strides[:2]


def gated_norm(residual, y=None, *, post=None, post_weight=None, post_bias=None, gate=None,
               gate_act="none", residual_scale: float = 1.0, branch_scale: float = 1.0, pre=None,
               pre_weight=None, pre_bias=None, mod_scale=None, mod_shift=None, eps: float = 1e-6,
               residual_out=None, h=None, dtype=None, stream=None):
    """The norms before and after a block with its gate and residual scale, on tokens
    [B, L, C]; see arthip_gated_norm. ``post`` and ``pre`` are "rms", "layer" or None,
    ``gate_act`` is "none", "sigmoid", "tanh" or "silu"; gate, mod_scale and mod_shift
    broadcast to [B, L, C] (no gate is one of 1), weights and biases are fp32 [C]. The residual has y's type or
    fp32. Returns (new residual, h); residual_out=residual updates in place, and without y
    and with a residual_scale of 1 the residual is returned as it is. h has y's type, or
    ``dtype`` where there is no y."""
    _need(residual is not None, "gated_norm: residual must be a tensor on a GPU")
    residual_scale = _float("gated_norm: residual_scale", residual_scale)
    branch_scale = _float("gated_norm: branch_scale", branch_scale)
    eps = _float("gated_norm: eps", eps)
    for name in (post, pre, gate_act):
        _need(name is None or isinstance(name, str), "gated_norm: norms and gate activations are texts")
    given = (residual, y, gate, mod_scale, mod_shift, post_weight, post_bias, pre_weight, pre_bias,
             residual_out, h)
    key = ("norm", *map(_sig, given), post, pre,
           gate_act, residual_scale, branch_scale, eps, dtype)
    plan = _plans.get(key)
    if plan is None:
        plan = _keep(key, _norm_plan(given, post, pre, gate_act, residual_scale, branch_scale, eps, dtype))
    template, dtype, new_residual, new_h = plan
    a = _lib.NormArgs.from_buffer_copy(template)
    device = residual.device
    a.residual = residual.data_ptr()
    new = residual
    if new_residual or residual_out is not None:
        new = residual_out if residual_out is not None else _like(residual, stream)
        a.residual_out = new.data_ptr()
    if new_h:
        h = _like(y, stream) if y is not None else _empty(residual.shape, dtype, device, stream)
    if h is not None:
        a.h = h.data_ptr()
    for name, t in zip(("y", "gate", "mod_scale", "mod_shift", "post_weight", "post_bias", "pre_weight",
                        "pre_bias"), given[1:9]):
        if t is not None:
            setattr(a, name, t.data_ptr())
    if a.residual_out or a.h:
        _call(_lib.lib().arthip_gated_norm, a, device, stream)
    return new, h


def _norm_plan(given, post, pre, gate_act, residual_scale, branch_scale, eps, dtype):
    """(checked arguments without pointers, type of h, whether a call makes a residual and an h)."""
    (residual, y, gate, mod_scale, mod_shift, post_weight, post_bias, pre_weight, pre_bias, residual_out,
     h) = given
    _need(residual.is_cuda, "gated_norm: residual must be a tensor on a GPU")
    _need(residual.dtype in _TYPES, f"gated_norm: unsupported type {residual.dtype}")
    _need(residual.dim() == 3, "gated_norm: residual must have 3 dimensions")
    _need(post in _NORMS and pre in _NORMS, "gated_norm: a norm is 'rms', 'layer' or None")
    _need(gate_act in _GATES, "gated_norm: unknown gate activation")
    _need(y is not None or (gate is None and post in (None, "none")),
          "gated_norm: gate or post norm without y")
    device, shape = residual.device, tuple(residual.shape)
    if y is not None:
        _need(y.dtype in _TYPES, "gated_norm: unsupported type of y")
        _need(dtype in (None, y.dtype), "gated_norm: h has y's type")
        dtype = y.dtype
    elif dtype is None:
        dtype = residual.dtype if h is None else h.dtype
    _need(dtype in _TYPES, f"gated_norm: unsupported type {dtype}")
    a = _lib.NormArgs()
    _sizes("residual", residual)
    _inner("residual", residual)
    a.residual_stride = residual.stride()[:2]
    if y is not None:
        _check("y", y, device, dtype, 3)
        _need(tuple(y.shape) == shape, "gated_norm: y must have the residual's shape")
        _inner("y", y)
        a.y_stride = y.stride()[:2]
    for name, t in (("gate", gate), ("mod_scale", mod_scale), ("mod_shift", mod_shift)):
        if t is not None:
            setattr(a, name + "_stride", _spread(name, t, shape, device, dtype))
    for name, t in (("post_weight", post_weight), ("post_bias", post_bias),
                    ("pre_weight", pre_weight), ("pre_bias", pre_bias)):
        if t is not None:
            _check(name, t, device, torch.float32, 1)
            _need(t.shape[0] == shape[2] and t.is_contiguous(),
                  f"gated_norm: {name} must be contiguous [C]")
    a.dtype, a.residual_dtype = _TYPES[dtype], _TYPES[residual.dtype]
    a.post, a.pre, a.gate_act = _NORMS[post], _NORMS[pre], _GATES[gate_act]
    a.batch, a.tokens, a.channels = shape
    a.eps, a.residual_scale, a.branch_scale = eps, residual_scale, branch_scale
    if residual_out is not None:
        _check("residual_out", residual_out, device, residual.dtype, 3)
        _need(tuple(residual_out.shape) == shape, "gated_norm: residual_out must have the residual's shape")
        _inner("residual_out", residual_out)
    a.residual_out_stride = (_contiguous(shape) if residual_out is None else residual_out.stride())[:2]
    if h is not None:
        _check("h", h, device, dtype, 3)
        _need(tuple(h.shape) == shape, "gated_norm: h must have the residual's shape")
        _inner("h", h)
    a.h_stride = (_contiguous(shape) if h is None else h.stride())[:2]
    normed = pre not in (None, "none") or mod_scale is not None or mod_shift is not None
    return (bytes(a), dtype, residual_out is None and (y is not None or residual_scale != 1.0),
            h is None and normed)
