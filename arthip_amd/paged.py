"""A paged cache of keys and values over libarthip.so, for networks that read a clip or a
text piece by piece.

``cache_write`` puts new tokens' keys and values into their pages, ``paged_attention``
lets the new tokens look at them, ``key_weights`` adds up the attention weight that each
cached key gathers, and ``cache_evict`` cuts the cache to the keys that gathered most.
They mirror the C entry points of the same names, which include/arthip.h describes, and
keep the rules of :mod:`arthip_amd.transformer` (strides, streams, errors). Inference only.

The cache is two tensors [pages, page_size, Hk, D] and, all int32 on the GPU, ``pages``
[B, n] (each sequence's pages in order), ``kv_len`` [B] (its slots in use, the new tokens
among them) and ``q_offsets`` [B + 1] (its rows among the new tokens, which lie packed;
None: one token a sequence). They are read when a call runs: a captured call may be
replayed as they change. ``weights`` (fp32) and ``positions`` (int32) are [B, Hk, slots].
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .transformer import (_TYPES, _bool, _call, _check, _contiguous, _empty, _float, _inner, _int, _keep, _like,
                          _need, _plans, _sig, _sizes)


def _pages(name, a, k_cache, v_cache, pages, kv_len, q_offsets, tokens) -> torch.device:
    """Checks the cache and fills in its sizes."""
    _need(isinstance(k_cache, torch.Tensor) and k_cache.is_cuda, f"{name}: k_cache must be a tensor on a GPU")
    _need(k_cache.dtype in (torch.float16, torch.bfloat16), f"{name}: unsupported type {k_cache.dtype}")
    _need(k_cache.dim() == 4, f"{name}: k_cache must be [pages, page_size, Hk, D]")
    device = k_cache.device
    _sizes("k_cache", k_cache)
    _inner("k_cache", k_cache)
    a.k_cache_stride = k_cache.stride()[:3]
    if v_cache is not None:
        _check("v_cache", v_cache, device, k_cache.dtype, 4)
        _need(v_cache.shape == k_cache.shape, f"{name}: v_cache must have k_cache's shape")
        _inner("v_cache", v_cache)
        a.v_cache_stride = v_cache.stride()[:3]
    _check("pages", pages, device, torch.int32, 2)
    _sizes("pages", pages)
    _inner("pages", pages)
    batch = pages.shape[0]
    _check("kv_len", kv_len, device, torch.int32, 1)
    _need(kv_len.shape[0] == batch and (kv_len.is_contiguous() or batch <= 1), f"{name}: kv_len must be contiguous [B]")
    if q_offsets is not None:
        _check("q_offsets", q_offsets, device, torch.int32, 1)
        _need(q_offsets.shape[0] == batch + 1 and q_offsets.is_contiguous(),
              f"{name}: q_offsets must be contiguous [B + 1]")
    p = a.p
    p.pages_stride = pages.stride(0)
    p.batch, p.tokens, p.max_pages = batch, batch if tokens is None else tokens, pages.shape[1]
    p.pool_pages, p.page_size, p.k_heads, p.head_dim = k_cache.shape
    p.dtype = _TYPES[k_cache.dtype]
    return device


def _address(a, k_cache, v_cache, pages, kv_len, q_offsets) -> None:
    a.k_cache = k_cache.data_ptr()
    if v_cache is not None:
        a.v_cache = v_cache.data_ptr()
    p = a.p
    p.pages, p.kv_len = pages.data_ptr(), kv_len.data_ptr()
    if q_offsets is not None:
        p.q_offsets = q_offsets.data_ptr()


def _per_slot(name, what, t, device, dtype, batch, heads) -> tuple:
    """Strides of [B, Hk, slots]."""
    _check(what, t, device, dtype, 3)
    _sizes(what, t)
    _need(t.shape[0] == batch and t.shape[1] == heads, f"{name}: {what} must be [B, Hk, slots]")
    _inner(what, t)
    return t.stride()[:2]


def cache_write(k, v, k_cache, v_cache, pages, kv_len, q_offsets=None, *, positions=None, token_positions=None,
                stream=None):
    """New tokens' keys and values [T, Hk, D] into their sequences' last slots; see
    arthip_cache_write. ``positions`` gets the tokens' ``token_positions`` (int32 [T])."""
    key = ("write", _sig(k), _sig(v), _sig(k_cache), _sig(v_cache), _sig(pages), _sig(kv_len), _sig(q_offsets),
           _sig(positions), _sig(token_positions))
    template = _plans.get(key) or _keep(key, _write_plan(k, v, k_cache, v_cache, pages, kv_len, q_offsets, positions,
                                                         token_positions))
    a = _lib.CacheWriteArgs.from_buffer_copy(template)
    _address(a, k_cache, v_cache, pages, kv_len, q_offsets)
    a.k, a.v = k.data_ptr(), v.data_ptr()
    if positions is not None:
        a.positions, a.token_positions = positions.data_ptr(), token_positions.data_ptr()
    _call(_lib.lib().arthip_cache_write, a, k_cache.device, stream)


def _write_plan(k, v, k_cache, v_cache, pages, kv_len, q_offsets, positions, token_positions) -> bytes:
    a = _lib.CacheWriteArgs()
    _need(k is not None and v is not None and v_cache is not None, "cache_write: k, v and v_cache are needed")
    _need(k.dim() == 3, "cache_write: k must be [T, Hk, D]")
    device = _pages("cache_write", a, k_cache, v_cache, pages, kv_len, q_offsets, k.shape[0])
    for name, t in (("k", k), ("v", v)):
        _check(name, t, device, k_cache.dtype, 3)
        _sizes(name, t)
        _need(t.shape[0] == k.shape[0] and t.shape[1:] == k_cache.shape[2:], f"cache_write: {name} must be [T, Hk, D]")
        _inner(name, t)
        setattr(a, name + "_stride", t.stride()[:2])
    _need((positions is None) == (token_positions is None), "cache_write: positions and token_positions come together")
    if positions is not None:
        a.positions_stride = _per_slot("cache_write", "positions", positions, device, torch.int32, pages.shape[0],
                                       k_cache.shape[2])
        a.slots = positions.shape[2]
        _check("token_positions", token_positions, device, torch.int32, 1)
        _need(token_positions.shape[0] == k.shape[0] and token_positions.is_contiguous(),
              "cache_write: token_positions must be contiguous [T]")
    return bytes(a)


def _scores(name, scale, cap, causal, left) -> tuple:
    return (None if scale is None else _float(f"{name}: scale", scale), _float(f"{name}: cap", cap),
            _bool(f"{name}: causal", causal), None if left is None else _int(f"{name}: left", left))


def _heads(name, a, q, device, k_cache, scores) -> None:
    _check("q", q, device, k_cache.dtype, 3)
    _sizes("q", q)
    _need(q.shape[2] == k_cache.shape[3], f"{name}: q must be [T, Hq, D] of the cache's head_dim")
    _need(k_cache.shape[2] > 0 and q.shape[1] % k_cache.shape[2] == 0,
          f"{name}: q's heads must be a multiple of the cache's")
    _inner("q", q)
    scale, cap, causal, left = scores
    _need(left is None or left >= 0, f"{name}: left counts keys")
    a.q_stride = q.stride()[:2]
    a.q_heads = q.shape[1]
    a.scale = 1.0 / math.sqrt(q.shape[2]) if scale is None else scale
    a.cap, a.causal, a.left = cap, causal, -1 if left is None else left


def _workspace(a, workspace, need, device, stream):
    """The workspace, which has to live until the call is enqueued."""
    if workspace is None and need > 0:
        workspace = _empty((need,), torch.uint8, device, stream)
    elif workspace is not None:
        _need(isinstance(workspace, torch.Tensor), "workspace must be a tensor on a GPU")
        _check("workspace", workspace, device, torch.uint8, 1)
        _inner("workspace", workspace)
    if workspace is not None:
        a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
    return workspace


def paged_attention(q, k_cache, v_cache, pages, kv_len, q_offsets=None, *, scale: float | None = None,
                    cap: float = 0.0, causal: bool = True, left: int | None = None, out=None,
                    return_lse: bool = False, workspace=None, stream=None):
    """softmax(score) V of the new tokens' queries [T, Hq, D] over their sequences' slots;
    see arthip_paged_attention. ``left`` counts the slots before a token's own that it sees
    (None: all); after cache_evict these are not the tokens last written. Returns out, or (out, lse) with lse fp32 [T, Hq]; rows behind the last
    sequence are not written. Without ``workspace`` (uint8) a call makes it."""
    scores = _scores("paged_attention", scale, cap, causal, left)
    key = ("paged", _sig(q), _sig(k_cache), _sig(v_cache), _sig(pages), _sig(kv_len), _sig(q_offsets), scores, _sig(out))
    template, need = _plans.get(key) or _keep(key, _attention_plan(q, k_cache, v_cache, pages, kv_len, q_offsets, scores,
                                                                   out))
    a = _lib.PagedAttentionArgs.from_buffer_copy(template)
    _address(a, k_cache, v_cache, pages, kv_len, q_offsets)
    if out is None:
        out = _like(q, stream)
    a.q, a.out = q.data_ptr(), out.data_ptr()
    lse = None
    if return_lse:
        lse = _empty(q.shape[:2], torch.float32, q.device, stream)
        a.lse = lse.data_ptr()
    workspace = _workspace(a, workspace, need, q.device, stream)
    _call(_lib.lib().arthip_paged_attention, a, q.device, stream)
    return (out, lse) if return_lse else out


def _attention_plan(q, k_cache, v_cache, pages, kv_len, q_offsets, scores, out):
    """(checked arguments without pointers, bytes of workspace)."""
    a = _lib.PagedAttentionArgs()
    _need(v_cache is not None, "paged_attention: v_cache must be a tensor on a GPU")
    _need(q is not None and q.dim() == 3, "paged_attention: q must be [T, Hq, D]")
    device = _pages("paged_attention", a, k_cache, v_cache, pages, kv_len, q_offsets, q.shape[0])
    _heads("paged_attention", a, q, device, k_cache, scores)
    if out is not None:
        _check("out", out, device, q.dtype, 3)
        _need(out.shape == q.shape, "paged_attention: out must have q's shape")
        _inner("out", out)
    a.out_stride = (_contiguous(q.shape) if out is None else out.stride())[:2]
    a.p.pages = a.p.kv_len = 16  # any address: sizes alone decide the workspace
    a.p.q_offsets = None if q_offsets is None else 16
    need = _lib.lib().arthip_paged_attention_workspace(ctypes.byref(a))
    return bytes(a), need


def key_weights(q, k_cache, pages, kv_len, q_offsets, lse, weights, *, decay: float = 1.0, scale: float | None = None,
                cap: float = 0.0, causal: bool = True, left: int | None = None, out=None, workspace=None, stream=None):
    """decay * weights + the attention weight that the new tokens give each cached key,
    summed over the query heads of its key head, fp32 [B, Hk, slots]; see
    arthip_key_weights. ``lse`` is paged_attention's, of the same queries and options; queries
    whose strides reach past 2^30 values in 64 rows (token, head) are refused. out=weights
    adds in place."""
    scores = _scores("key_weights", scale, cap, causal, left)
    decay = _float("key_weights: decay", decay)
    key = ("weights", _sig(q), _sig(k_cache), _sig(pages), _sig(kv_len), _sig(q_offsets), _sig(lse), _sig(weights),
           scores, decay, _sig(out))
    template, need = _plans.get(key) or _keep(key, _weights_plan(q, k_cache, pages, kv_len, q_offsets, lse, weights,
                                                                 scores, decay, out))
    a = _lib.KeyWeightsArgs.from_buffer_copy(template)
    _address(a, k_cache, None, pages, kv_len, q_offsets)
    if out is None:
        out = _like(weights, stream)
    a.q, a.lse, a.weights, a.out = q.data_ptr(), lse.data_ptr(), weights.data_ptr(), out.data_ptr()
    workspace = _workspace(a, workspace, need, q.device, stream)
    _call(_lib.lib().arthip_key_weights, a, q.device, stream)
    return out


def _weights_plan(q, k_cache, pages, kv_len, q_offsets, lse, weights, scores, decay, out):
    """(checked arguments without pointers, bytes of workspace)."""
    a = _lib.KeyWeightsArgs()
    _need(q is not None and q.dim() == 3, "key_weights: q must be [T, Hq, D]")
    device = _pages("key_weights", a, k_cache, None, pages, kv_len, q_offsets, q.shape[0])
    _heads("key_weights", a, q, device, k_cache, scores)
    _check("lse", lse, device, torch.float32, 2)
    _need(lse.shape == q.shape[:2] and lse.is_contiguous(), "key_weights: lse must be contiguous [T, Hq]")
    batch, heads = pages.shape[0], k_cache.shape[2]
    a.weights_stride = _per_slot("key_weights", "weights", weights, device, torch.float32, batch, heads)
    a.slots = weights.shape[2]
    a.out_stride = _contiguous(weights.shape)[:2]
    if out is not None:
        a.out_stride = _per_slot("key_weights", "out", out, device, torch.float32, batch, heads)
        _need(out.shape == weights.shape, "key_weights: out must have weights' shape")
    a.decay = decay
    a.p.pages = a.p.kv_len = 16
    a.p.q_offsets = None if q_offsets is None else 16
    need = _lib.lib().arthip_key_weights_workspace(ctypes.byref(a))
    return bytes(a), need


def cache_evict(k_cache, v_cache, pages, kv_len, weights, keep: int, *, recent: int = 0, first: int = 0,
                positions=None, stream=None):
    """Cuts each sequence to ``keep`` slots a key head, those with the largest weights and
    the protected ones (the last ``recent`` positions, and those below ``first``); see
    arthip_cache_evict. The caches change in place. Returns (kv_len int32 [B], weights
    [B, Hk, slots], kept int32 [B, Hk, keep], positions [B, Hk, slots] or None), all new;
    kept[b, h, s] is the slot that is now in slot s. Pages from the new length on are free."""
    keep, recent = _int("cache_evict: keep", keep), _int("cache_evict: recent", recent)
    first = _int("cache_evict: first", first)
    key = ("evict", _sig(k_cache), _sig(v_cache), _sig(pages), _sig(kv_len), _sig(weights), _sig(positions), keep,
           recent, first)
    template = _plans.get(key) or _keep(key, _evict_plan(k_cache, v_cache, pages, kv_len, weights, positions, keep,
                                                         recent, first))
    a = _lib.CacheEvictArgs.from_buffer_copy(template)
    _address(a, k_cache, v_cache, pages, kv_len, None)
    a.weights = weights.data_ptr()
    device = k_cache.device
    new_len = _like(kv_len, stream)
    new_weights = _like(weights, stream)
    kept = _empty(weights.shape[:2] + (keep,), torch.int32, device, stream)
    a.new_len, a.weights_out, a.kept = new_len.data_ptr(), new_weights.data_ptr(), kept.data_ptr()
    new_positions = None
    if positions is not None:
        new_positions = _like(positions, stream)
        a.positions, a.positions_out = positions.data_ptr(), new_positions.data_ptr()
    _call(_lib.lib().arthip_cache_evict, a, device, stream)
    return new_len, new_weights, kept, new_positions


def _evict_plan(k_cache, v_cache, pages, kv_len, weights, positions, keep, recent, first) -> bytes:
    a = _lib.CacheEvictArgs()
    _need(v_cache is not None, "cache_evict: v_cache must be a tensor on a GPU")
    _need(keep > 0, "cache_evict: keep must be positive")
    device = _pages("cache_evict", a, k_cache, v_cache, pages, kv_len, None, None)
    batch, heads = pages.shape[0], k_cache.shape[2]
    a.weights_stride = _per_slot("cache_evict", "weights", weights, device, torch.float32, batch, heads)
    if positions is not None:
        a.positions_stride = _per_slot("cache_evict", "positions", positions, device, torch.int32, batch, heads)
        _need(positions.shape == weights.shape, "cache_evict: positions must have weights' shape")
    a.slots, a.keep, a.recent, a.first = weights.shape[2], keep, recent, first
    return bytes(a)
