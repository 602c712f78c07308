"""The transformer operators from their definitions, in float64 on the CPU, with the
error that a kernel which sums in fp32 and rounds its results once may show.

Every function takes tensors of the kernels' types and returns (result, tolerance)
pairs, elementwise. u is the unit roundoff of the result's type, E that of fp32."""

from __future__ import annotations

import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}  # half the least subnormal
E = 2.0 ** -24


def rope(x, pos, axis, freqs, pairs=False, inverse=False):
    """[B, L, H, D] by positions [axes, B, L]. The angle is exact to fp32 (2^-25 turns),
    sine and cosine to about 2 E, the two products and their sum add 2 E: 8 E of
    |a| + |b| covers them with 2 pi 2^-25 < 4 E for the angle."""
    n = len(freqs)
    w = torch.tensor(freqs, dtype=torch.float64)
    angle = pos.double().cpu()[torch.tensor(axis)].permute(1, 2, 0) * w
    if inverse:
        angle = -angle
    cos, sin = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
    x64 = x.double().cpu()
    out, tol = x64.clone(), torch.zeros_like(x64)
    first = slice(0, 2 * n, 2) if pairs else slice(0, n)
    second = slice(1, 2 * n, 2) if pairs else slice(n, 2 * n)
    a, b = x64[..., first], x64[..., second]
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    spread = (a.abs() + b.abs()) * 12 * E
    u = UNIT[x.dtype]
    tol[..., first] = u * out[..., first].abs() + spread + TINY[x.dtype]
    tol[..., second] = u * out[..., second].abs() + spread + TINY[x.dtype]
    return out, tol


def _norm(x, err, kind, weight, bias, eps):
    """A norm of x that carries an absolute error err. Means of n values summed in a
    tree of fp32 sums are off by at most 24 E of the largest value (a thread adds up to
    32 values of its own, then 10 levels; their errors average, 24 is not reached)."""
    if kind in (None, "none"):
        return x, err
    top = x.abs().amax(-1, keepdim=True)
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
        err = err + err.amax(-1, keepdim=True) + 26 * E * top
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    w = 1.0 if weight is None else weight.double().cpu()
    b = torch.zeros(()) if bias is None else bias.double().cpu()
    y = x * r
    # d(x r) = r dx + x dr, |dr / r| <= r mean|dx| sqrt(n).. <= r max|dx| + 24 E
    err = r * err + y.abs() * (r * err.amax(-1, keepdim=True) + 32 * E)
    out = y * w + b
    return out, err * (w if weight is None else w.abs()) + 2 * E * out.abs() + 2 * E * b.abs()


def gated_norm(residual, y=None, *, post=None, post_weight=None, post_bias=None, gate=None,
               gate_act="none", residual_scale=1.0, branch_scale=1.0, pre=None, pre_weight=None,
               pre_bias=None, mod_scale=None, mod_shift=None, eps=1e-6, dtype=None):
    dtype = dtype or (residual.dtype if y is None else y.dtype)
    r = residual.double().cpu() * residual_scale
    err = 2 * E * r.abs()
    if y is not None:
        y64 = y.double().cpu()
        n, nerr = _norm(y64, torch.zeros_like(y64), post, post_weight, post_bias, eps)
        g = torch.ones((), dtype=torch.float64) if gate is None else gate.double().cpu()
        act = {"none": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh,
               "silu": torch.nn.functional.silu}[gate_act]
        a = act(g)
        # The hardware exponential and its argument: 2^-21 relative for gates below 16.
        gerr = (2.0 ** -20 if gate_act != "none" else 0.0) * a.abs() + 2 * E * a.abs()
        term = branch_scale * a * n
        err = err + abs(branch_scale) * (gerr * n.abs() + a.abs() * nerr) + 3 * E * (term.abs() + r.abs())
        r = r + term
    h, herr = _norm(r, err, pre, pre_weight, pre_bias, eps)
    if mod_scale is not None:
        m = 1 + mod_scale.double().cpu()
        h, herr = h * m, herr * m.abs() + 2 * E * (h * m).abs() + 2 * E * h.abs()
    if mod_shift is not None:
        h = h + mod_shift.double().cpu()
        herr = herr + 2 * E * h.abs() + 2 * E * mod_shift.double().cpu().abs()
    ru, hu = UNIT[residual.dtype], UNIT[dtype]
    return (r, err + ru * (r.abs() + err) + TINY[residual.dtype]), \
        (h, herr + hu * (h.abs() + herr) + TINY[dtype])


def visible(b, lq, lk, *, causal=False, window=(None, None), q_start=None, kv_len=None,
            prefix=None, docs=None):
    """[B, Lq, Lk] truth values."""
    j = torch.arange(lk)[None, None, :]
    start = torch.full((b,), lk - lq) if q_start is None else q_start.cpu().long()
    p = start[:, None, None] + torch.arange(lq)[None, :, None]
    see = torch.ones(b, lq, lk, dtype=torch.bool)
    left, right = window[0], 0 if causal else window[1]
    if left is not None:
        see &= j >= p - left
    if right is not None:
        see &= j <= p + right
    if prefix is not None:
        see |= j < prefix.cpu().long()[:, None, None]
    if kv_len is not None:
        see &= j < kv_len.cpu().long()[:, None, None]
    if docs is not None:
        dq, dk = (d.cpu() if d.dim() == 2 else d.cpu()[None].expand(b, -1) for d in docs)
        see &= dq[:, :, None] == dk[:, None, :]
    return see, p


def attention(q, k, v, *, scale=None, cap=0.0, causal=False, window=(None, None), q_start=None,
              kv_len=None, prefix=None, docs=None, codes=None, slopes=None, table=None, table_zero=0):
    """((out, tolerance), (lse, tolerance)).

    A score's error d: D products summed in fp32 (D E of the sum of their absolutes; the
    matrix unit's order does not matter for that bound), a few roundings of the scaled
    score and of the bias, the exponential's own 2^-21, the cap's tanh (2^-21 of cap). A
    weight is then off by d of itself, and by u when it is rounded to the type, so
    that the output is off by (u + 2 d) of sum p |v|, and by its own rounding."""
    b, lq, hq, dim = q.shape
    lk, hk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    see, p = visible(b, lq, lk, causal=causal, window=window, q_start=q_start, kv_len=kv_len,
                     prefix=prefix, docs=docs)
    out = torch.zeros(b, lq, hq, dim, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full((b, hq, lq), -math.inf, dtype=torch.float64)
    ltol = torch.zeros_like(lse)
    j = torch.arange(lk)[None, None, :]
    if codes is not None:
        cq, ck = (c.cpu().long() if c.dim() == 2 else c.cpu().long()[None].expand(b, -1) for c in codes)
        diff = cq[:, :, None] - ck[:, None, :]
    else:
        diff = p - j
    u, tiny = UNIT[q.dtype], TINY[q.dtype]
    for h in range(hq):
        q64, k64 = q[:, :, h].double().cpu(), k[:, :, h * hk // hq].double().cpu()
        v64 = v[:, :, h * hk // hq].double().cpu()
        s = torch.matmul(q64, k64.transpose(1, 2)) * scale
        clean = torch.where(see.any(1)[..., None], k64, torch.zeros(())).nan_to_num(0, 0, 0)
        d = dim * E * abs(scale) * torch.matmul(q64.abs(), clean.abs().transpose(1, 2)) + 4 * E * s.nan_to_num(0).abs()
        if cap > 0:
            s = cap * torch.tanh(s / cap)
            d = d + cap * 2.0 ** -20
        if slopes is not None:
            bias = -slopes[h].double().cpu() * diff.abs()
            s = s + bias
            d = d + 4 * E * bias.abs()
        if table is not None:
            bias = table[h].double().cpu()[(diff + table_zero).clamp(0, table.shape[1] - 1)]
            s = torch.where(bias == -math.inf, bias, s + bias)
            d = d + 4 * E * bias.nan_to_num(0, 0, 0).abs()
        s = torch.where(see, s, -math.inf)
        if lk == 0:
            continue
        top = s.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        w = torch.exp(s - top)
        total = w.sum(-1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
        dmax = torch.where(s > -math.inf, d + 4 * E * s.abs(), torch.zeros(())).amax(-1, keepdim=True) \
            + 2.0 ** -20 + 4 * E * top.abs() + lk * E
        hidden = w == 0
        for i in range(b):
            # Hidden keys add nothing, whatever they hold.
            vv = torch.where(hidden[i][..., None], torch.zeros(()), v64[i][None])
            out[i, :, h] = (w[i][..., None] * vv).sum(1)
            a = (w[i][..., None] * vv.abs()).sum(1)
            tol[i, :, h] = u * out[i, :, h].abs() + (u + 2.2 * dmax[i]) * a \
                + tiny * (1 + torch.where(hidden[i][..., None], torch.zeros(()), vv.abs()).sum(1))
        lse[:, h] = (torch.log(total) + top)[..., 0]
        ltol[:, h] = (dmax + 4 * E * lse[:, h, :, None].nan_to_num(0, 0, 0).abs())[..., 0]
    return (out, tol), (lse, ltol)


def check(got, want, name):
    """got within want's tolerance, infinities and NaN where want has them."""
    value, tol = want
    g = got.double().cpu()
    assert g.shape == value.shape, (name, g.shape, value.shape)
    assert torch.equal(torch.isnan(g), torch.isnan(value)), f"{name}: NaN in other places"
    odd = ~torch.isfinite(value) & ~torch.isnan(value)
    assert torch.equal(g[odd], value[odd]), f"{name}: infinities differ"
    ok = torch.isfinite(value)
    over = ((g - value).abs() - tol)[ok]
    if over.numel() and over.max() > 0:
        ratio = ((g - value).abs()[ok] / tol[ok].clamp_min(1e-300)).max()
        raise AssertionError(f"{name}: {int((over > 0).sum())} of {over.numel()} values off, "
                             f"the worst {ratio:.3g} times the tolerance")
