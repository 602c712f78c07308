"""The paged cache from its definitions, in float64 on the CPU, with the error that kernels
which sum in fp32 and round their results once may show. E is the unit roundoff of fp32.

A ``Cache`` holds random pages, in a pool whose slots that nobody uses are NaN."""

from __future__ import annotations

import math

import numpy as np
import torch

from tests import transformer_reference as ref

E = ref.E


class Cache:
    """Sequences of (new tokens, slots in use), their pages shuffled in the pool."""

    def __init__(self, seqs, hk, d, dtype, page=16, seed=0, heads_first=False, spare=3, room=1):
        g = torch.Generator().manual_seed(seed)
        self.g, self.page, self.hk, self.d, self.dtype = g, page, hk, d, dtype
        self.n = [s[0] for s in seqs]
        self.len = [s[1] for s in seqs]
        counts = [-(-x // page) for x in self.len]
        pool = sum(counts) + spare
        order = torch.randperm(pool, generator=g).tolist()
        # Entries past a sequence's pages name no page, or one of nobody's.
        table = torch.full((len(seqs), max(counts, default=0) + room), -1, dtype=torch.int32)
        for i, c in enumerate(counts):
            for j in range(c):
                table[i, j] = order.pop()
        if order and table.shape[1] > 0 and counts and counts[0] < table.shape[1]:
            table[0, -1] = order[0]
        shape = (pool, hk, page, d) if heads_first else (pool, page, hk, d)
        k, v = (torch.full(shape, math.nan, dtype=dtype) for _ in "kv")
        if heads_first:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        self.k, self.v, self.table = k, v, table
        for i, n in enumerate(self.len):
            for cache in (k, v):
                self.put(cache, i, range(n), torch.randn(n, hk, d, generator=g).to(dtype))
        self.offsets = torch.tensor([0] + list(np.cumsum(self.n)), dtype=torch.int32)
        self.kv_len = torch.tensor(self.len, dtype=torch.int32)

    def put(self, cache, i, slots, rows):
        for s, row in zip(slots, rows):
            page = int(self.table[i, s // self.page])
            if 0 <= page < cache.shape[0]:
                cache[page, s % self.page] = row

    def rows(self, cache, i, n):
        """[n, Hk, D] of sequence i's slots; pages outside the pool are zeros."""
        out = torch.zeros(n, *cache.shape[2:], dtype=cache.dtype)
        for s in range(n):
            page = int(self.table[i, s // self.page])
            if 0 <= page < cache.shape[0]:
                out[s] = cache[page, s % self.page]
        return out

    def normal(self, *shape, dtype=None, std=1.0):
        return (torch.randn(*shape, generator=self.g) * std).to(dtype or self.dtype)

    def cuda(self):
        """(k, v, pages, kv_len, q_offsets) on the GPU; the pool keeps its strides."""
        return self.k.cuda(), self.v.cuda(), self.table.cuda(), self.kv_len.cuda(), self.offsets.cuda()


def attention(cache, q, *, scale=None, cap=0.0, causal=True, left=None):
    """((out, tolerance), (lse, tolerance)) of the rows that belong to a sequence. Parts of a row tile
    join with a few more fp32 roundings each than a single walk has; there are at most a quarter as
    many parts as tiles of 32 keys, which the bound's lk E holds with room. A token that sees a NaN
    score has a sum that is NaN, and so has its output (ref.attention leaves 0 there, as it asks whether
    the sum is positive)."""
    outs, lses = [], []
    for i, (n, lk) in enumerate(zip(cache.n, cache.len)):
        if n == 0:
            continue
        mine = q[int(cache.offsets[i]):int(cache.offsets[i]) + n]
        k, v = cache.rows(cache.k, i, lk), cache.rows(cache.v, i, lk)
        out, lse = ref.attention(mine[None], k[None], v[None], scale=scale, cap=cap, causal=causal,
                                 window=(left, None))
        outs.append([torch.where(torch.isnan(lse[0])[0].T[..., None], math.nan, out[0][0]), out[1][0]])
        lses.append([x[0].T for x in lse])
    if not outs:
        return ((torch.zeros(0, *q.shape[1:]).double(),) * 2, (torch.zeros(0, q.shape[1]).double(),) * 2)
    return tuple(torch.cat(x) for x in zip(*outs)), tuple(torch.cat(x) for x in zip(*lses))


def weights(cache, q, lse, old, *, decay=1.0, scale=None, cap=0.0, causal=True, left=None):
    """(out, tolerance). A term exp(s - lse) is off by its score's error (as in attention: D E of the
    sum of the products' absolutes and some roundings, 2^-20 of the cap), the roundings of its exponent
    (of s and lse in the base of 2, 4 E of each) and the exponential's 2^-21; N terms add up N E."""
    batch, hk, slots = old.shape
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    group = q.shape[1] // hk
    out, tol = torch.zeros(old.shape, dtype=torch.float64), torch.zeros(old.shape, dtype=torch.float64)
    for i, (n, lk) in enumerate(zip(cache.n, cache.len)):
        start = lk - n
        kept = max(0, min(start, slots))
        if decay != 0:
            out[i, :, :kept] = decay * old[i, :, :kept].double()
        tol[i] = 3 * E * out[i].abs()
        see, _ = ref.visible(1, n, lk, causal=causal, window=(left, None))
        k = cache.rows(cache.k, i, lk).double()
        used = min(lk, slots)
        first = int(cache.offsets[i])
        for h in range(q.shape[1]):
            q64, kh = q[first:first + n, h].double(), k[:, h // group]
            s = torch.matmul(q64, kh.T) * scale
            d = q.shape[2] * E * abs(scale) * torch.matmul(q64.abs(), kh.abs().T) + 8 * E * s.abs()
            if cap > 0:
                s = cap * torch.tanh(s / cap)
                d = d + cap * 2.0 ** -20
            base = lse[first:first + n, h].double()[:, None]
            p = torch.where(see[0] & (base > -math.inf), torch.exp(s - base), 0.0)
            p = torch.where(see[0], p, 0.0)
            err = d + 2.0 ** -20 + 4 * E * base.nan_to_num(0, 0, 0).abs()
            out[i, h // group, :used] += p.sum(0)[:used]
            tol[i, h // group, :used] += (p * (err + (n * group + 4) * E)).sum(0)[:used]
    return out, tol + E * out.abs()


def evict(cache, old, keep, *, recent=0, first=0, positions=None):
    """Changes the cache's pools; (kv_len, weights, kept, positions), all exact."""
    batch, hk, slots = old.shape
    new_len = torch.tensor([min(x, slots, keep) for x in cache.len], dtype=torch.int32)
    out = torch.zeros_like(old)
    kept = torch.full((batch, hk, keep), -1, dtype=torch.int32)
    places = None if positions is None else torch.full_like(positions, -1)
    for i, lk in enumerate(cache.len):
        n = min(lk, slots)
        rows = {id(c): cache.rows(c, i, n) for c in (cache.k, cache.v)}
        for h in range(hk):
            w = old[i, h, :n].tolist()
            place = list(range(n)) if positions is None else positions[i, h, :n].tolist()
            newest = max(place, default=0)

            def rank(s):
                safe = place[s] > newest - recent or place[s] < first
                return (not safe, math.isnan(w[s]) and not safe, 0.0 if safe or math.isnan(w[s]) else -w[s], s)

            stay = sorted(sorted(range(n), key=rank)[:keep])
            gone = [s for s in range(min(n, keep)) if s not in set(stay)]
            now = list(range(min(n, keep)))
            for to, of in zip(gone, [s for s in stay if s >= keep]):
                now[to] = of
                pages = [int(cache.table[i, s // cache.page]) for s in (to, of)]
                if all(0 <= p < cache.k.shape[0] for p in pages):
                    for c in (cache.k, cache.v):
                        c[pages[0], to % cache.page, h] = rows[id(c)][of, h]
            if now:
                kept[i, h, :len(now)] = torch.tensor(now, dtype=torch.int32)
                out[i, h, :len(now)] = old[i, h, now]
                if positions is not None:
                    places[i, h, :len(now)] = positions[i, h, now]
    return new_len, out, kept, places
