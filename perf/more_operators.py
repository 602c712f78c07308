"""A paged cache of keys and values as timed and checked cases: writing new tokens into
its pages, attention of new tokens over it, the attention weight that each cached key
gathers, and the eviction of the keys that gathered least.

They are what an image or video network that reads a clip piece by piece needs next to
its attention: new patches join the cache, look at it, and the cache is held to a
budget. Keys, values and queries are N(0, 1) like the output of a norm; lengths, pages'
number and masks follow from the case, values and the pages' places from the seed.
``run`` computes the operators in their plain form (elementary torch operations in 32
bits, rounded once at the end) or, where ``own`` is set, with the package's kernels.
"""

import math
import random

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One new token for each of four clips: launch and latency.
        {"name": "write_token", "op": "write", "dtype": "bf16", "b": 4, "n": 1, "mix": False, "lk": 4000, "ragged": True,
         "hk": 8, "d": 128, "page": 16, "positions": True},
        # Eight 1080p frames in 16-pixel patches (68 x 120) enter the cache at once.
        {"name": "write_video", "op": "write", "dtype": "fp16", "b": 1, "n": 65280, "mix": False, "lk": 65280,
         "ragged": False, "hk": 16, "d": 64, "page": 64, "positions": False},
        # One token over a short cache.
        {"name": "attn_token", "op": "attention", "dtype": "fp16", "b": 1, "n": 1, "mix": False, "lk": 777,
         "ragged": False, "hq": 16, "hk": 16, "d": 64, "page": 16, "cap": 0.0, "causal": True, "left": -1},
        # Sixteen sequences of different lengths, one token each.
        {"name": "attn_tokens", "op": "attention", "dtype": "bf16", "b": 16, "n": 1, "mix": False, "lk": 16384,
         "ragged": True, "hq": 32, "hk": 8, "d": 128, "page": 16, "cap": 0.0, "causal": True, "left": -1},
        # The next piece of a prompt over a long cache, with capped scores; an odd length.
        {"name": "attn_piece", "op": "attention", "dtype": "bf16", "b": 1, "n": 256, "mix": False, "lk": 32765,
         "ragged": False, "hq": 16, "hk": 2, "d": 128, "page": 64, "cap": 30.0, "causal": True, "left": -1},
        # What a server sees at one step: some sequences begin, the others go on by a token.
        {"name": "attn_mixed", "op": "attention", "dtype": "fp16", "b": 12, "n": 1537, "mix": True, "lk": 8192,
         "ragged": True, "hq": 32, "hk": 8, "d": 128, "page": 32, "cap": 0.0, "causal": True, "left": -1},
        # The patches of a 1080p frame look at all of it and at four frames before it.
        {"name": "attn_frame", "op": "attention", "dtype": "fp16", "b": 1, "n": 8160, "mix": False, "lk": 40800,
         "ragged": False, "hq": 12, "hk": 12, "d": 64, "page": 48, "cap": 0.0, "causal": False, "left": -1},
        # A whole prompt through pages, each token looking back 4096 keys.
        {"name": "attn_prompt", "op": "attention", "dtype": "bf16", "b": 1, "n": 8192, "mix": False, "lk": 8192,
         "ragged": False, "hq": 32, "hk": 8, "d": 128, "page": 64, "cap": 0.0, "causal": True, "left": 4096},
        # The weight that sixteen tokens leave on their caches' keys.
        {"name": "weights_tokens", "op": "weights", "dtype": "bf16", "b": 16, "n": 1, "mix": False, "lk": 16384,
         "ragged": True, "hq": 32, "hk": 8, "d": 128, "page": 16, "cap": 0.0, "causal": True, "left": -1, "decay": 0.99},
        # The same of a piece of a prompt.
        {"name": "weights_piece", "op": "weights", "dtype": "fp16", "b": 2, "n": 2000, "mix": False, "lk": 8192,
         "ragged": True, "hq": 32, "hk": 8, "d": 128, "page": 64, "cap": 0.0, "causal": True, "left": -1, "decay": 1.0},
        # One token too many in each of sixteen caches.
        {"name": "evict_token", "op": "evict", "dtype": "bf16", "b": 16, "lk": 2049, "ragged": False, "hk": 8, "d": 128,
         "page": 16, "keep": 2048, "recent": 256, "first": 4, "positions": True},
        # Long caches are cut to a quarter.
        {"name": "evict_quarter", "op": "evict", "dtype": "fp16", "b": 4, "lk": 32768, "ragged": True, "hk": 8, "d": 128,
         "page": 64, "keep": 8192, "recent": 1024, "first": 0, "positions": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = max(work(c)["flops"] for c in listed()), max(work(c)["bytes"] for c in listed())
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= limit[0] and w["bytes"] <= limit[1] and _scores(case) <= 2 ** 32:
            return case


def _draw(rng):
    op = rng.choice(["write", "attention", "attention", "attention", "weights", "evict"])
    case = {"op": op, "dtype": rng.choice(["fp16", "bf16"]), "b": 1, "ragged": rng.random() < 0.5}
    hk = rng.choice([1, 2, 4, 8, 12, 16])
    case.update(hk=hk, d=rng.choice([32, 64, 72, 80, 96, 128]), page=rng.choice([16, 32, 48, 64, 128]))
    if op == "evict":
        lk = _log_int(rng, 64, 32768)
        keep = max(8, int(lk * rng.uniform(0.2, 1.0)))
        case.update(b=_log_int(rng, 1, 32), lk=lk, keep=keep, recent=rng.randint(0, keep // 3),
                    first=rng.choice([0, 1, 4]), positions=rng.random() < 0.5)
        return case
    if op != "write":
        case.update(hq=hk * rng.choice([1, 1, 2, 4, 8]), cap=rng.choice([0.0, 0.0, 30.0, 50.0]), causal=rng.random() < 0.8,
                    left=rng.choice([-1, -1, -1, _log_int(rng, 16, 8192)]))
    kind = rng.choice(["token", "piece", "mixed", "prompt"])
    if kind == "token":
        case.update(b=_log_int(rng, 1, 64), n=1, mix=False, lk=_log_int(rng, 16, 32768))
    elif kind == "prompt":
        n = _log_int(rng, 16, 8192)
        case.update(b=rng.randint(1, 4), n=n, mix=False, lk=n, ragged=False)
    else:
        lk = _log_int(rng, 64, 32768)
        case.update(b=rng.randint(1, 12), lk=lk, n=_log_int(rng, 2, min(2048, lk)), mix=kind == "mixed")
    if op == "weights":
        case["decay"] = rng.choice([1.0, 0.99, 0.5])
    if op == "write":
        case["positions"] = rng.random() < 0.5
    return case


# -- geometry: what follows from the case alone ----------------------------------------

def _lengths(case):
    """Keys of each sequence, its new tokens among them."""
    r = random.Random(case["lk"] * 31 + case["b"])
    low = 0.125 if case["op"] != "evict" else 0.5
    lens = [max(1, int(case["lk"] * (1.0 if i == 0 or not case["ragged"] else r.uniform(low, 1.0))))
            for i in range(case["b"])]
    return [max(a, n) for a, n in zip(lens, _new(case))]


def _new(case):
    """New tokens of each sequence."""
    if case["op"] == "evict":
        return [0] * case["b"]
    if not case["mix"]:
        return [case["n"]] * case["b"]
    r = random.Random(case["n"] * 13 + case["b"])
    return [case["n"] if i == 0 else 1 if i % 3 else _log_int(r, 2, case["n"]) for i in range(case["b"])]


def _size(case):
    """Slots that the weights and positions have room for: some more than are in use."""
    return max(_lengths(case)) + 63


def _visible(case):
    """Pairs of a new token and a key that it sees, summed over the batch."""
    total = 0
    for lk, n in zip(_lengths(case), _new(case)):
        place = lk - n + np.arange(n, dtype=np.int64)
        hi = np.minimum(lk, place + 1) if case["causal"] else np.full(n, lk)
        lo = np.maximum(0, place - case["left"]) if case["left"] >= 0 else np.zeros(n, dtype=np.int64)
        total += int(np.sum(hi - lo))
    return total


def _scores(case):
    """Scores of the plain form, which pads the batch."""
    if case["op"] not in ("attention", "weights"):
        return 0
    return case["b"] * case["hq"] * max(_new(case)) * max(_lengths(case))


def _keys_read(case):
    """Keys that some new token sees."""
    total = 0
    for lk, n in zip(_lengths(case), _new(case)):
        total += min(lk, n + case["left"]) if case["left"] >= 0 else lk
    return total


def work(case):
    row = case["hk"] * case["d"] * 2
    if case["op"] == "write":
        t = sum(_new(case))
        return {"bytes": 4 * t * row + (4 * t * (1 + case["hk"]) if case["positions"] else 0), "flops": 0}
    if case["op"] == "evict":
        # Every weight is looked at and the kept ones written; a row moves for every slot that is
        # evicted below the budget. With weights in no order and none protected these are a share
        # of (n - keep) / n of the budget's slots.
        lens, keep = _lengths(case), case["keep"]
        arrays = 2 if case["positions"] else 1
        small = sum(case["hk"] * 4 * (arrays * (n + min(n, keep)) + min(n, keep)) for n in lens)
        moved = sum(keep * max(0, n - keep) / n for n in lens)
        return {"bytes": small + 4 * moved * row, "flops": 0}
    t, d = sum(_new(case)), case["d"]
    q = t * case["hq"] * d * 2
    if case["op"] == "attention":
        return {"bytes": 2 * q + 2 * _keys_read(case) * row + 4 * t * case["hq"],
                "flops": 4 * d * case["hq"] * _visible(case)}
    return {"bytes": q + _keys_read(case) * row + 4 * t * case["hq"] + 8 * case["hk"] * sum(_lengths(case)),
            "flops": 2 * d * case["hq"] * _visible(case)}


# -- inputs ----------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    b, hk, d, page = case["b"], case["hk"], case["d"], case["page"]
    lens, new = _lengths(case), _new(case)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dt)

    def ints(values):
        return torch.from_numpy(np.asarray(values, dtype=np.int32)).cuda()

    counts = [-(-n // page) for n in lens]
    pool = sum(counts) + 3  # some pages belong to nobody
    places = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    width = max(counts) + 1
    pages = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        pages[i, :n] = places[at:at + n]
        at += n
    st = {"case": case, "pages": pages, "kv_len": ints(lens), "k_cache": normal(pool, page, hk, d),
          "v_cache": normal(pool, page, hk, d)}
    if case["op"] != "evict":
        st["offsets"] = ints(np.concatenate([[0], np.cumsum(new)]))
    size, t = _size(case), sum(new)
    if case["op"] == "write":
        st["k"], st["v"] = normal(t, hk, d), normal(t, hk, d)
        if case["positions"]:
            st["positions"] = torch.full((b, hk, size), -1, dtype=torch.int32, device="cuda")
            st["token_positions"] = ints(np.concatenate([np.arange(n) + 5000 + 7 * i for i, n in enumerate(new)]))
    elif case["op"] == "evict":
        # Few keys gather most of the weight.
        st["weights"] = torch.randn(b, hk, size, generator=g, device="cuda").mul_(2.0).exp_()
        if case["positions"]:
            # Caches that have been cut before: slots in no order of time, positions with gaps.
            order = torch.rand(b, hk, size, generator=g, device="cuda").argsort(-1)
            st["positions"] = (order * 3 + 11).to(torch.int32)
    else:
        st["q"] = normal(t, case["hq"], d)
        if case["op"] == "weights":
            st["weights"] = torch.rand(b, hk, size, generator=g, device="cuda")
            st["lse"] = _plain_attention(case, st)[1]
    return st


# -- one pass --------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return {"write": _own_write, "attention": _own_attention, "weights": _own_weights,
                "evict": _own_evict}[case["op"]](case, state)
    return {"write": _plain_write, "attention": _plain_attention, "weights": _plain_weights,
            "evict": _plain_evict}[case["op"]](case, state)


def _own_write(case, st):
    from arthip_amd import paged
    more = {}
    if case["positions"]:
        more = {"positions": st["positions"], "token_positions": st["token_positions"]}
    paged.cache_write(st["k"], st["v"], st["k_cache"], st["v_cache"], st["pages"], st["kv_len"], st["offsets"], **more)
    return (st["k_cache"], st["v_cache"]) + ((st["positions"],) if case["positions"] else ())


def _view(case):
    return {"cap": case["cap"], "causal": case["causal"], "left": case["left"] if case["left"] >= 0 else None}


def _own_attention(case, st):
    from arthip_amd import paged
    return paged.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["pages"], st["kv_len"], st["offsets"],
                                 return_lse=True, **_view(case))


def _own_weights(case, st):
    from arthip_amd import paged
    return paged.key_weights(st["q"], st["k_cache"], st["pages"], st["kv_len"], st["offsets"], st["lse"],
                             st["weights"], decay=case["decay"], **_view(case))


def _own_evict(case, st):
    from arthip_amd import paged
    kept = paged.cache_evict(st["k_cache"], st["v_cache"], st["pages"], st["kv_len"], st["weights"], case["keep"],
                             recent=case["recent"], first=case["first"],
                             positions=st["positions"] if case["positions"] else None)
    return (st["k_cache"], st["v_cache"]) + tuple(x for x in kept if x is not None)


def _owners(st, t):
    """(sequence, slot) of each new token."""
    token = torch.arange(t, device="cuda")
    seq = torch.searchsorted(st["offsets"][1:].long(), token, right=True)
    new = st["offsets"][1:] - st["offsets"][:-1]
    return seq, (st["kv_len"] - new)[seq] + token - st["offsets"][seq]


def _plain_write(case, st):
    seq, slot = _owners(st, st["k"].shape[0])
    page = st["pages"][seq, slot // case["page"]].long()
    st["k_cache"][page, slot % case["page"]] = st["k"]
    st["v_cache"][page, slot % case["page"]] = st["v"]
    if not case["positions"]:
        return st["k_cache"], st["v_cache"]
    st["positions"][seq, :, slot] = st["token_positions"][:, None].expand(-1, case["hk"])
    return st["k_cache"], st["v_cache"], st["positions"]


def _gathered(cache, st, heads):
    """[B, heads, pages * page, D] in 32 bits."""
    x = cache[st["pages"].clamp(min=0).long()][:, :, :, heads]
    return x.flatten(1, 2).float().transpose(1, 2).contiguous()


def _padded(case, st):
    """Rows of the new tokens in [B, longest], and what they see (those that fill up: nothing)."""
    first = st["offsets"][:-1].long()
    new = st["offsets"][1:].long() - first
    i = torch.arange(max(_new(case)), device="cuda")
    live = i < new[:, None]
    rows = torch.where(live, first[:, None] + i, 0)
    j = torch.arange(st["pages"].shape[1] * case["page"], device="cuda")
    place = (st["kv_len"].long() - new)[:, None] + i
    sees = live[..., None] & (j < st["kv_len"][:, None, None])
    if case["causal"]:
        sees = sees & (j <= place[..., None])
    if case["left"] >= 0:
        sees = sees & (j >= place[..., None] - case["left"])
    return rows, sees


def _plain_scores(case, st, rows, sees, heads):
    group = case["hq"] // case["hk"]
    b, lq = rows.shape
    h0, h1 = heads.start, heads.stop
    q = st["q"][:, h0 * group:h1 * group].float()[rows]  # [B, Lq, heads, D]
    q = q.unflatten(2, (h1 - h0, group)).permute(0, 2, 3, 1, 4).reshape(b * (h1 - h0), group * lq, case["d"])
    k = _gathered(st["k_cache"], st, heads).flatten(0, 1).transpose(1, 2).contiguous()
    s = torch.bmm(q, k) * (1 / math.sqrt(case["d"]))
    if case["cap"] > 0:
        s = case["cap"] * torch.tanh(s / case["cap"])
    return s.reshape(b, h1 - h0, group, lq, -1).masked_fill(~sees[:, None, None], -math.inf)


def _head_steps(case):
    """Ranges of key heads whose scores fit into some GiB."""
    one = case["b"] * (case["hq"] // case["hk"]) * max(_new(case)) * (max(_lengths(case)) + 2 * case["page"])
    step = max(1, min(case["hk"], 2 ** 30 // one))
    return [slice(h, min(case["hk"], h + step)) for h in range(0, case["hk"], step)]


def _plain_attention(case, st):
    rows, sees = _padded(case, st)
    seq, _ = _owners(st, st["q"].shape[0])
    index = torch.arange(seq.numel(), device="cuda") - st["offsets"][seq]
    group = case["hq"] // case["hk"]
    out = torch.empty_like(st["q"])
    lse = torch.empty(st["q"].shape[:2], device="cuda")
    for heads in _head_steps(case):
        s = _plain_scores(case, st, rows, sees, heads)
        b, n, _, lq, lk = s.shape
        top = s.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        v = _gathered(st["v_cache"], st, heads)
        o = torch.bmm(p.reshape(b * n, group * lq, lk), v.flatten(0, 1)).reshape(b, n, group, lq, -1)
        o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)
        h = slice(heads.start * group, heads.stop * group)
        part = (torch.log(total) + top)[..., 0].permute(0, 3, 1, 2).flatten(2, 3)
        out[:, h] = o[seq, index].to(out.dtype)
        lse[:, h] = part[seq, index]
    return out, lse


def _plain_weights(case, st):
    rows, sees = _padded(case, st)
    group = case["hq"] // case["hk"]
    size = st["weights"].shape[2]
    slot = torch.arange(size, device="cuda")
    new = st["offsets"][1:] - st["offsets"][:-1]
    old = slot < (st["kv_len"] - new)[:, None]
    out = torch.where(old[:, None], case["decay"] * st["weights"], 0.0)
    for heads in _head_steps(case):
        s = _plain_scores(case, st, rows, sees, heads)
        b, n, _, lq, lk = s.shape
        lse = st["lse"][:, heads.start * group:heads.stop * group][rows].unflatten(2, (n, group)).permute(0, 2, 3, 1)
        p = torch.where(s == -math.inf, 0.0, torch.exp(s - lse[..., None]))
        used = min(size, lk)
        out[:, heads, :used] += p.sum((2, 3))[..., :used]
    return out


def _plain_evict(case, st):
    keep, size = case["keep"], st["weights"].shape[2]
    slot = torch.arange(size, device="cuda")
    n = st["kv_len"].long()[:, None, None]
    live = slot < n
    place = st["positions"].long() if case["positions"] else slot.expand_as(st["weights"])
    newest = torch.where(live, place, -1).amax(-1, keepdim=True)
    safe = (place > newest - case["recent"]) | (place < case["first"])
    key = torch.where(safe, math.inf, st["weights"]).masked_fill(~live, -math.inf)
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    chosen = torch.zeros_like(live.expand_as(key)).scatter(-1, order[..., :keep], True) & live
    # Chosen slots past the budget, in order, go to the others below it, in order.
    movers = torch.where(chosen & (slot >= keep), slot, size).sort(-1).values
    holes = ~chosen[..., :keep]
    rank = (holes.cumsum(-1) - 1).clamp(min=0)
    kept = torch.where(holes, movers.gather(-1, rank), slot[:keep])
    kept = torch.where(slot[:keep] < n, kept, -1)
    source = kept.clamp(min=0)
    target = torch.where(kept < 0, 0, slot[:keep])
    seq = torch.arange(case["b"], device="cuda")[:, None, None]
    head = torch.arange(case["hk"], device="cuda")[:, None]
    pages = st["pages"].long()
    for cache in (st["k_cache"], st["v_cache"]):
        rows = cache[pages[seq, source // case["page"]], source % case["page"], head]
        cache[pages[seq, target // case["page"]], target % case["page"], head] = rows
    weights = torch.zeros_like(st["weights"])
    weights[..., :keep] = torch.where(kept < 0, 0.0, st["weights"].gather(-1, source))
    got = st["k_cache"], st["v_cache"], st["kv_len"].clamp(max=keep), weights, kept.to(torch.int32)
    if not case["positions"]:
        return got
    positions = torch.full_like(st["positions"], -1)
    positions[..., :keep] = torch.where(kept < 0, -1, st["positions"].gather(-1, source))
    return got + (positions,)


# -- the definitions in 64 bits ---------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"write": _exact_write, "attention": _exact_attention, "weights": _exact_weights,
            "evict": _exact_evict}[case["op"]](case, st)


def _places(case, st, i):
    """Rows of sequence i's slots in the flattened pool."""
    n = _lengths(case)[i]
    table = np.asarray(st["pages"][i].cpu(), dtype=np.int64)
    slots = np.arange(n)
    return torch.from_numpy(table[slots // case["page"]] * case["page"] + slots % case["page"]).cuda()


def _exact_write(case, st):
    k, v = st["k_cache"].double(), st["v_cache"].double()
    t = 0
    for i, n in enumerate(_new(case)):
        at = _places(case, st, i)[-n:]
        k.flatten(0, 1)[at] = st["k"][t:t + n].double()
        v.flatten(0, 1)[at] = st["v"][t:t + n].double()
        if case["positions"]:
            first = _lengths(case)[i] - n
            st["positions"][i, :, first:first + n] = st["token_positions"][t:t + n]
        t += n
    return (k, v) + ((st["positions"],) if case["positions"] else ())


def _exact_blocks(case, st):
    """(sequence, head, first row, its rows' hidden-masked scores in 64 bits), piece by piece."""
    t, group = 0, case["hq"] // case["hk"]
    for i, (lk, n) in enumerate(zip(_lengths(case), _new(case))):
        at = _places(case, st, i)
        key = torch.arange(lk, device="cuda")
        for h in range(case["hq"]):
            k = st["k_cache"].flatten(0, 1)[at, h // group].double().T.contiguous()
            step = max(1, 2 ** 27 // lk)
            for r in range(0, n, step):
                m = min(step, n - r)
                s = torch.mm(st["q"][t + r:t + r + m, h].double(), k).div_(math.sqrt(case["d"]))
                if case["cap"] > 0:
                    s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
                ahead = key - (lk - n + r + torch.arange(m, device="cuda"))[:, None]
                if case["causal"]:
                    s.masked_fill_(ahead > 0, -math.inf)
                if case["left"] >= 0:
                    s.masked_fill_(ahead < -case["left"], -math.inf)
                yield i, h, at, t + r, s
        t += n


def _exact_attention(case, st):
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(st["q"].shape[:2], dtype=torch.float64, device="cuda")
    group = case["hq"] // case["hk"]
    for i, h, at, row, s in _exact_blocks(case, st):
        total = torch.logsumexp(s, -1)
        lse[row:row + s.shape[0], h] = total
        v = st["v_cache"].flatten(0, 1)[at, h // group].double()
        out[row:row + s.shape[0], h] = torch.mm(s.sub_(total[:, None]).exp_(), v)
    return out, lse


def _exact_weights(case, st):
    out = torch.zeros(st["weights"].shape, dtype=torch.float64, device="cuda")
    for i, (lk, n) in enumerate(zip(_lengths(case), _new(case))):
        out[i, :, :lk - n] = st["weights"][i, :, :lk - n].double() * case["decay"]
    group = case["hq"] // case["hk"]
    for i, h, _, row, s in _exact_blocks(case, st):
        s.sub_(st["lse"][row:row + s.shape[0], h].double()[:, None])
        out[i, h // group, :s.shape[1]] += s.exp_().sum(0)
    return out


def _exact_evict(case, st):
    keep = case["keep"]
    old = st["weights"].cpu().numpy()
    weights, kept = np.zeros_like(old), np.full(old.shape[:2] + (keep,), -1, dtype=np.int32)
    positions = place = None
    if case["positions"]:
        place = st["positions"].cpu().numpy().astype(np.int64)
        positions = np.full_like(place, -1, dtype=np.int32)
    k, v = st["k_cache"].double(), st["v_cache"].double()
    for i, n in enumerate(_lengths(case)):
        at = _places(case, st, i)
        for h in range(case["hk"]):
            time = place[i, h, :n] if case["positions"] else np.arange(n)
            safe = (time >= time.max() - case["recent"] + 1) | (time < case["first"])
            ranked = np.lexsort((np.arange(n), -old[i, h, :n], ~safe))
            stay = np.sort(ranked[:keep])
            map_ = np.arange(min(n, keep))
            gone = np.setdiff1d(map_, stay)
            map_[gone] = stay[stay >= keep]
            kept[i, h, :map_.size] = map_
            weights[i, h, :map_.size] = old[i, h, map_]
            if case["positions"]:
                positions[i, h, :map_.size] = time[map_]
            if gone.size:
                to, source = at[torch.from_numpy(gone).cuda()], at[torch.from_numpy(map_[gone]).cuda()]
                for x in (k, v):
                    x.flatten(0, 1)[to, h] = x.flatten(0, 1)[source, h]
    lens = torch.tensor(_lengths(case), dtype=torch.int32).clamp(max=keep)
    got = k, v, lens, torch.from_numpy(weights).double(), torch.from_numpy(kept)
    return got + ((torch.from_numpy(positions),) if case["positions"] else ())
