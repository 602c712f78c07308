"""The transformer operators of this package as timed and checked cases: rotary
positions with several axes, attention (tanh cap, distance bias, document and prefix
masks, ragged caches) and the norms around a gated residual.

They are the block of an image or video network: tokens are patches of a frame or of
a clip, grouped by window, frame or document. Activations are N(0, 1) like the output
of a norm; positions, masks and lengths follow from the case, values from the seed.
``run`` computes the operators in their plain form (elementary torch operations in 32
bits, rounded once at the end) or, where ``own`` is set, with the package's kernels.
"""

import math
import random

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
THETA = 10000.0


def listed():
    return [
        # One new token for each of four clips: 40 heads to turn, all launch and latency.
        {"name": "rope_token", "op": "rope", "dtype": "bf16", "b": 4, "grid": "1x1x1", "hq": 32, "hk": 8, "d": 128,
         "sections": "16+24+24", "per_axis": False, "pairs": False, "start": 4000},
        # Eight 1080p frames in 16-pixel patches (68 x 120), each axis with its own
        # frequencies, neighbouring values turned together.
        {"name": "rope_video", "op": "rope", "dtype": "fp16", "b": 1, "grid": "8x68x120", "hq": 16, "hk": 16, "d": 64,
         "sections": "8+12+12", "per_axis": True, "pairs": True, "start": 0},
        # One token a clip through the norms around a block: latency.
        {"name": "norm_token", "op": "norm", "dtype": "bf16", "res": "bf16", "b": 4, "l": 1, "c": 4096, "post": "rms",
         "pre": "rms", "gate": "channel", "act": "none", "mod": False},
        # Two clips of four 1080p frames in a diffusion block: layer norms, a tanh gate
        # and a modulation per clip.
        {"name": "norm_video", "op": "norm", "dtype": "fp16", "res": "fp16", "b": 2, "l": 32640, "c": 1024,
         "post": "layer", "pre": "layer", "gate": "batch", "act": "tanh", "mod": True},
        # An odd width with a residual stream in 32 bits and a sigmoid gate per token.
        {"name": "norm_odd", "op": "norm", "dtype": "bf16", "res": "fp32", "b": 3, "l": 1999, "c": 975, "post": "rms",
         "pre": "rms", "gate": "token", "act": "sigmoid", "mod": False},
        # A long causal prompt with shared key heads and capped scores.
        {"name": "attn_prompt", "op": "attention", "dtype": "bf16", "b": 1, "lq": 8192, "lk": 8192, "hq": 32, "hk": 8,
         "d": 128, "cap": 50.0, "causal": True, "bias": "none", "mask": "none"},
        # Quarter-HD features in 16 x 16 windows with a table of relative positions.
        {"name": "attn_windows", "op": "attention", "dtype": "fp16", "b": 2040, "lq": 256, "lk": 256, "hq": 6, "hk": 6,
         "d": 32, "cap": 0.0, "causal": False, "bias": "table", "mask": "none"},
        # Pictures of different sizes packed into one sequence, one document each.
        {"name": "attn_pictures", "op": "attention", "dtype": "fp16", "b": 1, "lq": 16384, "lk": 16384, "hq": 12,
         "hk": 12, "d": 64, "cap": 0.0, "causal": False, "bias": "none", "mask": "documents"},
        # A condition of some hundred tokens seen by all, then a causal rest; odd lengths.
        {"name": "attn_prefix", "op": "attention", "dtype": "bf16", "b": 2, "lq": 1537, "lk": 1537, "hq": 10, "hk": 10,
         "d": 80, "cap": 0.0, "causal": True, "bias": "none", "mask": "prefix"},
        # One token over a short cache.
        {"name": "attn_token", "op": "attention", "dtype": "fp16", "b": 1, "lq": 1, "lk": 777, "hq": 16, "hk": 16,
         "d": 64, "cap": 0.0, "causal": False, "bias": "none", "mask": "none"},
        # Sixteen sequences of different lengths, one token each, with a slope over the distance.
        {"name": "attn_tokens", "op": "attention", "dtype": "bf16", "b": 16, "lq": 1, "lk": 16384, "hq": 32, "hk": 8,
         "d": 128, "cap": 0.0, "causal": True, "bias": "slope", "mask": "lengths"},
        # The next piece of a prompt over a cache of the earlier ones.
        {"name": "attn_piece", "op": "attention", "dtype": "bf16", "b": 1, "lq": 256, "lk": 32768, "hq": 16, "hk": 2,
         "d": 128, "cap": 30.0, "causal": True, "bias": "none", "mask": "none"},
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
    op = rng.choice(["rope", "norm", "attention", "attention"])
    dtype = rng.choice(["fp16", "bf16"])
    if op == "rope":
        d = rng.choice([32, 64, 72, 80, 96, 128])
        f = rng.choice([d // 2, d // 2, d // 4])
        axes = rng.choice([1, 2, 3])
        cut = sorted(rng.sample(range(1, f), axes - 1))
        sections = "+".join(str(b - a) for a, b in zip([0] + cut, cut + [f]))
        grid = "1x1x1"
        if rng.random() < 0.75:
            grid = f"{rng.randint(1, 8)}x{_log_int(rng, 4, 68)}x{_log_int(rng, 4, 120)}"
        hk = rng.choice([1, 2, 4, 8, 16])
        return {"op": op, "dtype": dtype, "b": rng.randint(1, 4), "grid": grid, "hq": hk * rng.choice([1, 2, 4]),
                "hk": hk, "d": d, "sections": sections, "per_axis": rng.random() < 0.5, "pairs": rng.random() < 0.5,
                "start": rng.choice([0, rng.randint(0, 8000)])}
    if op == "norm":
        return {"op": op, "dtype": dtype, "res": rng.choice([dtype, "fp32"]), "b": rng.randint(1, 4),
                "l": _log_int(rng, 1, 32640), "c": _log_int(rng, 64, 4096), "post": rng.choice(["rms", "layer"]),
                "pre": rng.choice(["rms", "layer"]), "gate": rng.choice(["channel", "batch", "token"]),
                "act": rng.choice(["none", "sigmoid", "tanh"]), "mod": rng.random() < 0.5}
    d = rng.choice([32, 64, 80, 96, 128])
    hk = rng.choice([1, 2, 4, 8, 12])
    hq = hk * rng.choice([1, 1, 2, 4])
    case = {"op": op, "dtype": dtype, "b": 1, "lq": 1, "lk": 1, "hq": hq, "hk": hk, "d": d,
            "cap": rng.choice([0.0, 0.0, 30.0, 50.0]), "causal": False, "bias": "none", "mask": "none"}
    kind = rng.choice(["token", "piece", "prompt", "windows", "pictures"])
    if kind == "token":
        case.update(b=_log_int(rng, 1, 32), lk=_log_int(rng, 64, 32768), causal=True, mask=rng.choice(["none", "lengths"]),
                    bias=rng.choice(["none", "slope"]))
    elif kind == "piece":
        lk = _log_int(rng, 512, 32768)
        case.update(b=rng.randint(1, 2), lk=lk, lq=_log_int(rng, 2, min(512, lk)), causal=True,
                    bias=rng.choice(["none", "slope"]))
    elif kind == "prompt":
        case.update(b=rng.randint(1, 4), lk=_log_int(rng, 64, 8192), causal=True, mask=rng.choice(["none", "prefix"]),
                    bias=rng.choice(["none", "slope"]))
        case["lq"] = case["lk"]
    elif kind == "windows":
        n = rng.randint(7, 16) ** 2
        case.update(b=_log_int(rng, 16, 1024), lq=n, lk=n, bias=rng.choice(["none", "table"]))
    else:
        n = _log_int(rng, 1024, 16384)
        case.update(lq=n, lk=n, mask="documents", causal=rng.random() < 0.3)
    return case


# -- geometry: what follows from the case alone ----------------------------------------

def _grid(case):
    """Tokens along time, height and width."""
    return [int(n) for n in case["grid"].split("x")]


def _sections(case):
    """Turned pairs of each axis."""
    return [int(n) for n in case["sections"].split("+")]


def _positions(case):
    """[3, B, L] int32: time, height and width of each token."""
    t, h, w = _grid(case)
    grid = np.stack(np.meshgrid(np.arange(t), np.arange(h), np.arange(w), indexing="ij")).reshape(3, 1, -1)
    first = case["start"] + 17 * np.arange(case["b"]).reshape(1, -1, 1)
    return (grid + first * np.array([1, 0, 0]).reshape(3, 1, 1) if t * h * w > 1 else grid + first).astype(np.int32)


def _frequencies(case):
    """(axis, frequency) of each turned pair."""
    sections = _sections(case)
    n = sum(sections)
    axis = np.concatenate([np.full(s, a) for a, s in enumerate(sections)])
    if case["per_axis"]:
        freq = np.concatenate([THETA ** (-np.arange(s) / s) for s in sections])
    else:
        freq = THETA ** (-np.arange(n) / n)
    return axis, freq


def _lengths(case):
    """Keys of each sequence; between an eighth of the cache and all of it."""
    r = random.Random(case["lk"] * 31 + case["b"])
    return [max(1, int(case["lk"] * (1.0 if i == 0 else r.uniform(0.125, 1.0)))) for i in range(case["b"])]


def _documents(case):
    """Document of each token: pictures of 64 to 4096 patches, one after the other."""
    r = random.Random(case["lk"] * 17 + 5)
    sizes = []
    while sum(sizes) < case["lk"]:
        sizes.append(_log_int(r, 64, 4096))
    return np.repeat(np.arange(len(sizes)), sizes)[:case["lk"]].astype(np.int32)


def _prefix(case):
    return [max(1, case["lk"] // 5 - 7 * i) for i in range(case["b"])]


def _starts(case):
    """Position of each sequence's first query: the last keys are the queries' own."""
    n = _lengths(case) if case["mask"] == "lengths" else [case["lk"]] * case["b"]
    return [v - case["lq"] for v in n]


def _slopes(case):
    return 2.0 ** (-8.0 * np.arange(1, case["hq"] + 1) / case["hq"])


def _codes(case):
    """Tokens of a square window as one number each; differences of two name their offset."""
    n = math.isqrt(case["lk"])
    y, x = np.divmod(np.arange(case["lk"]), n)
    return (y * (2 * n - 1) + x).astype(np.int32), (2 * n - 1) ** 2, (n - 1) * (2 * n - 1) + (n - 1)


def _visible(case):
    """Pairs of a query and a key that it sees, summed over the batch."""
    lq, total = case["lq"], 0
    for i in range(case["b"]):
        lk = _lengths(case)[i] if case["mask"] == "lengths" else case["lk"]
        hi = np.minimum(lk, _starts(case)[i] + np.arange(lq) + 1) if case["causal"] else np.full(lq, lk)
        if case["mask"] == "prefix":
            hi = np.maximum(hi, _prefix(case)[i])
        if case["mask"] == "documents":
            doc = _documents(case)
            total += int(np.sum(np.minimum(hi, np.searchsorted(doc, doc, "right")) - np.searchsorted(doc, doc, "left")))
        else:
            total += int(hi.sum())
    return total


def _scores(case):
    return case["b"] * case["hq"] * case["lq"] * case["lk"] if case["op"] == "attention" else 0


def work(case):
    size = 2
    if case["op"] == "rope":
        tokens = case["b"] * math.prod(_grid(case))
        values = tokens * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * values * size + tokens * 12, "flops": values * 3}
    if case["op"] == "norm":
        values = case["b"] * case["l"] * case["c"]
        res = 4 if case["res"] == "fp32" else size
        rows = {"channel": 1, "batch": case["b"], "token": case["b"] * case["l"]}[case["gate"]]
        small = rows * case["c"] * size + (2 * case["b"] * case["c"] * size if case["mod"] else 0) + 8 * case["c"]
        return {"bytes": values * (2 * res + 2 * size) + small, "flops": values * 12}
    keys = sum(_lengths(case)) if case["mask"] == "lengths" else case["b"] * case["lk"]
    moved = (2 * case["b"] * case["lq"] * case["hq"] + 2 * keys * case["hk"]) * case["d"] * size
    return {"bytes": moved, "flops": 4 * case["d"] * case["hq"] * _visible(case)}


# -- inputs ----------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, dtype=dt, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    st = {"case": case}
    if case["op"] == "rope":
        b, l, d = case["b"], math.prod(_grid(case)), case["d"]
        st["q"], st["k"] = normal(b, l, case["hq"], d), normal(b, l, case["hk"], d)
        st["pos"] = torch.from_numpy(_positions(case)[:len(_sections(case))]).contiguous().cuda()
        if own:
            from arthip_amd import transformer
            st["plan"] = transformer.RopePlan(_sections(case), theta=THETA, per_axis=case["per_axis"],
                                              pairs=case["pairs"], device="cuda")
        else:
            axis, freq = _frequencies(case)
            st["axis"] = torch.from_numpy(axis).cuda()
            st["freq"] = torch.from_numpy(freq.astype(np.float32)).cuda()
    elif case["op"] == "norm":
        b, l, c = case["b"], case["l"], case["c"]
        st["residual"] = normal(b, l, c, dtype=TYPES[case["res"]], std=2.0)
        st["y"] = normal(b, l, c)
        st["gate"] = {"channel": lambda: normal(c, std=0.5), "batch": lambda: normal(b, 1, c, std=0.5),
                      "token": lambda: normal(b, l, c, std=0.5)}[case["gate"]]()
        for side in ("post", "pre"):
            st[side + "_weight"] = normal(c, dtype=torch.float32, std=0.1, mean=1.0)
            st[side + "_bias"] = normal(c, dtype=torch.float32, std=0.1) if case[side] == "layer" else None
        st["mod_scale"] = normal(b, 1, c, std=0.2) if case["mod"] else None
        st["mod_shift"] = normal(b, 1, c, std=0.2) if case["mod"] else None
    else:
        b, lq, lk, hq, hk, d = (case[n] for n in ("b", "lq", "lk", "hq", "hk", "d"))
        st["q"], st["k"], st["v"] = normal(b, lq, hq, d), normal(b, lk, hk, d), normal(b, lk, hk, d)

        def ints(values):
            return torch.from_numpy(np.asarray(values, dtype=np.int32)).cuda()

        st["kv_len"] = ints(_lengths(case)) if case["mask"] == "lengths" else None
        st["q_start"] = ints(_starts(case)) if case["mask"] == "lengths" else None
        st["prefix"] = ints(_prefix(case)) if case["mask"] == "prefix" else None
        st["docs"] = ints(_documents(case)) if case["mask"] == "documents" else None
        st["slopes"] = torch.from_numpy(_slopes(case).astype(np.float32)).cuda() if case["bias"] == "slope" else None
        if case["bias"] == "table":
            codes, n, st["zero"] = _codes(case)
            st["codes"] = ints(codes)
            st["table"] = normal(hq, n, dtype=torch.float32, std=0.5)
    return st


# -- one pass --------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return {"rope": _own_rope, "norm": _own_norm, "attention": _own_attention}[case["op"]](case, state)
    return {"rope": _plain_rope, "norm": _plain_norm, "attention": _plain_attention}[case["op"]](case, state)


def _own_rope(case, st):
    from arthip_amd import transformer
    return transformer.rope_axes(st["q"], st["k"], st["pos"], st["plan"])


def _own_norm(case, st):
    from arthip_amd import transformer
    return transformer.gated_norm(
        st["residual"], st["y"], post=case["post"], post_weight=st["post_weight"], post_bias=st["post_bias"],
        gate=st["gate"], gate_act=case["act"], branch_scale=0.5, pre=case["pre"], pre_weight=st["pre_weight"],
        pre_bias=st["pre_bias"], mod_scale=st["mod_scale"], mod_shift=st["mod_shift"], eps=1e-6)


def _own_attention(case, st):
    from arthip_amd import transformer
    bias = {}
    if case["bias"] == "slope":
        bias = {"slopes": st["slopes"]}
    elif case["bias"] == "table":
        bias = {"table": st["table"], "table_zero": st["zero"], "codes": (st["codes"], st["codes"])}
    docs = None if st["docs"] is None else (st["docs"], st["docs"])
    return transformer.attention(st["q"], st["k"], st["v"], cap=case["cap"], causal=case["causal"],
                                 kv_len=st["kv_len"], q_start=st["q_start"], prefix=st["prefix"], docs=docs,
                                 return_lse=True, **bias)


def _plain_rope(case, st):
    angle = st["pos"].float()[st["axis"]].permute(1, 2, 0) * st["freq"]
    cos, sin = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
    f = st["freq"].numel()

    def turn(x):
        x32 = x.float()
        if case["pairs"]:
            a, b = x32[..., 0:2 * f:2], x32[..., 1:2 * f:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x32[..., :f], x32[..., f:2 * f]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, x32[..., 2 * f:]], -1).to(x.dtype)

    return turn(st["q"]), turn(st["k"])


def _plain_norm(case, st):
    def norm(x, kind, weight, bias):
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
        return x + bias if kind == "layer" else x

    y = norm(st["y"].float(), case["post"], st["post_weight"], st["post_bias"])
    gate = st["gate"].float()
    if case["act"] == "sigmoid":
        gate = 1 / (1 + torch.exp(-gate))
    elif case["act"] == "tanh":
        gate = torch.tanh(gate)
    res = st["residual"].float() + 0.5 * gate * y
    h = norm(res, case["pre"], st["pre_weight"], st["pre_bias"])
    if case["mod"]:
        h = h * (1 + st["mod_scale"].float()) + st["mod_shift"].float()
    return res.to(st["residual"].dtype), h.to(st["y"].dtype)


def _plain_attention(case, st):
    b, lq, lk, hq, hk, d = (case[n] for n in ("b", "lq", "lk", "hq", "hk", "d"))
    dev, group = st["q"].device, hq // hk
    i = torch.arange(lq, device=dev)[:, None]
    j = torch.arange(lk, device=dev)[None, :]
    start = (st["q_start"] if st["q_start"] is not None else torch.tensor([lk - lq], device=dev))[:, None, None]
    visible = None
    if case["causal"]:
        visible = j <= start + i
        if st["prefix"] is not None:
            visible = visible | (j < st["prefix"][:, None, None])
    if st["kv_len"] is not None:
        live = j < st["kv_len"][:, None, None]
        visible = live if visible is None else visible & live
    if st["docs"] is not None:
        same = st["docs"][:, None] == st["docs"][None, :]
        visible = same if visible is None else visible & same
    out = torch.empty(b, lq, hq, d, dtype=st["q"].dtype, device=dev)
    lse = torch.empty(b, hq, lq, device=dev)
    step = max(1, min(hk, 2 ** 30 // max(1, b * group * lq * lk)))
    for h in range(0, hk, step):
        n = min(step, hk - h)
        q = st["q"][:, :, h * group:(h + n) * group].float().permute(0, 2, 1, 3).reshape(b, n, group * lq, d)
        k = st["k"][:, :, h:h + n].float().permute(0, 2, 3, 1).contiguous()
        v = st["v"][:, :, h:h + n].float().permute(0, 2, 1, 3).contiguous()
        s = (torch.matmul(q, k) * (1 / math.sqrt(d))).reshape(b, n * group, lq, lk)
        if case["cap"] > 0:
            s = case["cap"] * torch.tanh(s / case["cap"])
        if case["bias"] == "slope":
            s = s - st["slopes"][h * group:(h + n) * group, None, None] * (start + i - j).abs().float()[:, None]
        elif case["bias"] == "table":
            offset = st["codes"][:, None] - st["codes"][None, :] + st["zero"]
            s = s + st["table"][h * group:(h + n) * group, offset.long()]
        if visible is not None:
            s = torch.where(visible if visible.dim() == 2 else visible[:, None], s, -math.inf)
        top = s.amax(-1, keepdim=True)
        top = torch.where(top == -math.inf, 0.0, top)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p.reshape(b, n, group * lq, lk), v).reshape(b, n * group, lq, d)
        o = torch.where(total > 0, o / total, 0.0)
        out[:, :, h * group:(h + n) * group] = o.permute(0, 2, 1, 3).to(out.dtype)
        lse[:, h * group:(h + n) * group] = (torch.log(total) + top)[..., 0]
    return out, lse


# -- the definitions in 64 bits ---------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"rope": _exact_rope, "norm": _exact_norm, "attention": _exact_attention}[case["op"]](case, st)


def _exact_rope(case, st):
    axis, freq = _frequencies(case)
    pos = torch.from_numpy(_positions(case).astype(np.float64))
    angle = torch.stack([pos[a] * w for a, w in zip(axis.tolist(), freq.tolist())], -1).cuda()
    unit = torch.polar(torch.ones_like(angle), angle)[:, :, None, :]
    n = freq.size

    def turn(x):
        x = x.double()
        head, tail = x[..., :2 * n], x[..., 2 * n:]
        head = head.unflatten(-1, (n, 2)) if case["pairs"] else head.unflatten(-1, (2, n)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(head.contiguous()) * unit)
        z = z if case["pairs"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), tail], -1)

    return turn(st["q"]), turn(st["k"])


def _exact_norm(case, st):
    def wide(name):
        return None if st[name] is None else st[name].double()

    def norm(x, side):
        second = x.square().mean(-1, keepdim=True)
        if case[side] == "rms":
            return x / (second + 1e-6).sqrt() * wide(side + "_weight")
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        return (x - mean) / (var + 1e-6).sqrt() * wide(side + "_weight") + wide(side + "_bias")

    act = {"none": lambda g: g, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["act"]]
    res = torch.addcmul(wide("residual"), act(wide("gate")), norm(wide("y"), "post"), value=0.5)
    h = norm(res, "pre")
    if case["mod"]:
        h = h + h * wide("mod_scale") + wide("mod_shift")
    return res, h


def _exact_attention(case, st):
    b, lq, lk, hq, hk, d = (case[n] for n in ("b", "lq", "lk", "hq", "hk", "d"))
    out = torch.zeros(b, lq, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(b, hq, lq, dtype=torch.float64, device="cuda")
    key = torch.arange(lk, device="cuda")
    lengths = _lengths(case) if case["mask"] == "lengths" else [lk] * b
    if case["bias"] == "table":
        codes, _, zero = _codes(case)
        codes = torch.from_numpy(codes.astype(np.int64)).cuda()
    if case["mask"] == "documents":
        docs = torch.from_numpy(_documents(case)).cuda()
    items = max(1, min(b, 2 ** 27 // (lq * lk)))
    for b0 in range(0, b, items):
        b1 = min(b, b0 + items)
        place = torch.tensor(_starts(case)[b0:b1], device="cuda")[:, None] + torch.arange(lq, device="cuda")
        keep = (key < torch.tensor(lengths[b0:b1], device="cuda")[:, None])[:, None, :].expand(b1 - b0, lq, lk)
        if case["causal"]:
            first = torch.tensor(_prefix(case)[b0:b1] if case["mask"] == "prefix" else [0] * (b1 - b0), device="cuda")
            keep = keep & ((key <= place[..., None]) | (key < first[:, None, None]))
        if case["mask"] == "documents":
            keep = keep & (docs[None, :, None] == docs[None, None, :])
        for h in range(hq):
            q = st["q"][b0:b1, :, h].double().contiguous()
            k = st["k"][b0:b1, :, h * hk // hq].double().transpose(1, 2).contiguous()
            v = st["v"][b0:b1, :, h * hk // hq].double().contiguous()
            s = torch.bmm(q, k).div_(math.sqrt(d))
            if case["cap"] > 0:
                s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
            if case["bias"] == "slope":
                s -= (2.0 ** (-8.0 * (h + 1) / hq)) * (place[..., None] - key).abs()
            elif case["bias"] == "table":
                s += st["table"][h].double()[codes[:, None] - codes[None, :] + zero]
            s = s.masked_fill(~keep, -math.inf)
            total = torch.logsumexp(s, -1)
            lse[b0:b1, h] = total
            out[b0:b1, :, h] = torch.bmm(s.sub_(total[..., None]).exp_(), v)
    return out, lse
