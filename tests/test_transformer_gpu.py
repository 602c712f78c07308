"""The transformer operators on the GPU against their definitions in float64
(tests/transformer_reference.py, whose tolerances are derived there): types, head
layouts, lengths, masks, strides, streams, graphs and values that are not finite."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from arthip_amd import _lib
from arthip_amd import transformer as tr
from arthip_amd.engine import EngineError
from tests import transformer_reference as ref

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _normal(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


# -- rotary positions ------------------------------------------------------------------

ROPE = [
    # dtype, B, L, Hq, Hk, D, sections, pairs, per_axis, order
    (BF16, 1, 1, 4, 2, 128, (16, 24, 24), False, False, "blocks"),
    (F16, 2, 5, 3, 3, 64, (8, 12, 12), True, True, "blocks"),
    (F16, 1, 33, 32, 8, 128, (16, 24, 24), False, False, "cycle"),
    (BF16, 3, 7, 5, 1, 72, (36,), True, False, "blocks"),
    (F16, 1, 9, 2, 2, 72, (9, 9), False, True, "blocks"),      # half of a head turned
    (F32, 2, 11, 3, 1, 80, (10, 20, 10), False, True, "cycle"),
    (F32, 1, 3, 1, 1, 32, (16,), True, False, "blocks"),
    (BF16, 1, 300, 1, 1, 6, (1, 1), True, True, "blocks"),      # odd counts: single values
    (F16, 1, 4, 2, 1, 2, (1,), False, False, "blocks"),
    (F16, 1, 4, 70, 3, 512, (100, 28), False, False, "blocks"),
    (BF16, 5, 257, 6, 2, 96, (2, 46), True, True, "blocks"),
]


def _rope_case(dtype, b, l, hq, hk, d, sections, seed=0, top=9000):
    g = _gen(seed)
    q, k = _normal(g, b, l, hq, d, dtype=dtype), _normal(g, b, l, hk, d, dtype=dtype)
    pos = torch.randint(-top, top, (len(sections), b, l), generator=g, dtype=torch.int32).cuda()
    return q, k, pos


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dtype,b,l,hq,hk,d,sections,pairs,per_axis,order", ROPE)
def test_rope(dtype, b, l, hq, hk, d, sections, pairs, per_axis, order, inverse):
    q, k, pos = _rope_case(dtype, b, l, hq, hk, d, sections)
    plan = tr.RopePlan(sections, per_axis=per_axis, pairs=pairs, order=order)
    qo, ko = tr.rope_axes(q, k, pos, plan, inverse=inverse)
    for name, x, got in (("q", q, qo), ("k", k, ko)):
        ref.check(got, ref.rope(x, pos, plan.axis, plan.freqs, pairs, inverse), name)


def test_rope_large_positions_keep_their_phase():
    q, k, pos = _rope_case(F32, 1, 64, 2, 1, 64, (16, 16), top=2 ** 31 - 1)
    plan = tr.RopePlan((16, 16))
    qo, _ = tr.rope_axes(q, k, pos, plan)
    ref.check(qo, ref.rope(q, pos, plan.axis, plan.freqs), "q")


@pytest.mark.parametrize("pairs", [False, True])
def test_rope_in_place_strides_and_one_side(pairs):
    """q and k as views of one projection, turned in place; values past the turned ones
    and the rest of the buffer stay."""
    g = _gen(3)
    qkv = _normal(g, 2, 6, 8, 80, dtype=F16)
    want = qkv.clone()
    pos = torch.randint(0, 500, (2, 6), generator=g, dtype=torch.int32).cuda()  # for every batch item
    plan = tr.RopePlan((5, 15), pairs=pairs)
    q, k = qkv[:, :, :4], qkv[:, :, 4:6]
    fresh_q, fresh_k = tr.rope_axes(q, k, pos, plan)
    full = pos[:, None].expand(2, 2, 6)
    ref.check(fresh_q, ref.rope(q, full, plan.axis, plan.freqs, pairs), "q")
    assert torch.equal(qkv, want)
    out = tr.rope_axes(q, None, pos, plan, q_out=q)
    assert out[1] is None and torch.equal(q, fresh_q) and torch.equal(k, want[:, :, 4:6])
    tr.rope_axes(None, k, pos, plan, k_out=k)
    assert torch.equal(k, fresh_k) and torch.equal(qkv[:, :, 6:], want[:, :, 6:])
    # heads first, and an odd element offset
    flat = _normal(g, 2 * 3 * 6 * 40 + 1, dtype=F16)[1:]
    q = flat.view(2, 3, 6, 40).permute(0, 2, 1, 3)
    got, _ = tr.rope_axes(q, None, pos, plan)
    ref.check(got, ref.rope(q, full, plan.axis, plan.freqs, pairs), "permuted")


def test_rope_more_tokens_than_a_launch_takes():
    """An odd number of pairs goes value by value: 2^24 tokens of 255 pairs take 2^32 threads."""
    n, step = 2 ** 24 + 3, 1021
    q, _, pos = _rope_case(F16, 1, step, 1, 1, 510, (255,))
    plan = tr.RopePlan((255,))
    want = tr.rope_axes(q, None, pos, plan)[0]
    ref.check(want, ref.rope(q, pos, plan.axis, plan.freqs), "q")
    far = q.repeat(1, n // step + 1, 1, 1)[:, :n]
    tr.rope_axes(far, None, pos.repeat(1, 1, n // step + 1)[:, :, :n], plan, q_out=far)
    for first in (0, 2 ** 23 // step * step, (n // step - 1) * step, n // step * step):
        got = far[:, first:first + step]
        assert torch.equal(got, want[:, :got.shape[1]]), first


def test_rope_inverse_is_the_transpose():
    q, k, pos = _rope_case(F32, 1, 40, 2, 2, 64, (16, 16))
    plan = tr.RopePlan((16, 16), theta=500.0)
    qo, _ = tr.rope_axes(q, k, pos, plan)
    _, kb = tr.rope_axes(q, k, pos, plan, inverse=True)
    back, _ = tr.rope_axes(qo, None, pos, plan, inverse=True)
    assert (back - q).abs().max() < 4e-6 * q.abs().max()
    a, b = (qo.double() * k.double()).sum(), (q.double() * kb.double()).sum()
    assert (a - b).abs() < 1e-6 * (q.double().norm() * k.double().norm())


# -- attention -------------------------------------------------------------------------

def _qkv(seed, dtype, b, lq, lk, hq, hk, d, std=1.0):
    g = _gen(seed)
    return (_normal(g, b, lq, hq, d, dtype=dtype, std=std), _normal(g, b, lk, hk, d, dtype=dtype, std=std),
            _normal(g, b, lk, hk, d, dtype=dtype))


def _attend(q, k, v, name="", **kw):
    out, lse = tr.attention(q, k, v, return_lse=True, **kw)
    want = ref.attention(q, k, v, **kw)
    ref.check(out, want[0], name + " out")
    ref.check(lse, want[1], name + " lse")
    return out, lse


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d", [8, 32, 40, 64, 80, 96, 128, 136, 256])
def test_attention_head_dims(dtype, d):
    for lq, lk, hq, hk in ((1, 70, 2, 2), (45, 130, 4, 2), (300, 65, 3, 1)):
        _attend(*_qkv(d, dtype, 1, lq, lk, hq, hk, d), name=f"{lq}x{lk}")


@pytest.mark.parametrize("lk", [0, 1, 31, 32, 33, 63, 64, 65, 127, 200])
def test_attention_lengths(lk):
    for lq in (1, 2, 33, 129):
        _attend(*_qkv(lk, F16, 2, lq, lk, 2, 1, 64), name=f"{lq}x{lk}")


@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 65), (2, 64), (17, 17), (64, 64), (65, 130), (130, 65),
                                   (257, 257), (40, 300)])
@pytest.mark.parametrize("heads", [(4, 4), (4, 1), (6, 2)])
def test_attention_causal(lq, lk, heads):
    """Also more queries than keys: the first rows see nothing."""
    out, lse = _attend(*_qkv(lq + lk, BF16, 2, lq, lk, *heads, 64), causal=True)
    empty = max(lq - lk, 0)
    assert not out[:, :empty].any() and torch.isneginf(lse[:, :, :empty]).all()
    assert torch.isfinite(lse[:, :, empty:]).all()


@pytest.mark.parametrize("window", [(0, 0), (7, 3), (64, 0), (None, 5), (100, None), (1000, 1000)])
def test_attention_window(window):
    q, k, v = _qkv(5, F16, 1, 150, 210, 2, 2, 32)
    _attend(q, k, v, window=window)
    _attend(q, k, v, window=window, q_start=_ints([-40]))
    _attend(q, k, v, window=window, q_start=_ints([500]))


@pytest.mark.parametrize("lq", [1, 90])
def test_attention_positions_far_from_the_keys(lq):
    """Positions of 31 bits keep their place: a window ends before the keys or reaches them."""
    q, k, v = _qkv(58, F16, 2, lq, 100, 2, 1, 32)
    top = 2 ** 31 - 200
    reach = 2 ** 30
    for start, window in ((top, (reach, None)), (top, (reach, 0)), (-top, (None, reach)), (-top, (0, reach))):
        out, lse = tr.attention(q, k, v, window=window, q_start=_ints([start, start]), return_lse=True)
        assert not out.any() and torch.isneginf(lse).all(), (start, window)
    _attend(q, k, v, window=(reach, None), q_start=_ints([reach, reach + 50]))
    _attend(q, k, v, window=(None, reach), q_start=_ints([-reach, -reach + 50]))
    _attend(q, k, v, window=(None, 0), q_start=_ints([top, -top]))


@pytest.mark.parametrize("lq", [1, 5, 140])
def test_attention_prefix_and_lengths(lq):
    q, k, v = _qkv(6, BF16, 4, lq, 190, 4, 2, 64)
    kv_len = _ints([190, 0, 1, 100])
    q_start = _ints([190 - lq, 0, 0, 60])
    prefix = _ints([0, 50, 190, 33])
    _attend(q, k, v, kv_len=kv_len)
    _attend(q, k, v, causal=True, kv_len=kv_len, q_start=q_start)
    _attend(q, k, v, causal=True, prefix=prefix)
    _attend(q, k, v, window=(20, 0), prefix=prefix, kv_len=kv_len, q_start=q_start)
    # lengths and prefixes outside the cache are taken to its ends
    far = _ints([1000, -5, 191, 100])
    a = tr.attention(q, k, v, causal=True, kv_len=far, prefix=far)
    b = tr.attention(q, k, v, causal=True, kv_len=_ints([190, 0, 190, 100]), prefix=_ints([190, 0, 190, 100]))
    assert torch.equal(a, b)


def test_attention_documents():
    g = _gen(7)
    q, k, v = _qkv(7, F16, 2, 330, 330, 2, 1, 64)
    packed = torch.repeat_interleave(torch.arange(6), torch.tensor([1, 100, 63, 65, 40, 61])).int().cuda()
    _attend(q, k, v, docs=(packed, packed))
    _attend(q, k, v, docs=(packed, packed), causal=True)
    mixed = torch.randint(-3, 3, (2, 330), generator=g, dtype=torch.int32).cuda()  # in no order
    _attend(q, k, v, docs=(mixed, mixed))
    _attend(q, k, v, docs=(mixed, mixed), window=(50, 20), prefix=_ints([9, 70]))
    other = packed + 4  # some queries' documents hold no key
    out, lse = _attend(q, k, v, docs=(other, packed))
    gone = (other > 5).cpu()
    assert not out[:, gone].any() and torch.isneginf(lse[:, :, gone]).all()


def test_attention_documents_long():
    """More tiles than one look over the documents covers."""
    n = 140000
    q, k, v = _qkv(8, BF16, 1, 3, n, 1, 1, 32)
    doc_k = (torch.arange(n) // 1000).int().cuda()
    doc_q = _ints([0, 139, 70])
    _attend(q, k, v, docs=(doc_q, doc_k))


@pytest.mark.parametrize("lq", [2, 40])
def test_attention_longest_cache(lq):
    """2^30 keys, whose documents and codes take 2^32 bytes: the last ones, in turn of the
    query's document and of another, by their codes' distance. (K and V are one token, repeated.)"""
    n = 2 ** 30
    q, k, v = _qkv(55, F16, 1, lq, 1, 1, 1, 32)
    doc_k = torch.zeros(n, dtype=torch.int32, device="cuda")
    last = torch.arange(101, device="cuda") % 2 + 1
    doc_k[-101:] = last
    code_k = torch.zeros(n, dtype=torch.int32, device="cuda")
    code_k[-101:] = torch.arange(101, device="cuda") % 7
    slopes = torch.tensor([0.5], device="cuda")
    doc_q, code_q = _ints([1] * lq), _ints([3] * lq)
    far, tail = (t.expand(1, n, 1, 32) for t in (k, v)), (t.expand(1, 101, 1, 32) for t in (k, v))
    out, lse = tr.attention(q, *far, docs=(doc_q, doc_k), codes=(code_q, code_k), slopes=slopes, return_lse=True)
    want = ref.attention(q, *tail, docs=(doc_q, doc_k[-101:]), codes=(code_q, code_k[-101:]), slopes=slopes)
    ref.check(out, want[0], "out")
    ref.check(lse, want[1], "lse")


def test_attention_documents_of_several_longest_caches():
    """Two sequences of 2^30 keys have 2^26 tiles, whose documents take 2^32 threads to look over.
    (The second one's documents are the first's, four keys on.)"""
    n = 2 ** 30
    q, k, v = _qkv(56, BF16, 2, 1, 1, 1, 1, 32)
    store = torch.zeros(n + 4, dtype=torch.int32, device="cuda")
    store[-50:] = torch.arange(50, device="cuda") % 2 + 1
    docs = (_ints([[1], [2]]), store.as_strided((2, n), (4, 1)))
    out, lse = tr.attention(q, k.expand(2, n, 1, 32), v.expand(2, n, 1, 32), docs=docs, return_lse=True)
    tail = [t.expand(2, 50, 1, 32) for t in (k, v)]
    want = ref.attention(q, *tail, docs=(docs[0], docs[1][:, -50:]))
    ref.check(out, want[0], "out")
    ref.check(lse, want[1], "lse")


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("lq,lk", [(1, 100), (81, 81), (200, 70)])
def test_attention_bias(lq, lk, cap):
    g = _gen(9)
    q, k, v = _qkv(9, F16, 2, lq, lk, 6, 2, 32)
    slopes = torch.rand(6, generator=g).cuda()
    _attend(q, k, v, slopes=slopes, cap=cap)
    _attend(q, k, v, slopes=slopes, cap=cap, causal=True, q_start=_ints([3, lk - lq]))
    table = _normal(g, 6, 41)
    _attend(q, k, v, table=table, table_zero=20, cap=cap)
    codes = (torch.randint(-40, 40, (2, lq), generator=g, dtype=torch.int32).cuda(),
             torch.randint(-40, 40, (lk,), generator=g, dtype=torch.int32).cuda())
    _attend(q, k, v, table=table, table_zero=20, codes=codes, cap=cap)
    _attend(q, k, v, table=table, table_zero=20, slopes=slopes, codes=codes, cap=cap, window=(30, 5))
    big = _normal(g, 6, 9000)  # more entries than a workgroup keeps on the chip
    _attend(q, k, v, table=big, table_zero=4500, cap=cap)


def _capped(q, k, v, scale, cap, slopes=None, table=None, table_zero=0):
    """((out, tolerance), (lse, tolerance)) with capped scores, as transformer_reference but for
    the cap's error: 2^-20 of the capped score, not of the cap. (cap tanh(s / cap) is no more
    sensitive to s than s itself; the fit of tanh x / x is off by 8e-8, the form from an
    exponential above 0.6 by a few 2^-24 of the cap, each with a few roundings.)"""
    E = ref.E
    lq, lk, hq, hk, dim = q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3]
    q64, k64, v64 = (t[0].double().cpu().transpose(0, 1) for t in (q, k, v))
    k64, v64 = (t.repeat_interleave(hq // hk, 0) for t in (k64, v64))
    raw = torch.matmul(q64, k64.transpose(1, 2)) * scale
    s = cap * torch.tanh(raw / cap)
    d = dim * E * abs(scale) * torch.matmul(q64.abs(), k64.abs().transpose(1, 2)) + 4 * E * raw.abs()
    d = torch.minimum(d, 2 * s.abs() + 2 * cap) + 2.0 ** -20 * s.abs()
    diff = torch.arange(lk - lq, lk)[:, None] - torch.arange(lk)
    if slopes is not None:
        bias = -slopes.double().cpu()[:, None, None] * diff.abs()
        s, d = s + bias, d + 4 * E * bias.abs()
    if table is not None:
        bias = table.double().cpu()[:, (diff + table_zero).clamp(0, table.shape[1] - 1)]
        s, d = s + bias, d + 4 * E * bias.abs()
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - top)
    total = w.sum(-1, keepdim=True)
    w = w / total
    dmax = (d + 4 * E * s.abs()).amax(-1, keepdim=True) + 2.0 ** -20 + 4 * E * top.abs() + lk * E
    u = ref.UNIT[q.dtype]
    out = torch.matmul(w, v64)
    tol = u * out.abs() + (u + 2.2 * dmax) * torch.matmul(w, v64.abs()) \
        + ref.TINY[q.dtype] * (1 + v64.abs().sum(1, keepdim=True))
    lse = (torch.log(total) + top)[..., 0]
    return (out.transpose(0, 1)[None], tol.transpose(0, 1)[None]), \
        (lse[None], dmax[None, ..., 0] + 4 * E * lse.abs()[None])


CAPS = [0.5, 20.0, 1e3, 1e4, 1e6, 1e10]


@pytest.mark.parametrize("cap", CAPS)
@pytest.mark.parametrize("lq,d", [(1, 64), (70, 64), (40, 128)])
@pytest.mark.parametrize("kind", ["plain", "slopes", "table", "negative"])
def test_attention_caps_of_any_size(cap, lq, d, kind):
    """A cap far above the scores leaves them as they are, with a bias and without."""
    g = _gen(50)
    q, k, v = _qkv(50, F16, 1, lq, 200, 4, 2, d)
    kw = {"scale": 0.125, "cap": cap}
    if kind == "slopes":
        kw["slopes"] = torch.rand(4, generator=g).cuda() * 0.05
    elif kind == "table":
        kw["table"], kw["table_zero"] = _normal(g, 4, 41), 20
    elif kind == "negative":
        kw["scale"] = -0.125
    out, lse = tr.attention(q, k, v, return_lse=True, **kw)
    want = _capped(q, k, v, **kw)
    ref.check(lse, want[1], "lse")
    ref.check(out, want[0], "out")


@pytest.mark.parametrize("slopes", [False, True])
def test_attention_small_scores_beside_capped_ones(slopes):
    """One row whose scores reach the cap leaves the other rows' small scores exact."""
    q, k, v = _qkv(51, BF16, 1, 40, 96, 2, 1, 64)
    q[0, 3], k[0, 50] = 100.0, 1.0  # q . k = 6400
    kw = {"scale": 1.0, "cap": 8e3}
    q[0, :3], q[0, 4:] = q[0, :3] * 0.01, q[0, 4:] * 0.01
    if slopes:
        kw["slopes"] = torch.tensor([0.01, 0.1], device="cuda")
    out, lse = tr.attention(q, k, v, return_lse=True, **kw)
    want = _capped(q, k, v, **kw)
    ref.check(lse, want[1], "lse")
    ref.check(out, want[0], "out")


def test_attention_window_table_in_two_dimensions():
    g = _gen(10)
    n, d = 7, 32
    q, k, v = _qkv(10, F16, 3, n * n, n * n, 2, 2, d)
    y, x = torch.arange(n * n) // n, torch.arange(n * n) % n
    codes = (y * (2 * n - 1) + x).int().cuda()
    zero = (n - 1) * (2 * n - 1) + n - 1
    table = _normal(g, 2, (2 * n - 1) ** 2)
    _attend(q, k, v, table=table, table_zero=zero, codes=(codes, codes))
    hidden = table.clone()
    hidden[:, zero + 1:] = -math.inf  # entries that hide: only offsets of zero or less are seen
    _attend(q, k, v, table=hidden, table_zero=zero, codes=(codes, codes))
    hidden[1] = -math.inf
    out, lse = _attend(q, k, v, table=hidden, table_zero=zero, codes=(codes, codes))
    assert not out[:, :, 1].any() and torch.isneginf(lse[:, 1]).all()


@pytest.mark.parametrize("cap,bias", [(1e-7, False), (1e-7, True), (1e-30, False), (1e-30, True), (3e38, False),
                                      (3e38, True)])
@pytest.mark.parametrize("zeros", [False, True])
def test_attention_caps_at_the_types_ends(cap, bias, zeros):
    """tanh's argument or its polynomial's coefficients pass the type's range: a cap near 0
    leaves all keys alike, a huge one changes nothing."""
    q, k, v = _qkv(52, BF16, 1, 33, 100, 2, 1, 64)
    if zeros:
        k.zero_()
    kw = {"slopes": torch.zeros(2, device="cuda")} if bias else {}
    out, lse = tr.attention(q, k, v, cap=cap, return_lse=True, **kw)
    want = ref.attention(q, torch.zeros_like(k) if cap < 1 else k, v)
    ref.check(lse, want[1], "lse")
    ref.check(out, want[0], "out")


@pytest.mark.parametrize("scale,std", [(0.0, 1.0), (-0.3, 1.0), (3.0, 3.0), (1e-4, 1.0)])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_attention_scale(scale, std, cap):
    """Peaked, flat and reversed scores; a running maximum that keeps growing."""
    q, k, v = _qkv(11, BF16, 1, 70, 300, 2, 1, 64, std=std)
    k = k * torch.linspace(0.1, 2, 300, device="cuda")[None, :, None, None].to(BF16)
    _attend(q, k, v, scale=scale, cap=cap)


@pytest.mark.parametrize("lq", [1, 100])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_hidden_values(lq, dtype):
    """NaN, infinities and the type's ends in places that no query, or not every query,
    sees."""
    q, k, v = _qkv(12, dtype, 2, lq, 200, 4, 2, 64)
    top = torch.finfo(dtype).max
    for bad in (math.nan, math.inf, -math.inf, top, -top):
        kb, vb = k.clone(), v.clone()
        kb[:, 150:], vb[:, 150:] = bad, bad
        _attend(q, kb, vb, f"{bad} past the length", kv_len=_ints([150, 149]))
        docs = (torch.zeros(lq).int().cuda(), (torch.arange(200) >= 150).int().cuda())
        _attend(q, kb, vb, f"{bad} in another document", docs=docs)
        table = torch.zeros(4, 2)
        table[:, 1] = -math.inf
        codes = (torch.zeros(lq).int().cuda(), -(torch.arange(200) >= 150).int().cuda())
        _attend(q, kb, vb, f"{bad} behind the table", table=table.cuda(), codes=codes)


@pytest.mark.parametrize("lq,n", [(1, 41), (1, 9000), (70, 41), (70, 9000), (70, 2 ** 30 + 16)])
def test_attention_hidden_values_behind_tables_of_any_size(lq, n):
    """Tables that a workgroup keeps on the chip, that it does not, and of more than 2^31
    entries a key head; only one of its offsets hides."""
    q, k, v = _qkv(53, F16, 1, lq, 150, 2, 1, 64)
    table = torch.zeros(2, n, device="cuda")
    table[:, 20:30] = _normal(_gen(53), 2, 10)
    table[:, 40] = -math.inf
    hidden = torch.arange(150) % 5 == 2
    codes = _ints([25] * lq), (hidden.int() * -15).cuda()
    seen = ~hidden
    want = tr.attention(q, k[:, seen], v[:, seen], table=table, codes=(codes[0], _ints([0] * int(seen.sum()))))
    for bad in (math.nan, math.inf):
        kb, vb = k.clone(), v.clone()
        kb[:, hidden], vb[:, hidden] = bad, bad
        got = tr.attention(q, kb, vb, table=table, codes=codes)
        # The same weights in another order of the keys: two roundings of 2^-11 each, of sums of |v| < 5.
        assert (got.double() - want.double()).abs().max() < 4 * 2 ** -11 * 5


@pytest.mark.parametrize("n", [41, 9000])
@pytest.mark.parametrize("lq", [1, 70])
def test_attention_table_of_the_types_lowest_value(lq, n):
    """The lowest finite value weighs keys by 0 beside others, and alike where there are no
    others: it hides nothing."""
    q, k, v = _qkv(54, F16, 1, lq, 150, 2, 2, 32)
    low = torch.finfo(F32).min
    some = torch.zeros(2, n, device="cuda")
    some[:, 7] = low
    keys = (torch.arange(150) % 3 == 1)
    codes = _ints([7] * lq), (keys.int() * 7).cuda()
    out, lse = tr.attention(q, k, v, table=some, codes=codes, return_lse=True)
    want = ref.attention(q, k[:, keys], v[:, keys])
    ref.check(out, want[0], "out beside others")
    ref.check(lse, want[1], "lse beside others")
    out, lse = tr.attention(q, k, v, table=torch.full((2, n), low, device="cuda"), return_lse=True)
    assert torch.isfinite(lse).all() and (lse < -1e38).all()
    # Every score rounds to the same number, so all keys weigh alike.
    want = ref.attention(q, torch.zeros_like(k), v)
    ref.check(out, want[0], "out alone")


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_hidden_from_some(bad):
    """A key that is not finite reaches the rows that see it and no other."""
    q, k, v = _qkv(13, F16, 1, 100, 100, 2, 1, 64)
    vb = v.clone()
    vb[0, 70, 0, 5] = bad
    vb[0, 80, 0, 6] = -bad
    out, _ = _attend(q, k, vb, causal=True)
    assert torch.isfinite(out[:, :70]).all() and not torch.isfinite(out[0, 70:, :, 5]).any()
    kb = k.clone()
    kb[0, 70] = math.nan
    out = tr.attention(q, kb, v, causal=True)
    assert torch.isfinite(out[:, :70]).all() and torch.isnan(out[:, 70:]).all()


@pytest.mark.parametrize("lq,lk", [(1, 64), (40, 200), (1, 4000)])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_values_at_the_types_end(lq, lk, sign):
    """A mean of fp16's largest number is that number, also where the weights' own rounding
    (here up, by 2^-11) makes more of it."""
    q = torch.zeros(1, lq, 1, 8, dtype=F16, device="cuda")
    k = torch.zeros(1, lk, 1, 8, dtype=F16, device="cuda")
    q[..., 0], k[:, 0, :, 0] = 1, 1
    v = torch.full_like(k, sign * torch.finfo(F16).max)
    # All keys but the first weigh 0.500245, next to the middle of two fp16 numbers.
    out = tr.attention(q, k, v, scale=-math.log(0.500245))
    assert torch.equal(out, v[:, :1].expand(1, lq, 1, 8))
    v[:, :, :, 3] = math.inf
    out = tr.attention(q, k, v, scale=-math.log(0.500245))
    assert torch.isposinf(out[..., 3]).all() and torch.equal(out[..., 4:], v[:, :1, :, 4:].expand(1, lq, 1, 4))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("lq,hq", [(1, 8), (8192, 8)])
@pytest.mark.parametrize("depth", [14.0, 17.5, 19.0])
def test_attention_many_keys_of_small_weight(dtype, lq, hq, depth):
    """One key far above 2^17 others, whose weights lie among fp16's subnormal numbers or below
    but add up. The first key's V is 0, the others' 1: the result is their share."""
    n = 2 ** 17
    q = torch.zeros(1, lq, hq, 32, dtype=dtype, device="cuda")
    k = torch.zeros(1, n, hq, 32, dtype=dtype, device="cuda")
    v = torch.ones(1, n, hq, 32, dtype=dtype, device="cuda")
    q[..., 0], k[:, 0, :, 0], v[:, 0] = depth, 1, 0
    out, lse = tr.attention(q, k, v, scale=1.0, return_lse=True)
    tail = (n - 1) * math.exp(-depth)
    want = tail / (1 + tail)
    # Each weight's rounding to the type (fp16: 2^-11, subnormal from 2^-14 / 128 on, where a
    # weight is off by 2^-25 / 128 at most), the exponential's argument (2^-20), the result's own rounding.
    u = ref.UNIT[dtype]
    small = n * 2.0 ** -32 if dtype == F16 else 0.0
    assert (out.double() - want).abs().max() < (2 * u + 2 ** -18) * want + small + ref.TINY[dtype]
    # The running sum's additions, as in transformer_reference.attention.
    assert (lse.double() - (depth + math.log1p(tail))).abs().max() < n * ref.E + 1e-5


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("depth", [20.0, 200.0])
def test_attention_seen_values_of_small_weight(dtype, bad, depth):
    """A value that is not finite reaches the rows that see it also where its weight rounds
    to 0, in tiles that other rows do not see whole."""
    q, k, v = _qkv(57, dtype, 1, 100, 100, 2, 1, 64)
    q[..., 0], k[..., 0] = 1, 0
    k[0, 70, 0] = 0
    k[0, 70, 0, 0] = -depth  # e^-depth beside the others
    v[0, 70, 0, 5] = bad
    out = tr.attention(q, k, v, causal=True, scale=1.0)
    assert torch.isfinite(out[:, :70]).all()
    assert not torch.isfinite(out[0, 71:, :, 5]).any()
    assert torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 6:]).all()


def test_attention_layouts():
    """Heads before tokens, one projection's views, a broadcast key, gaps between tokens."""
    g = _gen(14)
    qkv = _normal(g, 2, 75, 12, 64, dtype=F16)
    q, k, v = qkv[:, :, :6], qkv[:, :, 6:9], qkv[:, :, 9:]
    plain, _ = _attend(q, k, v, causal=True)
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    out = torch.empty(2, 6, 75, 64, dtype=F16, device="cuda").transpose(1, 2)
    got = tr.attention(*heads, causal=True, out=out)
    assert got is out and torch.equal(out, plain)
    one = [t[:1].expand(2, -1, -1, -1) for t in (k, v)]
    _attend(q, *one)
    wide = torch.full((2, 75, 6, 96), math.nan, dtype=F16, device="cuda")
    wide[..., 16:80] = q
    assert torch.equal(tr.attention(wide[..., 16:80], k, v, causal=True), plain)
    assert torch.equal(tr.attention(q[:1], k[:1], v[:1], causal=True), plain[:1])


@pytest.mark.parametrize("lq", [1, 40])
def test_attention_long_strides(lq):
    """Keys whose offsets pass 32 bits."""
    n, step = 70, 2 ** 25
    store = torch.zeros(n * step + 64, dtype=F16, device="cuda")
    k = store.as_strided((1, n, 1, 64), (0, step, 64, 1))
    q, kd, vd = _qkv(15, F16, 1, lq, n, 2, 1, 64)
    k.copy_(kd)
    want = tr.attention(q, kd, vd)
    assert torch.equal(tr.attention(q, k, vd), want)
    k.copy_(vd)
    assert torch.equal(tr.attention(q, kd, k), want)


@pytest.mark.parametrize("lq,lk,hq,hk,b", [(1, 5000, 4, 1, 2), (3, 3000, 8, 2, 1), (100, 2500, 2, 1, 1),
                                           (300, 4000, 2, 2, 1), (1, 20000, 32, 8, 1), (40, 700, 1, 1, 1)])
def test_attention_split_keys(lq, lk, hq, hk, b):
    """Few rows over many keys, which are divided over workgroups and joined."""
    q, k, v = _qkv(16, BF16, b, lq, lk, hq, hk, 32)
    _attend(q, k, v)
    _attend(q, k, v, causal=True, kv_len=_ints([lk - 7 * i - 1 for i in range(b)]),
            q_start=_ints([lk - lq - 7 * i - 1 for i in range(b)]))
    _attend(q, k, v, window=(1000, 0), prefix=_ints([37] * b))
    none = _ints([0] * b)
    out, lse = _attend(q, k, v, kv_len=none)
    assert not out.any() and torch.isneginf(lse).all()


def test_attention_nothing_to_do():
    q, k, v = _qkv(17, F16, 2, 4, 9, 2, 2, 32)
    assert tr.attention(q[:0], k[:0], v[:0]).shape == (0, 4, 2, 32)
    assert tr.attention(q[:, :0], k, v).shape == (2, 0, 2, 32)
    out, lse = tr.attention(q, k[:, :0], v[:, :0], return_lse=True)
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.parametrize("docs", [False, True])
@pytest.mark.parametrize("codes", [False, True])
def test_attention_no_tokens_with_documents_and_codes(docs, codes):
    q, k, v = _qkv(17, BF16, 2, 4, 9, 2, 2, 32)

    def arrays(lq, lk):
        pair = _ints([1] * lq), _ints([1] * lk)
        return {**({"docs": pair} if docs else {}),
                **({"codes": pair, "slopes": torch.ones(2, device="cuda")} if codes else {})}

    assert tr.attention(q[:, :0], k, v, **arrays(0, 9)).shape == (2, 0, 2, 32)
    assert tr.attention(q[:, :0], k[:, :0], v[:, :0], **arrays(0, 0)).shape == (2, 0, 2, 32)
    out = torch.full_like(q, math.nan)
    got, lse = tr.attention(q, k[:, :0], v[:, :0], out=out, return_lse=True, prefix=_ints([0, 3]), **arrays(4, 0))
    assert got is out and not out.any() and torch.isneginf(lse).all()


def test_attention_masks_by_differences():
    """Moving a hidden key or value changes no bit; moving a seen one moves the output
    by its weight (a central difference of the value against the softmax's weight)."""
    q, k, v = _qkv(18, F16, 1, 50, 50, 1, 1, 32)
    base, lse = tr.attention(q, k, v, causal=True, return_lse=True)
    kb, vb = k.clone(), v.clone()
    kb[:, 30:], vb[:, 30:] = -kb[:, 30:], 5 * vb[:, 30:]
    moved = tr.attention(q, kb, vb, causal=True)
    assert torch.equal(moved[:, :30], base[:, :30])
    up, down = v.clone(), v.clone()
    up[0, 10, 0], down[0, 10, 0] = 64.0, -64.0
    diff = (tr.attention(q, k, up, causal=True).double() - tr.attention(q, k, down, causal=True).double()) / 128
    s = (q[0, :, 0].double() @ k[0, 10, 0].double()) / math.sqrt(32)
    weight = torch.exp(s - lse[0, 0].double())
    weight[:10] = 0
    # rounding of the weight (2^-11) and of the two results (2^-11 of at most 64 + max |v|)
    assert (diff[0, :, 0] - weight[:, None]).abs().max() < 2 ** -11 + 2 * 2 ** -11 * 68 / 128 + 1e-5


# -- norms around a gated residual ---------------------------------------------------------

NORM = [
    # dtype, residual, B, L, C, post, pre, gate shape, act, modulation, biases
    (BF16, BF16, 4, 1, 4096, "rms", "rms", "channel", "none", False, False),
    (F16, F16, 2, 37, 1024, "layer", "layer", "batch", "tanh", True, True),
    (BF16, F32, 3, 19, 975, "rms", "rms", "token", "sigmoid", False, False),
    (F16, F32, 1, 5, 1, "rms", "layer", "channel", "silu", False, True),
    (F16, F16, 1, 9, 7, "layer", "rms", "token", "none", True, False),
    (F32, F32, 2, 3, 513, "layer", "layer", "batch", "tanh", True, True),
    (F16, F16, 1, 3, 5120, "rms", None, None, "none", False, True),
    (BF16, BF16, 1, 3, 8200, None, "layer", "token", "silu", True, True),
    (BF16, F32, 1, 2, 32768, "layer", "rms", "channel", "sigmoid", True, True),
    (F32, F32, 1, 130, 64, None, None, "batch", "none", True, False),
    (F16, F16, 5, 41, 72, "rms", "rms", "channel", "none", False, False),
    (BF16, BF16, 1, 7, 2047, "layer", "layer", "token", "tanh", True, True),
]


def _norm_case(dtype, res, b, l, c, post, pre, gate, act, mod, bias, seed=0):
    g = _gen(seed + c)
    shapes = {"channel": (c,), "batch": (b, 1, c), "token": (b, l, c)}
    kw = {"post": post, "pre": pre, "gate_act": act, "branch_scale": 0.7, "residual_scale": 1.1}
    for side, kind in (("post", post), ("pre", pre)):
        if kind is not None:
            kw[side + "_weight"] = 1 + _normal(g, c, std=0.2)
            if bias:
                kw[side + "_bias"] = _normal(g, c, std=0.2)
    if gate is not None:
        kw["gate"] = _normal(g, *shapes[gate], dtype=dtype)
    if mod:
        kw["mod_scale"], kw["mod_shift"] = (_normal(g, b, 1, c, dtype=dtype, std=0.3) for _ in range(2))
    return _normal(g, b, l, c, dtype=res, std=2.0), _normal(g, b, l, c, dtype=dtype) + 0.5, kw


@pytest.mark.parametrize("dtype,res,b,l,c,post,pre,gate,act,mod,bias", NORM)
def test_gated_norm(dtype, res, b, l, c, post, pre, gate, act, mod, bias):
    r, y, kw = _norm_case(dtype, res, b, l, c, post, pre, gate, act, mod, bias)
    want = ref.gated_norm(r, y, **kw)
    new, h = tr.gated_norm(r, y, **kw)
    ref.check(new, want[0], "residual")
    if h is not None:
        ref.check(h, want[1], "h")
    again = tr.gated_norm(r, y, **kw)
    assert torch.equal(again[0], new) and (h is None or torch.equal(again[1], h))
    place = r.clone()
    out, _ = tr.gated_norm(place, y, residual_out=place, **kw)
    assert out is place and torch.equal(place, new)


@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh", "silu"])
@pytest.mark.parametrize("c", [5, 512, 975])
def test_gated_norm_activation_without_a_gate(act, c):
    """No gate stands for a gate of 1, which goes through the activation."""
    g = _gen(24)
    r, y = _normal(g, 2, 9, c, dtype=BF16), _normal(g, 2, 9, c, dtype=BF16)
    kw = {"post": "rms", "pre": "layer", "gate_act": act, "branch_scale": 0.7}
    want = ref.gated_norm(r, y, **kw)
    new, h = tr.gated_norm(r, y, **kw)
    ref.check(new, want[0], "residual")
    ref.check(h, want[1], "h")
    for got, of_one in zip((new, h), tr.gated_norm(r, y, gate=torch.ones(c, dtype=BF16, device="cuda"), **kw)):
        assert torch.equal(got, of_one)


def test_gated_norm_parts_alone():
    """The first norm of a network (no branch), the last residual (no norm after it)."""
    g = _gen(20)
    r, y = _normal(g, 2, 5, 136, dtype=BF16), _normal(g, 2, 5, 136, dtype=BF16)
    w = 1 + _normal(g, 136, std=0.1)
    same, h = tr.gated_norm(r, pre="rms", pre_weight=w)
    assert same is r
    ref.check(h, ref.gated_norm(r, pre="rms", pre_weight=w)[1], "h")
    new, h = tr.gated_norm(r, y, post="rms", post_weight=w)
    assert h is None
    ref.check(new, ref.gated_norm(r, y, post="rms", post_weight=w)[0], "residual")
    scaled, none = tr.gated_norm(r, residual_scale=0.5)
    assert none is None and torch.equal(scaled, r * 0.5)
    wide, h = tr.gated_norm(r.float(), pre="layer", dtype=F16)
    assert h.dtype == F16
    ref.check(h, ref.gated_norm(r.float(), pre="layer", dtype=F16)[1], "h of an fp32 residual")


def test_gated_norm_strides():
    """Views of wider tensors, misaligned rows, a broadcast residual, tokens of an image's
    interior."""
    g = _gen(21)
    big = _normal(g, 2, 9, 301, dtype=F16)
    y = _normal(g, 2, 9, 77, dtype=F16)
    for lo in (0, 1, 3, 8, 200):
        r = big[..., lo:lo + 77]
        want = ref.gated_norm(r, y, post="rms", pre="layer")
        new, h = tr.gated_norm(r, y, post="rms", pre="layer")
        ref.check(new, want[0], "residual")
        ref.check(h, want[1], "h")
        place = big.clone()
        tr.gated_norm(r, y, post="rms", pre="layer", residual_out=place[..., lo:lo + 77])
        assert torch.equal(place[..., lo:lo + 77], new)
        place[..., lo:lo + 77] = big[..., lo:lo + 77]
        assert torch.equal(place, big)
    one = big[:1, :1, :77].expand(2, 9, 77)
    ref.check(tr.gated_norm(one, y)[0], ref.gated_norm(one, y)[0], "broadcast residual")
    padded = _normal(g, 6, 10, 64, dtype=F16)  # rows of an image with a border
    inner = padded[1:5, 1:9]
    ref.check(tr.gated_norm(inner, pre="rms")[1], ref.gated_norm(inner, pre="rms")[1], "interior")


def test_gated_norm_large_mean_and_zeros():
    """A mean a thousand times the spread; rows of zeros; eps = 0 on them."""
    g = _gen(22)
    r = 1000 + _normal(g, 1, 4, 640)
    ref.check(tr.gated_norm(r, pre="layer")[1], ref.gated_norm(r, pre="layer")[1], "large mean")
    zero = torch.zeros(1, 3, 100, dtype=F16, device="cuda")
    assert not tr.gated_norm(zero, pre="rms")[1].any() and not tr.gated_norm(zero, pre="layer")[1].any()
    assert torch.isnan(tr.gated_norm(zero, pre="rms", eps=0.0)[1]).all()


def test_gated_norm_more_rows_than_a_launch_takes():
    """2^26 rows of a wave each number 2^32 threads."""
    n = 2 ** 26 + 5
    r = _normal(_gen(23), 4099, 8, dtype=F16).repeat(n // 4099 + 1, 1)[:n][None]
    new, h = tr.gated_norm(r, pre="rms", residual_scale=0.5)
    want = ref.gated_norm(r[:, :4099], pre="rms", residual_scale=0.5)
    ref.check(new[:, :4099], want[0], "residual")
    ref.check(h[:, :4099], want[1], "h")
    for got in (new, h):  # the rows repeat, so do the results
        whole = n // 4099 * 4099
        assert torch.equal(got[0, :whole].view(-1, 4099, 8), got[0, :4099].expand(n // 4099, -1, -1))
        assert torch.equal(got[0, whole:], got[0, :n - whole])


def test_gated_norm_rows_do_not_mix():
    """A row of NaN stays one row, also where rows share a workgroup."""
    for c in (64, 72, 700, 1024):
        r = _normal(_gen(c), 1, 11, c, dtype=F16)
        clean = tr.gated_norm(r, pre="layer")[1]
        r[0, 5, c // 2] = math.nan
        h = tr.gated_norm(r, pre="layer")[1]
        assert torch.isnan(h[0, 5]).all()
        keep = [i for i in range(11) if i != 5]
        assert torch.equal(h[0, keep], clean[0, keep])


# -- streams and graphs ------------------------------------------------------------------------

def _block_case():
    q, k, v = _qkv(30, F16, 1, 3, 3000, 4, 2, 64)
    kq = k[:, -3:].contiguous()
    g = _gen(30)
    res = _normal(g, 1, 3, 256, dtype=F16)
    pos = torch.randint(0, 99, (2, 1, 3), generator=g, dtype=torch.int32).cuda()
    return q, kq, k, v, pos, tr.RopePlan((16, 16)), res, {"post": "rms", "pre": "layer"}


def _run(case):
    q, kq, k, v, pos, plan, res, kw = case
    qr, kr = tr.rope_axes(q, kq, pos, plan)
    o, lse = tr.attention(qr, k, v, causal=True, return_lse=True)
    new, h = tr.gated_norm(res, o.flatten(2), **kw)
    return qr, kr, o, lse, new, h


def test_streams():
    """On a stream of their own, chosen as the current one or by its handle, the operators
    give the same bits, with inputs that the stream itself made just before."""
    case = _block_case()
    want = _run(case)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    q, k, v = case[0], case[2], case[3]
    with torch.cuda.stream(s):
        late = q + 0
        got = _run((late,) + case[1:])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.cuda.stream(s):
        late = want[0] + 0
    o = tr.attention(late, k, v, causal=True, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(o, want[2])


def test_results_belong_to_the_calls_stream():
    """Also where the handle is the default stream's, 0, as its users pass it."""
    q, k, v = _qkv(31, F16, 1, 3, 3000, 4, 2, 64)
    r = _normal(_gen(31), 1, 3, 256, dtype=F16)
    plan, pos = tr.RopePlan((16, 16)), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    want, y = tr.attention(q, k, v), r.clone()

    def owner(t):
        at = t.data_ptr()
        return next(s["stream"] for s in torch.cuda.memory_snapshot()
                    if s["address"] <= at < s["address"] + s["total_size"])

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (torch.cuda.default_stream(), side):
        out, lse = tr.attention(q, k, v, return_lse=True, stream=stream.cuda_stream)
        turned, _ = tr.rope_axes(q, None, pos, plan, stream=stream.cuda_stream)
        new, h = tr.gated_norm(r, y, pre="rms", stream=stream.cuda_stream)
        stream.synchronize()
        assert [owner(t) for t in (out, lse, turned, new, h)] == [stream.cuda_stream] * 5
        assert torch.equal(out, want)


def test_graph_replays():
    case = _block_case()
    want = _run(case)
    q = case[0]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(2):
            _run(case)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(case)
    other = -q
    first = q.clone()
    for turn in range(4):
        for t in got:
            t.zero_()
        q.copy_(other if turn % 2 else first)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(case)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), turn
        if turn % 2 == 0:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# -- refusals that need tensors on the GPU ---------------------------------------------------------

def test_refusals():
    q, k, v = _qkv(40, F16, 2, 4, 9, 4, 2, 32)
    bad = [
        (dict(q=q.float()), "unsupported type"),
        (dict(k=k.bfloat16()), "k must be"),
        (dict(v=v[:, :8]), "k and v"),
        (dict(k=k[:, :, :1], v=v[:, :, :1].expand(-1, -1, 3, -1)), "k and v"),
        (dict(q=q[:, :, :3]), "multiple of k_heads"),
        (dict(q=q[..., ::2], k=k[..., ::2], v=v[..., ::2]), "contiguous"),
        (dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), "multiple of 8"),
        (dict(q=q[..., 4:28], k=k[..., 4:28], v=v[..., 4:28]), "aligned"),
        (dict(kv_len=torch.ones(2, dtype=torch.int64, device="cuda")), "kv_len must be"),
        (dict(prefix=_ints([1])), "prefix must be"),
        (dict(docs=(_ints([0] * 4), _ints([0] * 8))), "doc_k must be"),
        (dict(slopes=torch.ones(2, device="cuda")), "slopes must be"),
        (dict(table=torch.ones(4, 0, device="cuda")), "table without entries"),
        (dict(cap=-1.0), "cap"),
        (dict(cap=math.nan), "cap"),
        (dict(scale=math.inf), "scale"),
        (dict(window=(-2, 0)), "window"),
        (dict(causal=True, window=(None, 3)), "causal"),
        (dict(out=q), "overlap"),
        (dict(out=torch.empty_like(q[:1]).expand(2, -1, -1, -1)), "zero stride"),
    ]
    for change, text in bad:
        args = {"q": q, "k": k, "v": v, **change}
        with pytest.raises(EngineError, match=text):
            tr.attention(args.pop("q"), args.pop("k"), args.pop("v"), **args)
    big_k = k[:, :1].expand(2, 5000, 2, 32)
    with pytest.raises(EngineError, match="workspace too small"):
        tr.attention(q, big_k, big_k, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    plan = tr.RopePlan((8, 8))
    pos = torch.zeros(2, 2, 4, dtype=torch.int32, device="cuda")
    for change, text in [(dict(pos=pos[:1]), "pos must be"), (dict(pos=pos.long()), "pos must be"),
                         (dict(plan=tr.RopePlan((8, 9))), "n_freq"), (dict(q=q.transpose(2, 3)), "must agree|contiguous|n_freq"),
                         (dict(q_out=q.transpose(0, 1)), "q_out"), (dict(k=k[:1]), "agree")]:
        args = {"q": q, "k": k[:, :4], "pos": pos, "plan": plan, **change}
        with pytest.raises(EngineError, match=text):
            tr.rope_axes(args.pop("q"), args.pop("k"), args.pop("pos"), args.pop("plan"), **args)
    r = _normal(_gen(1), 2, 3, 64, dtype=F16)
    w = torch.ones(64, device="cuda")
    for change, text in [(dict(y=r[:, :2]), "shape"), (dict(post="max"), "norm is"),
                         (dict(pre_weight=w.half()), "pre_weight"), (dict(gate=r[:, :, :32]), "broadcast"),
                         (dict(gate_act="relu"), "activation"), (dict(eps=-1.0), "eps"),
                         (dict(y=r.bfloat16()), "residual type"), (dict(y=None, gate=r), "without y"),
                         (dict(residual_out=r[:1].expand(2, -1, -1)), "zero stride"),
                         (dict(h=r, pre="rms"), "overlap")]:
        args = {"y": r.clone(), **change}
        with pytest.raises(EngineError, match=text):
            tr.gated_norm(r, args.pop("y"), **args)
    assert torch.isfinite(tr.attention(q, k, v)).all()  # nothing was left behind


# -- strides that torch cannot make -----------------------------------------------------------------

def _flipped(t, dims):
    """t's values in memory that goes backwards along some dimensions: (memory, address, strides)."""
    mem = t.flip(dims).contiguous()
    strides = list(mem.stride())
    at = mem.data_ptr()
    for d in dims:
        at += (t.shape[d] - 1) * strides[d] * t.element_size()
        strides[d] = -strides[d]
    return mem, at, strides


@pytest.mark.parametrize("dims", [(0,), (1,), (2,), (0, 1, 2)])
def test_negative_strides(dims):
    """Through the C entry points: every tensor backwards along the dimensions, outputs too."""
    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    for lq, lk in ((1, 70), (70, 70), (150, 1000)):
        q, k, v = _qkv(60, F16, 2, lq, lk, 4, 2, 64)
        want = tr.attention(q, k, v, causal=True)
        a = _lib.AttentionArgs()
        kept = []
        for name, t in (("q", q), ("k", k), ("v", v), ("out", torch.zeros_like(q))):
            mem, at, strides = _flipped(t, dims)
            kept.append(mem)
            setattr(a, name, at)
            setattr(a, name + "_stride", tuple(strides[:3]))
        a.scale, a.left, a.right = 0.125, -1, 0
        a.batch, a.q_tokens, a.k_tokens, a.q_heads, a.k_heads, a.head_dim = 2, lq, lk, 4, 2, 64
        work = torch.empty(lib.arthip_attention_workspace(ctypes.byref(a)), dtype=torch.uint8, device="cuda")
        a.workspace, a.workspace_bytes = work.data_ptr(), work.numel()
        assert lib.arthip_attention(ctypes.byref(a), stream) == 0, _lib.last_error()
        assert torch.equal(kept[3].flip(dims), want), (lq, lk)

    q, k, pos = _rope_case(BF16, 2, 9, 3, 3, 64, (8, 24))
    plan = tr.RopePlan((8, 24))
    want = tr.rope_axes(q, k, pos, plan)
    a = _lib.RopeArgs()
    kept = {}
    for name, t in (("q", q), ("k", k), ("q_out", torch.zeros_like(q)), ("k_out", torch.zeros_like(k))):
        kept[name], at, strides = _flipped(t, dims)
        setattr(a, name, at)
        setattr(a, name + "_stride", tuple(strides[:3]))
    kept["pos"], a.pos, strides = _flipped(pos, dims)
    a.pos_stride, a.packed = tuple(strides), plan.packed.data_ptr()
    a.n_freq, a.dtype, a.batch, a.tokens, a.q_heads, a.k_heads, a.head_dim = 32, 1, 2, 9, 3, 3, 64
    assert lib.arthip_rope_axes(ctypes.byref(a), stream) == 0, _lib.last_error()
    assert torch.equal(kept["q_out"].flip(dims), want[0]) and torch.equal(kept["k_out"].flip(dims), want[1])

    rows = [d for d in dims if d < 2] or [0, 1]
    g = _gen(61)
    r, y, gate = (_normal(g, 2, 9, 200, dtype=F16) for _ in range(3))
    want = tr.gated_norm(r, y, post="rms", gate=gate, gate_act="tanh", pre="layer")
    a = _lib.NormArgs()
    for name, t in (("residual", r), ("y", y), ("gate", gate), ("residual_out", torch.zeros_like(r)),
                    ("h", torch.zeros_like(r))):
        kept[name], at, strides = _flipped(t, rows)
        setattr(a, name, at)
        setattr(a, name + "_stride", tuple(strides[:2]))
    a.post, a.pre, a.gate_act, a.batch, a.tokens, a.channels = 1, 2, 2, 2, 9, 200
    a.eps, a.residual_scale, a.branch_scale = 1e-6, 1.0, 1.0
    assert lib.arthip_gated_norm(ctypes.byref(a), stream) == 0, _lib.last_error()
    assert torch.equal(kept["residual_out"].flip(rows), want[0]) and torch.equal(kept["h"].flip(rows), want[1])
