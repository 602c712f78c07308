"""The paged cache on the GPU against its definitions in float64 (tests/paged_reference.py,
whose tolerances are derived there): types, head layouts, lengths, pages, masks, strides,
streams, graphs, values that are not finite, and the operators one after the other."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from arthip_amd import _lib, paged
from arthip_amd.engine import EngineError
from tests import paged_reference as pref
from tests import transformer_reference as ref
from tests.paged_reference import Cache

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _bits(x):
    return x.contiguous().view(torch.int16 if x.element_size() == 2 else torch.int32).cpu()


def _same(a, b):
    assert torch.equal(_bits(a), _bits(b))


# -- writing -------------------------------------------------------------------------------

WRITES = [
    # dtype, Hk, D, page, [(new, slots)]
    (BF16, 8, 128, 16, [(1, 37), (1, 1), (1, 16), (1, 17)]),
    (F16, 3, 72, 48, [(5, 50), (0, 9), (33, 33), (1, 1), (0, 0), (17, 100)]),
    (F16, 1, 8, 16, [(200, 300)]),
    (BF16, 2, 256, 32, [(3, 40), (70, 70)]),
]


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("dtype,hk,d,page,seqs", WRITES)
def test_write(dtype, hk, d, page, seqs, heads_first):
    c = Cache(seqs, hk, d, dtype, page, heads_first=heads_first)
    t = sum(c.n)
    k, v = c.normal(t + 2, hk, d), c.normal(t + 2, hk, d)  # two rows behind the last sequence
    slots = max(c.len) + 3
    token_positions = torch.arange(t + 2, dtype=torch.int32) + 1000
    positions = torch.full((len(seqs), hk, slots), -7, dtype=torch.int32)
    dev = c.cuda()
    got = positions.cuda()
    paged.cache_write(k.cuda(), v.cuda(), *dev, positions=got, token_positions=token_positions.cuda())
    for i, (n, lk) in enumerate(seqs):
        at = int(c.offsets[i])
        c.put(c.k, i, range(lk - n, lk), k[at:at + n])
        c.put(c.v, i, range(lk - n, lk), v[at:at + n])
        positions[i, :, lk - n:lk] = token_positions[at:at + n]
    _same(dev[0], c.k)
    _same(dev[1], c.v)
    assert torch.equal(got.cpu(), positions)


def test_write_one_token_each_from_a_projection():
    """Without offsets; keys and values as views of one projection; positions with fewer slots."""
    c = Cache([(1, 20), (1, 5), (1, 33)], 2, 64, F16)
    qkv = c.normal(3, 8, 64).cuda()
    k, v = qkv[:, 4:6], qkv[:, 6:]
    dev = c.cuda()
    positions = torch.full((3, 2, 20), -1, dtype=torch.int32).cuda()
    paged.cache_write(k, v, *dev[:4], positions=positions, token_positions=torch.tensor([7, 8, 9], dtype=torch.int32).cuda())
    for i, lk in enumerate(c.len):
        c.put(c.k, i, [lk - 1], k[i:i + 1].cpu())
        c.put(c.v, i, [lk - 1], v[i:i + 1].cpu())
    _same(dev[0], c.k)
    _same(dev[1], c.v)
    want = torch.full((3, 2, 20), -1, dtype=torch.int32)
    want[0, :, 19], want[1, :, 4] = 7, 8
    assert torch.equal(positions.cpu(), want)


def test_write_pages_outside_the_pool_and_odd_lengths():
    """Bad pages, lengths below the new tokens' number and past the pages, offsets past the rows: what
    has a place is written, nothing else changes."""
    c = Cache([(4, 40), (6, 3), (5, 70), (2, 20)], 2, 32, BF16, 16)
    c.table[0, 2] = c.k.shape[0] + 5  # slots 32 to 47
    c.table[3, 1] = -2 ** 31
    c.kv_len[2] = 1000  # clamped to the table's slots
    k, v = c.normal(17, 2, 32), c.normal(17, 2, 32)
    c.offsets[4] = 99
    dev = c.cuda()
    before = [x.clone() for x in dev[:2]]
    paged.cache_write(k.cuda(), v.cuda(), *dev)
    room = c.table.shape[1] * 16
    for i, (n, lk, first) in enumerate([(4, 40, 0), (6, 3, 4), (5, room, 10), (2, 20, 15)]):
        for j in range(n):
            if lk - n + j >= 0:
                c.put(c.k, i, [lk - n + j], k[first + j:first + j + 1])
                c.put(c.v, i, [lk - n + j], v[first + j:first + j + 1])
    _same(dev[0], c.k)
    _same(dev[1], c.v)
    assert not torch.equal(_bits(dev[0]), _bits(before[0]))


def test_write_many_sequences():
    """More sequences than a workgroup keeps the offsets of."""
    c = Cache([(i % 3, 5 + i % 3) for i in range(1300)], 1, 8, F16, spare=0)
    t = sum(c.n)
    k, v = c.normal(t, 1, 8), c.normal(t, 1, 8)
    dev = c.cuda()
    paged.cache_write(k.cuda(), v.cuda(), *dev)
    for i, (n, lk) in enumerate(zip(c.n, c.len)):
        at = int(c.offsets[i])
        c.put(c.k, i, range(lk - n, lk), k[at:at + n])
        c.put(c.v, i, range(lk - n, lk), v[at:at + n])
    _same(dev[0], c.k)
    _same(dev[1], c.v)


# -- attention -------------------------------------------------------------------------------

def _attend(c, q, name="", **kw):
    k, v, pages, kv_len, offsets = c.cuda()
    out, lse = paged.paged_attention(q.cuda(), k, v, pages, kv_len, offsets, return_lse=True, **kw)
    want = pref.attention(c, q, **kw)
    t = sum(c.n)
    ref.check(out[:t], want[0], name + " out")
    ref.check(lse[:t], want[1], name + " lse")
    return out, lse


ATTENTION = [
    # dtype, Hq, Hk, D, page, [(new, slots)], options
    (F16, 4, 4, 64, 16, [(1, 77)], {}),
    (BF16, 8, 2, 128, 16, [(1, 1), (1, 40), (1, 500)], {}),
    (BF16, 8, 2, 128, 48, [(1, 5000)], {}),                                    # one token over many ranges
    (F16, 32, 1, 128, 32, [(1, 900), (1, 33)], {}),
    (F16, 48, 1, 64, 16, [(1, 200), (1, 7)], {}),                              # more heads than a wave's rows
    (BF16, 128, 1, 32, 16, [(2, 100)], {}),
    (F16, 6, 2, 72, 16, [(7, 50), (1, 3), (0, 20), (40, 40)], {}),
    (BF16, 5, 1, 80, 64, [(130, 300), (1, 64), (0, 0), (3, 65)], {}),
    (F16, 4, 2, 128, 80, [(300, 300)], {}),                                    # a whole prompt
    (BF16, 2, 2, 96, 16, [(65, 190), (64, 64), (63, 127)], {}),
    (F16, 12, 12, 64, 16, [(33, 290)], {"causal": False}),
    (BF16, 3, 1, 32, 16, [(20, 111), (1, 32)], {"causal": False}),
    (F16, 4, 1, 40, 16, [(9, 31), (50, 200)], {}),
    (BF16, 2, 1, 8, 16, [(3, 19), (1, 16)], {}),
    (F16, 2, 1, 136, 16, [(40, 100), (1, 50)], {}),
    (BF16, 4, 2, 256, 32, [(70, 150)], {}),
    (F16, 4, 2, 256, 16, [(1, 700)], {}),
    (BF16, 8, 2, 64, 16, [(50, 300), (1, 120)], {"left": 37}),
    (F16, 8, 2, 128, 16, [(1, 1000), (1, 90)], {"left": 100}),
    (F16, 4, 2, 64, 32, [(150, 150)], {"left": 0}),
    (BF16, 4, 4, 32, 16, [(60, 200)], {"left": 10, "causal": False}),
    (BF16, 8, 2, 128, 16, [(90, 200), (1, 64)], {"cap": 30.0}),
    (F16, 4, 2, 64, 16, [(40, 100)], {"cap": 0.5}),
    (F16, 4, 2, 64, 16, [(1, 300), (1, 20)], {"cap": 100.0}),
    (BF16, 2, 1, 128, 16, [(33, 80)], {"cap": 100.0, "scale": -0.3}),
    (F16, 2, 1, 64, 16, [(33, 80)], {"scale": -0.2}),
    (F16, 2, 1, 64, 16, [(1, 80)], {"scale": 0.0}),
    (BF16, 4, 2, 96, 16, [(1, 80), (1, 1)], {"cap": 50.0, "left": 20}),
    (F16, 4, 2, 64, 16, [(1, 3 + 5 * (i % 13)) for i in range(100)], {}),       # more sequences than lanes
    (BF16, 2, 2, 64, 16, [((i * 7) % 50 if i % 3 else 0, 50 + i) for i in range(70)], {}),
    (F16, 4, 1, 64, 16, [(40, 300)] + [(1, 20 + i) for i in range(20)], {}),    # few rows a sequence but in one
    (BF16, 8, 2, 128, 32, [(1, 2000 - 31 * i) for i in range(64)], {}),         # as many sequences as lanes
    (F16, 16, 1, 256, 16, [(100, 600), (1, 900)], {}),
]


@pytest.mark.parametrize("dtype,hq,hk,d,page,seqs,kw", ATTENTION)
def test_attention(dtype, hq, hk, d, page, seqs, kw):
    c = Cache(seqs, hk, d, dtype, page)
    _attend(c, c.normal(sum(c.n), hq, d), **kw)


@pytest.mark.parametrize("dtype,hq,hk,d,page,seqs,kw", [
    (F16, 12, 4, 72, 16, [(2001, 2500)], {}),                                  # rows and quads of no eight
    (BF16, 4, 2, 96, 32, [(1500, 1500), (33, 700)], {}),                       # of eight, and not, in one call
    (BF16, 8, 1, 128, 64, [(700, 6000)], {"cap": 20.0}),
    (F16, 3, 3, 40, 16, [(900, 1900), (1, 5000)], {"causal": False}),
    (F16, 2, 2, 256, 16, [(800, 1700)], {"left": 600}),
])
def test_attention_of_row_tiles_that_many_ranges_share(dtype, hq, hk, d, page, seqs, kw):
    c = Cache(seqs, hk, d, dtype, page)
    _attend(c, c.normal(sum(c.n), hq, d), **kw)


def test_attention_counts_alike_for_long_page_tables():
    """Sequences of few pages in a table of 2^20 slots, whose counts are of 64 bits: the same bits."""
    c = Cache([(40, 900), (1, 300), (17, 17), (0, 50)], 16, 64, F16)
    q = c.normal(sum(c.n), 64, 64).cuda()
    k, v, pages, kv_len, offsets = c.cuda()
    table = torch.full((4, 65536), -1, dtype=torch.int32, device="cuda")
    table[:, :pages.shape[1]] = pages
    want = paged.paged_attention(q, k, v, pages, kv_len, offsets, return_lse=True)
    got = paged.paged_attention(q, k, v, table, kv_len, offsets, return_lse=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_evict_without_slots():
    c = Cache([(1, 20), (0, 0)], 2, 64, F16)
    k, v, pages, kv_len, _ = c.cuda()
    new_len, weights, kept, _ = paged.cache_evict(k, v, pages, kv_len, torch.empty(2, 2, 0).cuda(), 5)
    assert (new_len == 0).all() and weights.shape == (2, 2, 0) and (kept == -1).all()


def test_attention_without_offsets_and_heads_first():
    c = Cache([(1, 70), (1, 4), (1, 300)], 2, 64, F16, heads_first=True)
    q = c.normal(3, 6, 64)
    want = _attend(c, q)
    k, v, pages, kv_len, _ = c.cuda()
    got = paged.paged_attention(q.cuda(), k, v, pages, kv_len, return_lse=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_lengths_below_the_new_tokens():
    """Tokens in front of the first slot see nothing: zeros, and -inf."""
    c = Cache([(30, 30), (6, 6), (3, 3)], 1, 64, BF16)
    q = c.normal(sum(c.n), 4, 64)
    k, v, pages, _, offsets = c.cuda()
    kv_len = torch.tensor([10, 0, -5], dtype=torch.int32).cuda()
    out, lse = paged.paged_attention(q.cuda(), k, v, pages, kv_len, offsets, return_lse=True)
    assert torch.equal(out[:20], torch.zeros_like(out[:20])) and (lse[:20] == -math.inf).all()
    assert torch.equal(out[30:], torch.zeros_like(out[30:])) and (lse[30:] == -math.inf).all()
    cut = Cache([(30, 30), (6, 6), (3, 3)], 1, 64, BF16)
    cut.n, cut.len = [10, 0, 0], [10, 0, 0]
    want = pref.attention(cut, q[20:30])
    ref.check(out[20:30], want[0], "out")
    ref.check(lse[20:30], want[1], "lse")


def test_attention_leaves_rows_behind_the_last_sequence():
    c = Cache([(5, 40), (1, 9)], 2, 64, F16)
    q = c.normal(20, 4, 64)
    k, v, pages, kv_len, offsets = c.cuda()
    out = torch.full((20, 4, 64), 3.0, dtype=F16).cuda()
    wide = torch.full((20, 4, 96), 3.0, dtype=F16).cuda()
    paged.paged_attention(q.cuda(), k, v, pages, kv_len, offsets, out=out)
    qw = torch.cat([q, q], 1).cuda()[:, :4]  # strided queries and output
    paged.paged_attention(qw, k, v, pages, kv_len, offsets, out=wide[:, :, :64])
    want = pref.attention(c, q)[0]
    ref.check(out[:6], want, "out")
    assert (out[6:] == 3).all() and (wide[6:] == 3).all() and (wide[:, :, 64:] == 3).all()
    assert torch.equal(wide[:6, :, :64], out[:6])


def test_attention_pages_outside_the_pool_are_zeros():
    c = Cache([(20, 100), (1, 64)], 1, 64, BF16, 16)
    c.table[0, 1], c.table[0, 5], c.table[1, 3] = -3, c.k.shape[0], 2 ** 31 - 1
    _attend(c, c.normal(21, 4, 64))


@pytest.mark.parametrize("d", [32, 128, 256])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_hidden_infinities(dtype, d):
    """Infinities and NaN in K and V: tokens that do not see them are as without, others get what the
    definition gives."""
    for n, lk in ((100, 160), (1, 60)):
        c = Cache([(n, lk), (1, 33)], 2, d, dtype)
        q = c.normal(n + 1, 4, d)
        for slot, value in ((lk - 1, math.inf), (lk - 30, math.nan), (lk - n // 2 - 1, -math.inf)):
            page, at = int(c.table[0, slot // 16]), slot % 16
            c.v[page, at, 0, 3] = value
        c.k[int(c.table[0, (lk - 1) // 16]), (lk - 1) % 16, 1] = math.nan
        _attend(c, q, f"{n} over {lk}")


@pytest.mark.parametrize("dtype,d", [(F16, 64), (F16, 128), (BF16, 128), (BF16, 32)])
def test_attention_scores_that_grow(dtype, d):
    """Scores that rise by hundreds from tile to tile, and fall again; hidden keys are the largest."""
    for n, lk in ((70, 500), (1, 700)):
        c = Cache([(n, lk)], 1, d, dtype)
        for slot in range(lk):
            page, at = int(c.table[0, slot // 16]), slot % 16
            c.k[page, at] *= 0.25 + 4 * min(slot, lk - slot) / lk
        c.k[int(c.table[0, (lk - 1) // 16]), (lk - 1) % 16] *= 8
        _attend(c, c.normal(n, 4, d, std=6.0))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_means_of_the_largest_numbers(dtype):
    """A mean of the type's largest numbers, less the weights' room, is finite."""
    top = 65504.0 if dtype == F16 else 2.0 ** 117
    c = Cache([(40, 300), (1, 3000)], 1, 128, dtype)
    c.v[~torch.isnan(c.v)] = top
    q = c.normal(41, 4, 128)
    k, v, pages, kv_len, offsets = c.cuda()
    out = paged.paged_attention(q.cuda(), k, v, pages, kv_len, offsets)
    assert (out.float() / top - 1).abs().max() <= 2 * ref.UNIT[dtype]


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("depth", [20.0, 200.0])
@pytest.mark.parametrize("dtype,d,n,lk", [(F16, 64, 1, 5000), (BF16, 128, 1, 5000), (BF16, 64, 100, 6000),
                                          (F16, 128, 100, 6000)])
def test_attention_seen_values_of_small_weight(dtype, d, n, lk, depth, bad):
    """A value that is not finite reaches the rows that see it also where its weight rounds to 0 beside
    the others', in its own range of keys or when the ranges are joined."""
    for first, last in ((70, 70), (0, 3000)):  # keys that weigh e^-depth of the others
        c = Cache([(n, lk)], 1, d, dtype)
        q = c.normal(n, 4, d)
        q[..., 0] = 1
        for slot in range(lk):
            c.k[int(c.table[0, slot // 16]), slot % 16, 0, 0] = -depth if first <= slot <= last else 0.0
        c.v[int(c.table[0, 4]), 6, 0, 5] = bad  # slot 70
        k, v, pages, kv_len, offsets = c.cuda()
        out = paged.paged_attention(q.cuda(), k, v, pages, kv_len, offsets, scale=1.0)
        assert not torch.isfinite(out[..., 5]).any(), last
        assert torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 6:]).all(), last


def test_attention_sequences_that_share_pages():
    """A common beginning lies in the cache once."""
    c = Cache([(3, 70), (1, 66)], 2, 64, F16)
    c.table[1, :4] = c.table[0, :4]
    _attend(c, c.normal(4, 4, 64))


def test_attention_same_bits_whatever_the_stream():
    c = Cache([(90, 400), (1, 333), (1, 2000)], 2, 128, BF16)
    q = c.normal(92, 8, 128).cuda()
    dev = c.cuda()
    want = paged.paged_attention(q, *dev, return_lse=True)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        a = paged.paged_attention(q, *dev, return_lse=True)
    b = paged.paged_attention(q, *dev, return_lse=True, stream=side.cuda_stream)
    torch.cuda.synchronize()
    for got in (a, b):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_past_four_gib():
    """Pages whose bytes lie past 32 bits in the pool, and a sequence that mixes near and far ones."""
    page, hk, d = 64, 8, 128
    pool = 2 ** 32 // (page * hk * d * 2) + 300
    g = torch.Generator().manual_seed(3)
    k = torch.empty(pool, page, hk, d, dtype=BF16, device="cuda")
    v = torch.empty(pool, page, hk, d, dtype=BF16, device="cuda")
    places = [pool - 1, 5, pool - 200, 0, pool - 7]
    c = Cache([(40, 300)], hk, d, BF16, page, spare=0, room=0)
    table = torch.tensor([places], dtype=torch.int32).cuda()
    for i, at in enumerate(places):
        k[at], v[at] = c.k[int(c.table[0, i])].cuda(), c.v[int(c.table[0, i])].cuda()
    q = torch.randn(40, 16, d, generator=g).to(BF16)
    out, lse = paged.paged_attention(q.cuda(), k, v, table, c.kv_len.cuda(), c.offsets.cuda(), return_lse=True)
    want = pref.attention(c, q)
    ref.check(out, want[0], "out")
    ref.check(lse, want[1], "lse")
    old = torch.rand(1, hk, 300, generator=g)
    got = paged.key_weights(q.cuda(), k, table, c.kv_len.cuda(), c.offsets.cuda(), lse, old.cuda())
    ref.check(got, pref.weights(c, q, lse.cpu(), old), "weights")
    new = c.normal(40, hk, d)
    paged.cache_write(new.cuda(), new.cuda(), k, v, table, c.kv_len.cuda(), c.offsets.cuda())
    rows = torch.cat([k[at] for at in places])[260:300]
    assert torch.equal(rows.cpu(), new)


# -- key weights -----------------------------------------------------------------------------

def _weigh(c, hq, slots, decay=1.0, q=None, **kw):
    q = c.normal(sum(c.n), hq, c.d) if q is None else q
    k, v, pages, kv_len, offsets = c.cuda()
    lse = pref.attention(c, q, **kw)[1][0].float()
    old = torch.rand(len(c.n), c.hk, slots, generator=c.g) * 3
    got = paged.key_weights(q.cuda(), k, pages, kv_len, offsets, lse.cuda(), old.cuda(), decay=decay, **kw)
    ref.check(got, pref.weights(c, q, lse, old, decay=decay, **kw), "weights")
    return got


@pytest.mark.parametrize("dtype,hq,hk,d,page,seqs,kw", [x for x in ATTENTION])
def test_weights(dtype, hq, hk, d, page, seqs, kw):
    c = Cache(seqs, hk, d, dtype, page)
    _weigh(c, hq, max(c.len) + 5, **kw)


def test_weights_ranges_of_rows_decay_and_fewer_slots():
    """Rows divided among workgroups; slots that end inside a tile; old weights that decay, or are not
    looked at."""
    c = Cache([(1500, 1700), (7, 1000)], 1, 64, F16, 32)
    q = c.normal(1507, 2, 64)
    for slots, decay in ((1700, 0.9), (777, 1.0), (2000, 0.5)):
        _weigh(c, 2, slots, decay, q)
    k, v, pages, kv_len, offsets = c.cuda()
    lse = pref.attention(c, q)[1][0].float()
    odd = torch.full((2, 1, 1700), math.nan)
    got = paged.key_weights(q.cuda(), k, pages, kv_len, offsets, lse.cuda(), odd.cuda(), decay=0.0)
    ref.check(got, pref.weights(c, q, lse, torch.zeros(2, 1, 1700)), "decay 0")


def test_weights_in_place_and_strided():
    c = Cache([(30, 100), (1, 40)], 2, 64, BF16)
    q = c.normal(31, 4, 64)
    dev = c.cuda()
    lse = pref.attention(c, q)[1][0].float().cuda()
    old = torch.rand(2, 2, 120, generator=c.g)
    want = paged.key_weights(q.cuda(), dev[0], *dev[2:], lse, old.cuda())
    wide = torch.zeros(2, 2, 200).cuda()
    wide[:, :, :120] = old.cuda()
    view = wide[:, :, :120]
    got = paged.key_weights(q.cuda(), dev[0], *dev[2:], lse, view, out=view)
    assert got is view and torch.equal(view, want) and (wide[:, :, 120:] == 0).all()


def test_weights_hidden_nan_in_k():
    c = Cache([(80, 130), (1, 20)], 1, 128, F16)
    q = c.normal(81, 4, 128)
    lse = pref.attention(c, q)[1][0].float()
    old = torch.zeros(2, 1, 140)
    want, tol = pref.weights(c, q, lse, old)
    slot = 129  # seen by the last token alone
    c.k[int(c.table[0, slot // 16]), slot % 16] = math.nan
    dev = c.cuda()
    got = paged.key_weights(q.cuda(), dev[0], *dev[2:], lse.cuda(), old.cuda())
    keep = torch.ones(140, dtype=torch.bool)
    keep[slot] = False
    ref.check(got[:, :, keep], (want[:, :, keep], tol[:, :, keep]), "others")
    assert torch.isnan(got[0, 0, slot])


def test_weights_of_tokens_that_saw_nothing():
    c = Cache([(10, 10)], 1, 64, F16)
    q = c.normal(10, 2, 64)
    k, v, pages, _, offsets = c.cuda()
    kv_len = torch.tensor([4], dtype=torch.int32).cuda()
    out, lse = paged.paged_attention(q.cuda(), k, v, pages, kv_len, offsets, return_lse=True)
    got = paged.key_weights(q.cuda(), k, pages, kv_len, offsets, lse, torch.ones(1, 1, 12).cuda())
    assert abs(float(got.sum()) - 8) < 1e-5 and (got[0, 0, 4:] == 0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("dtype,hq,d,n,lk,cap", [
    (F16, 2, 64, 300, 500, 0.0), (BF16, 4, 128, 300, 500, 0.0), (BF16, 1, 256, 300, 300, 30.0), (F16, 3, 40, 200, 333, 100.0),
    (F16, 2, 64, 3, 500, 0.0), (BF16, 4, 128, 7, 500, 30.0), (F16, 8, 256, 4, 90, 0.0),
])
def test_weights_of_tokens_without_a_sum_are_nothing_whatever_they_hold(dtype, hq, d, n, lk, cap, bad):
    """A lse of -inf leaves a token's query out, also one that is not finite, in the middle of others and
    at their end, and keys that are not finite which no one else sees."""
    c = Cache([(n, lk)], 1, d, dtype)
    q = c.normal(n, hq, d)
    lse = pref.attention(c, q, cap=cap)[1][0].float()
    out = [0, n // 2, n - 1] if n > 3 else [1, n - 1]
    lse[out] = -math.inf
    q[out] = 0
    old = torch.rand(1, 1, lk + 9, generator=c.g)
    c.k[int(c.table[0, (lk - 1) // 16]), (lk - 1) % 16] = 0  # seen by the last token alone
    want = pref.weights(c, q, lse, old, cap=cap)
    q[out] = bad
    c.k[int(c.table[0, (lk - 1) // 16]), (lk - 1) % 16] = bad
    k, _, pages, kv_len, offsets = c.cuda()
    got = paged.key_weights(q.cuda(), k, pages, kv_len, offsets, lse.cuda(), old.cuda(), cap=cap)
    ref.check(got, want, "weights")


@pytest.mark.parametrize("group,n", [(1, 40), (4, 70), (8, 3)])
def test_weights_of_queries_that_lie_far_apart(group, n):
    """Queries kept heads first, a head 2^24 values and more after the one before, and tokens as far
    apart: what paged_attention takes."""
    c = Cache([(n, 200)], 1, 64, F16)
    q = c.normal(n, group, 64)
    want = _weigh(c, group, 210, q=q)
    k, v, pages, kv_len, offsets = c.cuda()
    far = 2 ** 24 + 64
    heads = torch.zeros(group * far, dtype=F16, device="cuda").as_strided((n, group, 64), (64, far, 1))
    tokens = torch.zeros(min(n, 5) * far, dtype=F16, device="cuda").as_strided((min(n, 5), group, 64), (far, 64, 1))
    g = torch.Generator().manual_seed(0)
    old = torch.rand(1, 1, 210, generator=g).cuda()
    lse = paged.paged_attention(q.cuda(), k, v, pages, kv_len, offsets, return_lse=True)[1]
    heads.copy_(q)
    a = paged.key_weights(heads, k, pages, kv_len, offsets, lse, old)
    assert torch.equal(a, paged.key_weights(q.cuda(), k, pages, kv_len, offsets, lse, old))
    assert torch.equal(paged.paged_attention(heads, k, v, pages, kv_len, offsets),
                       paged.paged_attention(q.cuda(), k, v, pages, kv_len, offsets))
    if group >= 4:
        few = torch.tensor([0, len(tokens)], dtype=torch.int32).cuda()
        tokens.copy_(q[:len(tokens)])
        b = paged.key_weights(tokens, k, pages, kv_len, few, lse[:len(tokens)], old)
        assert torch.equal(b, paged.key_weights(q[:len(tokens)].cuda(), k, pages, kv_len, few, lse[:len(tokens)], old))


@pytest.mark.parametrize("group,token,head", [(2, 64, 2 ** 29 - 2176), (8, 107374080, 64), (3, 192, 2 ** 28 - 24 * 192)])
def test_weights_of_queries_as_far_apart_as_they_may_be(group, token, head):
    """Strides just below the limit, from memory of up to 2 GiB: (64 / group + 2) token + group head < 2^30."""
    n = 10 if token > 2 ** 20 else 70
    c = Cache([(n, 100)], 1, 64, BF16)
    q = c.normal(n, group, 64).cuda()
    k, v, pages, kv_len, offsets = c.cuda()
    far = torch.empty((n - 1) * token + (group - 1) * head + 64, dtype=BF16, device="cuda")
    far = far.as_strided((n, group, 64), (token, head, 1))
    far.copy_(q)
    lse = paged.paged_attention(q, k, v, pages, kv_len, offsets, return_lse=True)[1]
    old = torch.zeros(1, 1, 100).cuda()
    assert torch.equal(paged.key_weights(far, k, pages, kv_len, offsets, lse, old),
                       paged.key_weights(q, k, pages, kv_len, offsets, lse, old))


# -- eviction --------------------------------------------------------------------------------

EVICT = [
    # Hk, D, page, slots in use, slots, keep, recent, first, positions
    (2, 64, 16, [100, 65, 64, 3, 0], 110, 64, 0, 0, False),
    (1, 128, 16, [2049, 2049, 1000], 2100, 2048, 256, 4, True),
    (3, 8, 48, [500, 300, 77], 520, 100, 30, 2, False),
    (2, 72, 16, [400, 399], 400, 1, 0, 0, False),
    (1, 32, 32, [700], 700, 50, 50, 0, True),            # all protected
    (1, 16, 16, [5000, 4100], 5005, 1500, 100, 1, True),  # rows moved by a kernel of their own
    (1, 8, 64, [9000], 9001, 8990, 0, 0, False),
    (1, 8, 64, [20000], 20000, 3000, 10, 0, True),
    (1, 8, 128, [40000, 39], 40010, 30000, 0, 7, False),  # more slots than registers
    (2, 32, 16, [200], 150, 100, 10, 0, False),           # more slots in use than weights
]


def _evict(c, weights, keep, positions=None, **kw):
    dev = c.cuda()
    got = paged.cache_evict(*dev[:4], weights.cuda(), keep, positions=None if positions is None else positions.cuda(), **kw)
    want = pref.evict(c, weights, keep, positions=positions, **kw)
    for name, a, b in zip(("kv_len", "weights", "kept", "positions"), got, want):
        if b is None:
            assert a is None
        else:
            assert torch.equal(_bits(a) if a.dtype == F32 else a.cpu(), _bits(b) if b.dtype == F32 else b), name
    _same(dev[0], c.k)
    _same(dev[1], c.v)
    return got


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("hk,d,page,lens,slots,keep,recent,first,placed", EVICT)
def test_evict(hk, d, page, lens, slots, keep, recent, first, placed, ties):
    c = Cache([(0, n) for n in lens], hk, d, F16, page)
    weights = torch.rand(len(lens), hk, slots, generator=c.g)
    if ties:
        weights = (weights * 4).floor() - 1
    positions = None
    if placed:
        positions = torch.stack([torch.randperm(3 * slots, generator=c.g)[:slots] for _ in range(len(lens) * hk)])
        positions = positions.reshape(len(lens), hk, slots).to(torch.int32)
    _evict(c, weights, keep, positions, recent=recent, first=first)


def test_evict_odd_weights():
    """NaN comes last, -0 equals 0, infinities and the least numbers have their place."""
    c = Cache([(0, 60), (0, 60)], 2, 32, BF16)
    pool = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-45, -1e-45, 3.4e38, -3.4e38, -math.nan, 1.0])
    weights = pool[torch.randint(0, len(pool), (2, 2, 64), generator=c.g)]
    for keep in (55, 40, 20, 5):
        _evict(c, weights, keep)
    _evict(c, torch.full((2, 2, 64), math.nan), 30)


def test_evict_pages_outside_the_pool():
    c = Cache([(0, 100)], 1, 32, F16)
    c.table[0, 1], c.table[0, 6] = -1, 2 ** 30
    _evict(c, torch.rand(1, 1, 100, generator=c.g), 50)


def test_evict_positions_at_the_ends_of_their_type():
    c = Cache([(0, 40)], 1, 32, F16)
    positions = torch.arange(40, dtype=torch.int32).reshape(1, 1, 40) - 2 ** 31
    _evict(c, torch.rand(1, 1, 40, generator=c.g), 20, positions, recent=5)
    c = Cache([(0, 40)], 1, 32, F16)
    _evict(c, torch.rand(1, 1, 40, generator=c.g), 20, 2 ** 31 - 1 - torch.arange(40, dtype=torch.int32).reshape(1, 1, 40),
           recent=5)


# Caches longer than the registers of the selecting workgroup hold (40960 slots: all of EVICT's are
# shorter), whose weights are read anew in every pass; more than the 8192 moves that are listed at once; rows moved by the
# selecting workgroup itself or by a kernel of their own.
EVICT_LONG = [
    (1, 8, 64, [41500, 70], 41500, 11700, 100, 3, True),   # read anew, two lists of moves
    (1, 8, 128, [50001], 50001, 3000, 0, 0, False),        # the same without positions, one list
    (2, 8, 64, [41100, 41050], 41100, 200, 10, 0, True),   # read anew, few moves
    (1, 8, 64, [40960, 399], 40960, 11700, 0, 5, False),   # in registers, two lists
    (1, 16, 64, [20000], 20100, 250, 50, 0, True),         # in registers, few moves
    (2, 8, 16, [3000, 4000], 4096, 1500, 9, 2, True),      # four slots a lane, a kernel of their own
]


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("hk,d,page,lens,slots,keep,recent,first,placed", EVICT_LONG)
def test_evict_long_caches(hk, d, page, lens, slots, keep, recent, first, placed, ties):
    c = Cache([(0, n) for n in lens], hk, d, F16, page)
    weights = torch.rand(len(lens), hk, slots, generator=c.g)
    if ties:
        weights = (weights * 4).floor() - 1
    positions = None
    if placed:
        positions = torch.stack([torch.randperm(3 * slots, generator=c.g)[:slots] for _ in range(len(lens) * hk)])
        positions = positions.reshape(len(lens), hk, slots).to(torch.int32)
    _evict(c, weights, keep, positions, recent=recent, first=first)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,kw", [(32, {}), (64, {"cap": 30.0}), (96, {}), (128, {"left": 300}), (256, {}),
                                  (72, {"cap": 100.0}), (128, {"causal": False})])
def test_weights_of_few_rows_over_a_ring_of_tiles(dtype, d, kw):
    """Workgroups of six tiles of 32 keys each (more than the ring has): lengths that end in the middle
    of one, a page outside the pool, a sequence with more than 32 rows beside short ones."""
    seqs = [(1, 5120), (40, 900), (1, 3777), (0, 700), (1, 1), (3, 2500)]
    c = Cache(seqs, 32, d, dtype)
    c.table[1, 5], c.table[2, 100] = -1, 2 ** 30
    _weigh(c, 64 if d < 128 else 32, 5120, 0.9, **kw)


MANY = [
    # More sequences than the kernel that counts their tiles takes at once, none of which has new
    # tokens where it goes on to the next.
    (F16, 2, 1, 8, [(0 if 1000 <= i < 1060 else i % 3, 5 + i % 4) for i in range(1300)], {}),
    (BF16, 4, 2, 16, [(1, 1 + i % 20) for i in range(1025)], {"cap": 30.0}),
    # So many that they are looked for in three steps.
    (F16, 1, 1, 8, [(1 if i % 5 else 0, 1 + i % 3) for i in range(4100)], {}),
    # One with more row tiles than lanes: of a wave's rows, and of four waves'.
    (F16, 32, 1, 32, [(1, 9 + i) for i in range(30)] + [(0, 3)] * 69 + [(70, 200)] + [(1, 20)] * 30, {}),
    (BF16, 32, 1, 64, [(0, 3)] * 30 + [(300, 333)] + [(3, 20)] * 40, {"left": 60}),
]


@pytest.mark.parametrize("dtype,hq,hk,d,seqs,kw", MANY)
def test_attention_and_weights_of_many_sequences(dtype, hq, hk, d, seqs, kw):
    c = Cache(seqs, hk, d, dtype, spare=1, room=0)
    q = c.normal(sum(c.n), hq, d)
    _attend(c, q, **kw)
    _weigh(c, hq, max(c.len), q=q, **kw)


# -- together --------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,cap", [(F16, 0.0), (BF16, 30.0)])
def test_a_clip_read_piece_by_piece(dtype, cap):
    """Two clips of different lengths through a cache of 96 slots: every piece is written, looks at the
    cache, leaves its weight, and the cache is cut to 64 slots. Each step against the definition on the
    state that the kernels left."""
    hk, hq, d, page, room, keep = 2, 4, 64, 16, 96, 64
    c = Cache([(0, 0), (0, 0)], hk, d, dtype, page, spare=2 * room // page + 2, room=room // page)
    order = torch.randperm(c.k.shape[0], generator=c.g)[:2 * room // page].reshape(2, -1)
    c.table[:] = order.to(torch.int32)
    k, v, pages, kv_len, _ = c.cuda()
    weights = torch.full((2, hk, room), math.nan).cuda()
    positions = torch.full((2, hk, room), -1, dtype=torch.int32).cuda()
    now = [0, 0]
    for step, new in enumerate([(32, 20), (32, 1), (30, 32), (1, 1), (32, 0), (17, 32), (32, 32)]):
        t = sum(new)
        c.n = list(new)
        c.offsets = torch.tensor([0, new[0], t], dtype=torch.int32)
        kv_len += torch.tensor(new, dtype=torch.int32).cuda()
        c.len = kv_len.tolist()
        place = torch.cat([torch.arange(n, dtype=torch.int32) + p for n, p in zip(new, now)])
        now = [a + b for a, b in zip(now, new)]
        q, nk, nv = c.normal(t, hq, d), c.normal(t, hk, d), c.normal(t, hk, d)
        old = weights.cpu()
        at = c.offsets.cuda()
        paged.cache_write(nk.cuda(), nv.cuda(), k, v, pages, kv_len, at, positions=positions, token_positions=place.cuda())
        out, lse = paged.paged_attention(q.cuda(), k, v, pages, kv_len, at, cap=cap, return_lse=True)
        weights = paged.key_weights(q.cuda(), k, pages, kv_len, at, lse, weights, decay=0.9, cap=cap)
        first = 0
        for i, (n, lk) in enumerate(zip(c.n, c.len)):
            c.put(c.k, i, range(lk - n, lk), nk[first:first + n])
            c.put(c.v, i, range(lk - n, lk), nv[first:first + n])
            first += n
        _same(k, c.k)
        want = pref.attention(c, q, cap=cap)
        ref.check(out, want[0], f"out of piece {step}")
        ref.check(lse, want[1], f"lse of piece {step}")
        ref.check(weights, pref.weights(c, q, lse.cpu(), old, decay=0.9, cap=cap), f"weights of piece {step}")
        old, places = weights.cpu(), positions.cpu()
        kv_len, weights, kept, positions = paged.cache_evict(k, v, pages, kv_len, weights, keep, recent=16, first=4,
                                                             positions=positions)
        want = pref.evict(c, old, keep, recent=16, first=4, positions=places)
        assert torch.equal(kv_len.cpu(), want[0]) and torch.equal(kept.cpu(), want[2])
        assert torch.equal(_bits(weights), _bits(want[1])) and torch.equal(positions.cpu(), want[3])
        _same(k, c.k)
        _same(v, c.v)


def test_a_captured_step_follows_the_lengths():
    """A step of single tokens captured once and replayed as the caches grow and are cut; between the
    replays the program's own eager work."""
    hk, hq, d, room, keep = 2, 4, 64, 256, 200
    c = Cache([(1, 150), (1, 190), (1, 7)], hk, d, F16, room=room // 16)
    for i in range(3):  # pages for the growth
        have = -(-c.len[i] // 16)
        c.table[i, have:] = -1
    pool = c.k.shape[0]
    grown = torch.full((pool + 60, 16, hk, d), math.nan, dtype=F16)
    grown_v = grown.clone()
    grown[:pool], grown_v[:pool] = c.k, c.v
    c.k, c.v = grown, grown_v
    spare = list(range(pool, pool + 60))
    for i in range(3):
        for j in range(room // 16):
            if int(c.table[i, j]) < 0:
                c.table[i, j] = spare.pop()
    k, v, pages, kv_len, _ = c.cuda()
    q, nk, nv = c.normal(3, hq, d).cuda(), c.normal(3, hk, d).cuda(), c.normal(3, hk, d).cuda()
    weights = torch.rand(3, hk, room, generator=c.g).cuda()

    def step():
        paged.cache_write(nk, nv, k, v, pages, kv_len)
        out, lse = paged.paged_attention(q, k, v, pages, kv_len, return_lse=True)
        new = paged.key_weights(q, k, pages, kv_len, None, lse, weights)
        return (out, lse, new) + paged.cache_evict(k, v, pages, kv_len, new, keep, recent=20)

    state = [x.clone() for x in (k, v, kv_len, weights)]

    def reset(values):
        for x, y in zip((k, v, kv_len, weights), values):
            x.copy_(y)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    reset(state)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    with torch.cuda.graph(other):
        again = step()
    for i in range(5):
        reset(state)
        start = [x.clone() for x in state]
        graph.replay()
        torch.cuda.synchronize()
        first = [x.clone() for x in got if x is not None] + [k.clone(), v.clone()]
        reset(start)
        other.replay()
        second = [x.clone() for x in again if x is not None] + [k.clone(), v.clone()]
        reset(start)
        eager = [x for x in step() if x is not None] + [k.clone(), v.clone()]
        torch.cuda.synchronize()
        for a, b, e in zip(first, second, eager):
            assert torch.equal(_bits(a), _bits(e)) and torch.equal(_bits(b), _bits(e)), i
        # The next step: one slot more for each, what the eviction left.
        q.copy_(c.normal(3, hq, d))
        nk.copy_(c.normal(3, hk, d))
        state = [k.clone(), v.clone(), eager[3] + 1, eager[4].clone()]


def test_workspace_given_and_too_small():
    c = Cache([(1, 900)], 1, 64, F16)
    q = c.normal(1, 4, 64).cuda()
    dev = c.cuda()
    want = paged.paged_attention(q, *dev)
    a = _lib.PagedAttentionArgs()
    a.p.batch = a.p.tokens = 1
    a.p.max_pages, a.p.pool_pages, a.p.page_size = dev[2].shape[1], dev[0].shape[0], 16
    a.p.k_heads, a.p.head_dim, a.q_heads, a.left = 1, 64, 4, -1
    a.p.pages = a.p.kv_len = 16
    need = _lib.lib().arthip_paged_attention_workspace(ctypes.byref(a))
    assert need > 0
    workspace = torch.full((need,), 255, dtype=torch.uint8).cuda()
    assert torch.equal(paged.paged_attention(q, *dev, workspace=workspace), want)
    with pytest.raises(EngineError, match="workspace too small"):
        paged.paged_attention(q, *dev, workspace=workspace[:need - 1])


def test_no_tokens():
    c = Cache([(0, 20), (0, 0)], 2, 64, F16)
    dev = c.cuda()
    q = torch.empty(0, 4, 64, dtype=F16).cuda()
    out, lse = paged.paged_attention(q, *dev, return_lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    old = torch.rand(2, 2, 30).cuda()
    got = paged.key_weights(q, dev[0], *dev[2:], lse, old, decay=0.5)
    want = torch.zeros_like(old)
    want[0, :, :20] = old[0, :, :20] * 0.5
    assert torch.equal(got, want)
    paged.cache_write(torch.empty(0, 2, 64, dtype=F16).cuda(), torch.empty(0, 2, 64, dtype=F16).cuda(), *dev)
    _same(dev[0], c.k)
    # Rows, but none of them a sequence's.
    q = torch.zeros(3, 4, 64, dtype=F16).cuda()
    out = torch.full((3, 4, 64), 2.0, dtype=F16).cuda()
    paged.paged_attention(q, *dev, out=out)
    assert (out == 2).all()
