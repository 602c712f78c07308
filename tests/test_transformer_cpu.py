"""The transformer operators' host side, without a GPU: the C entry points refuse
arguments that would read or write out of range before any launch, frequencies are
packed in fp64, calls without tokens succeed."""

from __future__ import annotations

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from arthip_amd import _lib
from arthip_amd import transformer as tr
from arthip_amd.engine import EngineError

BUF = 1 << 20  # stands for a device buffer; never read here


def _refused(fn, args, text):
    assert fn(ctypes.byref(args), None) == 1
    assert text in _lib.last_error(), _lib.last_error()


def _set(args, **fields):
    for name, value in fields.items():
        setattr(args, name, value)
    return args


def _attention(**change):
    a = _lib.AttentionArgs()
    _set(a, q=BUF, k=BUF * 2, v=BUF * 3, out=BUF * 4, scale=0.1, left=-1, right=-1, dtype=0, batch=2,
         q_tokens=5, k_tokens=7, q_heads=4, k_heads=2, head_dim=64, q_stride=(1280, 256, 64),
         k_stride=(896, 128, 64), v_stride=(896, 128, 64), out_stride=(1280, 256, 64))
    return _set(a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "type"), (dict(dtype=-1), "type"), (dict(batch=-1), "negative"),
    (dict(q_tokens=-1), "negative"), (dict(k_tokens=-4), "negative"), (dict(k_heads=0), "multiple of k_heads"),
    (dict(q_heads=3), "multiple of k_heads"), (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"),
    (dict(head_dim=264), "head_dim"), (dict(q_tokens=2 ** 30 + 1), "too many tokens"),
    (dict(q_heads=2 ** 20, k_heads=1, q_tokens=2 ** 12), "too many tokens"),
    (dict(batch=2 ** 24, q_tokens=64), "too large"), (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"), (dict(cap=-0.5), "cap"), (dict(cap=math.inf), "cap"),
    (dict(left=-2), "window"), (dict(right=2 ** 30 + 1), "window"), (dict(doc_q=BUF), "come together"),
    (dict(code_k=BUF), "come together"), (dict(table=BUF, table_len=0), "without entries"),
    (dict(table=BUF, table_len=5, table_zero=2 ** 30 + 1), "table_zero"), (dict(q=None), "null"),
    (dict(out=None), "null"), (dict(v=None), "null"), (dict(k=BUF + 8), "aligned"),
    (dict(out=BUF + 2), "aligned"), (dict(q_stride=(1280, 260, 64)), "strides"),
    (dict(v_stride=(896, 128, 4)), "strides"), (dict(lse=BUF + 2), "misaligned"),
    (dict(kv_len=BUF + 1), "misaligned"), (dict(out=BUF), "overlap"), (dict(out=BUF * 3), "overlap"),
    (dict(out_stride=(0, 256, 64)), "zero stride"), (dict(out_stride=(1280, 256, 0)), "zero stride"),
])
def test_attention_refusals(change, text):
    _refused(_lib.lib().arthip_attention, _attention(**change), text)


def test_attention_workspace():
    """Few rows over many keys need one, and a call without it is refused; many rows, or
    few keys, need none."""
    lib = _lib.lib()
    size = lambda a: lib.arthip_attention_workspace(ctypes.byref(a))  # noqa: E731
    assert size(_attention()) == 0
    assert size(_attention(batch=64, q_tokens=4096, k_tokens=4096, q_heads=32, k_heads=8)) == 0
    long = _attention(q_tokens=1, k_tokens=100000)
    need = size(long)
    assert need > 0
    _refused(lib.arthip_attention, long, f"{need} bytes")
    _refused(lib.arthip_attention, _set(long, workspace=BUF * 8, workspace_bytes=need - 1), "workspace")
    _refused(lib.arthip_attention, _set(long, workspace=BUF * 8 + 4, workspace_bytes=need), "misaligned")
    for a in (_attention(k_heads=0), _attention(batch=0), _attention(q_tokens=0), _attention(q_heads=0),
              _attention(batch=-1)):
        assert size(a) == 0
    assert lib.arthip_attention_workspace(None) == 0


def test_calls_without_tokens():
    lib = _lib.lib()
    for change in (dict(batch=0), dict(q_tokens=0), dict(q_heads=0)):
        a = _attention(q=None, k=None, v=None, out=None, **change)
        assert lib.arthip_attention(ctypes.byref(a), None) == 0
    for change in (dict(batch=0), dict(tokens=0)):
        assert lib.arthip_rope_axes(ctypes.byref(_rope(q=None, k=None, **change)), None) == 0
        n = _norm(residual=None, **change)
        assert lib.arthip_gated_norm(ctypes.byref(n), None) == 0
    assert lib.arthip_attention(None, None) == 1 and "null" in _lib.last_error()
    assert lib.arthip_rope_axes(None, None) == 1 and "null" in _lib.last_error()
    assert lib.arthip_gated_norm(None, None) == 1 and "null" in _lib.last_error()


def _rope(**change):
    a = _lib.RopeArgs()
    _set(a, q=BUF, k=BUF * 2, q_out=BUF * 3, k_out=BUF * 4, pos=BUF * 5, packed=BUF * 6, batch=2, tokens=3,
         q_heads=4, k_heads=2, head_dim=64, n_freq=32, dtype=0, q_stride=(768, 256, 64),
         k_stride=(384, 128, 64), q_out_stride=(768, 256, 64), k_out_stride=(384, 128, 64),
         pos_stride=(6, 3, 1))
    return _set(a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "type"), (dict(tokens=-1), "negative"), (dict(k_heads=-1), "negative"),
    (dict(batch=2 ** 16, tokens=2 ** 16), "too many tokens"), (dict(q_heads=65536, k_heads=1), "too many heads"),
    (dict(head_dim=63), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=514), "head_dim"),
    (dict(n_freq=0), "n_freq"), (dict(n_freq=33), "n_freq"), (dict(pairs=2), "0 or 1"),
    (dict(inverse=-1), "0 or 1"), (dict(q=None), "null query"), (dict(k_out=None), "null key"),
    (dict(pos=None), "null positions"), (dict(packed=None), "null positions"), (dict(q=BUF + 1), "misaligned"),
    (dict(packed=BUF + 8), "misaligned"), (dict(pos=BUF + 2), "misaligned"),
    (dict(q_out_stride=(768, 0, 64)), "zero stride"), (dict(k_out_stride=(0, 128, 64)), "zero stride"),
    (dict(q_out=BUF, q_out_stride=(768, 64, 192)), "in place"),
])
def test_rope_refusals(change, text):
    _refused(_lib.lib().arthip_rope_axes, _rope(**change), text)


def test_rope_pack():
    lib = _lib.lib()
    freqs, axis = [1.0, 0.25, 1e-4], [0, 2, 1]
    f, x = (ctypes.c_double * 3)(*freqs), (ctypes.c_int32 * 3)(*axis)
    size = lib.arthip_rope_packed_bytes(3)
    assert size == 48 and lib.arthip_rope_packed_bytes(0) == 0 and lib.arthip_rope_packed_bytes(-1) == 0
    buf = ctypes.create_string_buffer(size)
    assert lib.arthip_rope_pack(f, x, 3, 3, buf, size) == 0
    got = np.frombuffer(buf.raw, dtype=np.dtype([("turns", "<f8"), ("axis", "<i4"), ("pad", "<i4")]))
    np.testing.assert_array_equal(got["turns"], np.array(freqs) / (2 * math.pi))
    np.testing.assert_array_equal(got["axis"], axis)
    for args, text in [((None, x, 3, 3, buf, size), "null"), ((f, x, 0, 3, buf, size), "null"),
                       ((f, x, 3, 3, buf, size - 1), "small"), ((f, x, 3, 2, buf, size), "axis"),
                       (((ctypes.c_double * 3)(1.0, math.nan, 1.0), x, 3, 3, buf, size), "finite")]:
        assert lib.arthip_rope_pack(*args) == 1 and text in _lib.last_error()


def test_rope_plan_frequencies():
    """The plan's frequencies and axes (host logic; the packed copy stays on the CPU)."""
    plan = tr.RopePlan((2, 1, 1), theta=100.0, device="cpu")
    assert plan.axis == (0, 0, 1, 2)
    np.testing.assert_allclose(plan.freqs, [100.0 ** (-f / 4) for f in range(4)], rtol=1e-15)
    plan = tr.RopePlan((2, 1, 1), theta=100.0, order="cycle", per_axis=True, scale=(1, 2, 0.5), device="cpu")
    assert plan.axis == (0, 1, 2, 0)
    np.testing.assert_allclose(plan.freqs, [1, 2, 0.5, 0.1], rtol=1e-15)
    assert tr.RopePlan((1, 1), freqs=(3.0, 4.0), device="cpu").freqs == (3.0, 4.0)
    for kw in (dict(sections=()), dict(sections=(0,)), dict(sections=(-1, 2)), dict(sections=(2,), order="x"),
               dict(sections=(2,), theta=0.0), dict(sections=(2,), scale=(1, 2)), dict(sections=(2,), freqs=(1.0,)),
               dict(sections=(1,), freqs=(math.inf,))):
        with pytest.raises(EngineError):
            tr.RopePlan(kw.pop("sections"), device="cpu", **kw)


def _norm(**change):
    a = _lib.NormArgs()
    _set(a, residual=BUF, y=BUF * 2, residual_out=BUF * 3, h=BUF * 4, batch=2, tokens=3, channels=64, dtype=0,
         residual_dtype=0, post=1, pre=2, gate_act=0, eps=1e-6, residual_scale=1.0, branch_scale=1.0,
         residual_stride=(192, 64), y_stride=(192, 64), residual_out_stride=(192, 64), h_stride=(192, 64))
    return _set(a, **change)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=3), "type"), (dict(dtype=0, residual_dtype=1), "residual type"),
    (dict(dtype=2, residual_dtype=0), "residual type"), (dict(post=3), "unknown norm"),
    (dict(pre=-1), "unknown norm"), (dict(gate_act=4), "activation"), (dict(tokens=-1), "negative"),
    (dict(batch=2 ** 16, tokens=2 ** 15), "too many"), (dict(channels=0), "channels"),
    (dict(channels=32769), "channels"), (dict(eps=-1e-6), "eps"), (dict(eps=math.nan), "eps"),
    (dict(branch_scale=math.inf), "scale"), (dict(residual_scale=math.nan), "scale"),
    (dict(residual=None), "null residual"), (dict(residual_out=None, h=None, pre=0), "no output"),
    (dict(y=None), "without y"), (dict(h=None), "without h"), (dict(h=None, pre=0, mod_shift=BUF), "without h"),
    (dict(residual=BUF + 1), "misaligned"), (dict(y=BUF + 1), "misaligned"), (dict(pre_weight=BUF + 2), "misaligned"),
    (dict(residual_out_stride=(0, 64)), "zero stride"), (dict(h_stride=(192, 0)), "zero stride"),
    (dict(residual_out=BUF, residual_out_stride=(384, 128)), "in place"), (dict(h=BUF), "overlap"),
    (dict(h=BUF * 2), "overlap"), (dict(h=BUF * 3), "overlap"), (dict(residual_out=BUF * 2), "overlap"),
])
def test_norm_refusals(change, text):
    _refused(_lib.lib().arthip_gated_norm, _norm(**change), text)


def test_tensors_must_be_on_a_gpu():
    x = torch.zeros(1, 2, 2, 32, dtype=torch.float16)
    with pytest.raises(EngineError, match="on a GPU"):
        tr.attention(x, x, x)
    with pytest.raises(EngineError, match="on a GPU"):
        tr.rope_axes(x, x, torch.zeros(1, 1, 2, dtype=torch.int32), tr.RopePlan((16,), device="cpu"))
    with pytest.raises(EngineError, match="on a GPU"):
        tr.gated_norm(torch.zeros(1, 2, 64), pre="rms")


# -- the Python layer, with the launch replaced --------------------------------------------

class _Gpu(torch.Tensor):
    """A host tensor that says it is on a GPU; nothing here launches."""
    is_cuda = property(lambda self: True)


def _gpu(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Gpu)


@pytest.fixture
def launches(monkeypatch):
    """The argument structs of the calls made, copied in place of the launch."""
    seen = []
    monkeypatch.setattr(tr, "_plans", {})
    monkeypatch.setattr(tr, "_call", lambda fn, args, device, stream: seen.append(type(args).from_buffer_copy(args)))
    return seen


NUMBERS = [
    ("norm", "eps", 1e-3), ("norm", "residual_scale", 0.25), ("norm", "branch_scale", 2.0),
    ("attention", "scale", 0.75), ("attention", "cap", 7.0), ("attention", "table_zero", 3),
    ("attention", "causal", True), ("rope", "inverse", True),
]


def test_windows_are_read_at_each_call(launches):
    left, right = torch.tensor(5), torch.tensor(2)
    _use("attention", window=(left, right))
    left.fill_(9), right.fill_(0)
    _use("attention", window=(left, right))
    assert [(a.left, a.right) for a in launches] == [(5, 2), (9, 0)]
    for bad in ((1.5, None), ("x", None), (None, torch.ones(2))):
        with pytest.raises(EngineError, match="window"):
            _use("attention", window=bad)


def _use(op, **kw):
    if op == "norm":
        tr.gated_norm(_gpu(1, 2, 64), _gpu(1, 2, 64), pre="rms", **kw)
    elif op == "attention":
        tr.attention(_gpu(1, 4, 2, 32), _gpu(1, 4, 2, 32), _gpu(1, 4, 2, 32), table=_gpu(2, 9, dtype=torch.float32),
                     **kw)
    else:
        plan = tr.RopePlan((16,), device="cpu")
        tr.rope_axes(_gpu(1, 2, 2, 32), None, _gpu(1, 1, 2, dtype=torch.int32), plan, **kw)


@pytest.mark.parametrize("op,name,value", NUMBERS)
def test_numbers_are_read_at_each_call(launches, op, name, value):
    """A parameter of no dimensions that changes in place between two calls counts with the
    value that it has at each."""
    field, first = ("right", -1) if name == "causal" else (name, 0)
    number = torch.zeros((), dtype=torch.tensor(value).dtype)
    _use(op, **{name: number})
    number.copy_(torch.tensor(value))
    _use(op, **{name: number})
    assert getattr(launches[0], field) == first
    assert getattr(launches[1], field) == (0 if name == "causal" else np.float32(value))
    for other in (value, np.array(value)):
        _use(op, **{name: other})
        assert getattr(launches[-1], field) == getattr(launches[1], field)


@pytest.mark.parametrize("op,name,value", [n for n in NUMBERS if n[1] not in ("causal", "inverse")])
@pytest.mark.parametrize("bad", ["much", None, (1.0, 2.0), torch.ones(2)])
def test_numbers_that_are_none(launches, op, name, value, bad):
    if name == "scale" and bad is None:
        return  # 1 / sqrt(D)
    with pytest.raises(EngineError, match=name):
        _use(op, **{name: bad})
    assert not launches


# -- shapes that no operator takes ---------------------------------------------------------

@pytest.mark.parametrize("change", [
    dict(q_heads=2, k_heads=4), dict(q_heads=3, k_heads=2), dict(head_dim=60), dict(head_dim=512),
    dict(q_tokens=2 ** 31 - 1), dict(batch=2 ** 24, q_tokens=64),
])
def test_attention_shapes_without_a_workspace(change):
    """No workspace, and a refusal, for shapes that the call does not take."""
    lib = _lib.lib()
    a = _attention(k_tokens=100000, **change)
    assert lib.arthip_attention_workspace(ctypes.byref(a)) == 0
    assert lib.arthip_attention(ctypes.byref(a), None) == 1


def test_attention_fewer_query_heads_than_key_heads(launches):
    q, k = _gpu(1, 4, 2, 32), _gpu(1, 5000, 4, 32)
    with pytest.raises(EngineError, match="multiple of k_heads"):
        tr.attention(q, k, k)
    with pytest.raises(EngineError, match="multiple of k_heads"):
        tr.attention(_gpu(1, 4, 3, 32), k[:, :, :2], k[:, :, :2])
    assert not launches


@pytest.mark.parametrize("q_tokens", [1, 2 ** 8, 2 ** 9, 2 ** 10, 2 ** 30])
def test_attention_sizes_whose_product_passes_64_bits(q_tokens):
    a = _attention(batch=2 ** 30, q_tokens=q_tokens, q_heads=2 ** 30, k_heads=2 ** 30)
    assert _lib.lib().arthip_attention_workspace(ctypes.byref(a)) == 0
    _refused(_lib.lib().arthip_attention, a, "too large")


@pytest.mark.parametrize("empty", [dict(q_tokens=0), dict(batch=0), dict(q_heads=0)])
def test_calls_without_queries_take_documents_and_codes(empty):
    """An empty tensor has no address: a pair's one side may be NULL where there is nothing to do."""
    lib = _lib.lib()
    for pair in (dict(doc_k=BUF * 8), dict(code_k=BUF * 8), dict(doc_q=BUF * 8, code_q=BUF * 8)):
        a = _attention(**empty, **pair)
        assert lib.arthip_attention(ctypes.byref(a), None) == 0, _lib.last_error()


def test_tensors_that_a_call_makes_belong_to_its_stream(monkeypatch):
    """The handle 0 is the default stream, which no external stream can stand for."""
    import contextlib
    used = []

    class External:
        def __init__(self, handle, device=None):
            assert handle != 0
            self.handle = handle

    class Default:
        handle = 0

    @contextlib.contextmanager
    def on(stream):
        used.append(stream.handle)
        yield

    monkeypatch.setattr(torch.cuda, "ExternalStream", External)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: Default())
    monkeypatch.setattr(torch.cuda, "stream", on)
    for handle in (0, 4096):
        tr._empty((2, 3), torch.float32, torch.device("cpu"), handle)
        tr._like(torch.zeros(2, 3), handle)
    assert used == [0, 0, 4096, 4096]
    tr._empty((2, 3), torch.float32, torch.device("cpu"), None)
    assert len(used) == 4


@pytest.mark.parametrize("kw", [dict(window=(2 ** 32 + 5, None)), dict(window=(None, 2 ** 31)), dict(table_zero=2 ** 32),
                                dict(table_zero=-2 ** 32 + 1)])
def test_whole_numbers_past_32_bits(launches, kw):
    with pytest.raises(EngineError, match="window|table_zero"):
        _use("attention", **kw)
    assert not launches


def test_sizes_past_32_bits(launches):
    """Broadcast tensors can name more entries than a size of the C struct holds."""
    n = 2 ** 32 + 4
    one, two = _gpu(1, 1, 2, 32), _gpu(1, 4, 2, 32)
    long = one.expand(1, n, 2, 32)
    pos = _gpu(1, 1, 1, dtype=torch.int32)
    row, table = _gpu(1, 1, 64), _gpu(2, 1, dtype=torch.float32)
    for call in (lambda: tr.attention(two, long, long), lambda: tr.attention(long, two, two),
                 lambda: tr.rope_axes(long, None, pos.expand(1, 1, n), tr.RopePlan((16,), device="cpu")),
                 lambda: tr.gated_norm(row.expand(1, n, 64), row.expand(1, n, 64), pre="rms"),
                 lambda: tr.gated_norm(row.expand(n, 1, 64), row.expand(n, 1, 64), pre="rms")):
        with pytest.raises(EngineError, match="too"):
            call()
    assert not launches


@pytest.mark.parametrize("kw,text", [
    (dict(docs=torch.zeros(2, 4, dtype=torch.int32)), "docs"), (dict(codes=torch.zeros(4, dtype=torch.int32)), "codes"),
    (dict(docs=(None, None)), "docs"), (dict(docs=(1, 2, 3)), "docs"), (dict(codes=5), "codes"), (dict(docs=()), "docs"),
    (dict(window=5), "window"), (dict(window=(1, 2, 3)), "window"), (dict(window=None), "window"),
    (dict(window=torch.tensor(3)), "window"),
])
def test_pairs_that_are_none(launches, kw, text):
    with pytest.raises(EngineError, match=text):
        _use("attention", **kw)
    assert not launches


def test_lists_are_pairs(launches):
    docs = [_gpu(4, dtype=torch.int32), _gpu(1, 4, dtype=torch.int32)]
    _use("attention", docs=docs, codes=docs, window=[3, 1])
    assert len(launches) == 1 and (launches[0].left, launches[0].right) == (3, 1)


def test_windows_of_any_two_numbers(launches):
    for window in (np.array([3, 1]), torch.tensor([3, 1]), iter((3, 1)), torch.Size((3, 1))):
        _use("attention", window=window)
        assert (launches[-1].left, launches[-1].right) == (3, 1)


@pytest.mark.parametrize("name", ["post", "pre", "gate_act"])
def test_names_that_are_none(launches, name):
    for bad in (["rms"], {"rms": 1}, 5):
        with pytest.raises(EngineError, match="gated_norm"):
            tr.gated_norm(_gpu(1, 2, 64), _gpu(1, 2, 64), **{name: bad})
    assert not launches


def test_launches_of_more_threads_than_one_takes(tmp_path):
    """launch_parts of transformer.h, host code only, built with g++ (tests/launch_parts.cc)."""
    gxx = shutil.which("g++")
    if gxx is None or not Path("/opt/rocm/include/hip/hip_runtime.h").exists():
        pytest.skip("g++ or the HIP headers are not available")
    here = Path(__file__).resolve().parent
    exe = tmp_path / "launch_parts"
    subprocess.run([gxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    str(here.parent / "arthip_amd" / "csrc"), str(here / "launch_parts.cc"), "-o", str(exe)],
                   check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("rows,heads,dim,more,split", [
    (13 * 128, 20, 128, {}, False),  # 260 workgroups of a CU's two: their halves would take three turns
    (16 * 128, 16, 128, {}, True), (20 * 128, 15, 64, {}, True), (20 * 128, 20, 64, {}, False),
    (20 * 128, 15, 64, dict(slopes=BUF * 8), False), (20 * 128, 15, 64, dict(cap=100.0), False),
    (20 * 128, 15, 32, dict(slopes=BUF * 8), True), (1, 512, 128, {}, True), (1, 640, 128, {}, False),
    (13 * 128, 20, 256, {}, True), (16 * 128, 16, 256, {}, False), (25 * 128, 20, 256, {}, False),
    (1, 640, 64, {}, True), (1, 672, 64, {}, False), (1, 576, 48, {}, False), (1, 512, 256, {}, False),
])
def test_attention_divides_long_walks_into_what_the_chip_holds_at_once(rows, heads, dim, more, split):
    a = _attention(batch=1, q_tokens=rows, k_tokens=4096, q_heads=heads, k_heads=heads, head_dim=dim, **more)
    assert (_lib.lib().arthip_attention_workspace(ctypes.byref(a)) > 0) == split


def test_attention_workspace_counts_the_bias(launches):
    """The Python layer sizes the workspace for the call's own arguments."""
    q, k = _gpu(1, 20 * 128, 15, 64), _gpu(1, 4096, 15, 64)
    for kw in (dict(slopes=_gpu(15, dtype=torch.float32)), dict(table=_gpu(15, 5, dtype=torch.float32)), dict(cap=100.0)):
        tr.attention(q, k, k, **kw)
        assert not launches[-1].workspace
    tr.attention(q, k, k)
    assert launches[-1].workspace_bytes > 0
