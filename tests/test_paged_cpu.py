"""The paged cache's host side, without a GPU: the C entry points refuse arguments that would
read or write out of range before any launch, the Python calls refuse tensors that do not fit,
calls without sequences succeed."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from arthip_amd import _lib, paged
from arthip_amd.engine import EngineError

BUF = 1 << 20  # stands for a device buffer; never read here
MANY = 1 << 40  # bytes of a workspace, more than any call needs


def _set(args, **fields):
    for name, value in fields.items():
        to = args.p if hasattr(type(args.p), name) else args
        setattr(to, name, value)
    return args


def _refused(fn, args, text):
    assert fn(ctypes.byref(args), None) == 1
    assert text in _lib.last_error(), _lib.last_error()


def _base(a, **change):
    _set(a, pages=BUF, kv_len=BUF * 2, q_offsets=BUF * 3, pages_stride=9, batch=2, tokens=5, max_pages=9, pool_pages=20,
         page_size=16, k_heads=2, head_dim=64, dtype=0, k_cache=BUF * 5, k_cache_stride=(2048, 128, 64))
    return _set(a, **change)


def _write(**change):
    a = _base(_lib.CacheWriteArgs(), k=BUF * 6, v=BUF * 7, v_cache=BUF * 8, v_cache_stride=(2048, 128, 64),
              k_stride=(128, 64), v_stride=(128, 64), positions=BUF * 9, token_positions=BUF * 10,
              positions_stride=(200, 100), slots=100)
    return _set(a, **change)


def _attention(**change):
    a = _base(_lib.PagedAttentionArgs(), q=BUF * 6, out=BUF * 7, v_cache=BUF * 8, v_cache_stride=(2048, 128, 64),
              workspace=BUF * 9, workspace_bytes=MANY, q_stride=(256, 64), out_stride=(256, 64), scale=0.1, q_heads=4,
              causal=1, left=-1)
    return _set(a, **change)


def _weights(**change):
    a = _base(_lib.KeyWeightsArgs(), q=BUF * 6, lse=BUF * 7, weights=BUF * 8, out=BUF * 9, workspace=BUF * 10,
              workspace_bytes=MANY, q_stride=(256, 64), weights_stride=(200, 100), out_stride=(200, 100), scale=0.1,
              decay=1.0, q_heads=4, causal=1, left=-1, slots=100)
    return _set(a, **change)


def _evict(**change):
    a = _base(_lib.CacheEvictArgs(), v_cache=BUF * 6, v_cache_stride=(2048, 128, 64), weights=BUF * 7, new_len=BUF * 8,
              weights_out=BUF * 9, kept=BUF * 10, weights_stride=(200, 100), slots=100, keep=64, recent=8, first=2)
    return _set(a, **change)


CALLS = [("arthip_cache_write", _write), ("arthip_paged_attention", _attention), ("arthip_key_weights", _weights),
         ("arthip_cache_evict", _evict)]


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "type"), (dict(batch=-1), "negative"), (dict(max_pages=-1), "negative"),
    (dict(pool_pages=-1), "negative"), (dict(batch=65537, tokens=65537), "sequences"), (dict(k_heads=0), "k_heads"),
    (dict(head_dim=60), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(head_dim=264), "head_dim"),
    (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"), (dict(page_size=65552), "page_size"),
    (dict(max_pages=2 ** 26 + 1), "too many tokens"), (dict(kv_len=None), "null lengths"), (dict(pages=None), "null pages"),
    (dict(pages=BUF + 2), "misaligned"), (dict(kv_len=BUF + 1), "misaligned"),
])
@pytest.mark.parametrize("name,make", CALLS)
def test_page_refusals(name, make, change, text):
    _refused(getattr(_lib.lib(), name), make(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(k_cache=None), "null k_cache"), (dict(k_cache=BUF + 8), "aligned"),
    (dict(k_cache_stride=(2048, 132, 64)), "multiples of 8"), (dict(k_cache_stride=(2048, 2 ** 24 + 8, 64)), "slot's stride"),
    (dict(k_cache_stride=(2048, -128, 64)), "slot's stride"), (dict(k_cache_stride=(-2048, 128, 64)), "page's stride"),
    (dict(k_cache_stride=(2 ** 30 + 8, 128, 64)), "page's stride"),
    (dict(page_size=128, k_cache_stride=(2048, 2 ** 24, 64)), "slots within"),
])
@pytest.mark.parametrize("name,make", CALLS)
def test_pool_refusals(name, make, change, text):
    _refused(getattr(_lib.lib(), name), make(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(tokens=-1), "negative"), (dict(tokens=2 ** 30 + 1), "too many tokens"),
    (dict(q_offsets=None), "one token"), (dict(q_offsets=BUF + 3), "misaligned"),
])
@pytest.mark.parametrize("name,make", CALLS[:3])
def test_offset_refusals(name, make, change, text):
    _refused(getattr(_lib.lib(), name), make(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "null key"), (dict(v=BUF + 4), "aligned"), (dict(k_stride=(128, 60)), "multiples of 8"),
    (dict(v_cache=None), "null v_cache"), (dict(v_cache=BUF * 5), "overlap"), (dict(k=BUF * 5), "overlap"),
    (dict(k_cache_stride=(0, 128, 64)), "zero stride"), (dict(v_cache_stride=(2048, 0, 64)), "zero stride"),
    (dict(v_cache_stride=(2048, 128, 0)), "zero stride"), (dict(token_positions=None), "come together"),
    (dict(positions=BUF + 2), "misaligned"), (dict(positions_stride=(0, 100)), "zero stride"), (dict(slots=-1), "slots"),
])
def test_write_refusals(change, text):
    _refused(_lib.lib().arthip_cache_write, _write(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(q_heads=3), "multiple of k_heads"), (dict(q_heads=-2), "multiple of k_heads"),
    (dict(q_heads=258), "128 query heads"), (dict(tokens=2 ** 24, q_heads=256), "too many tokens"),
    (dict(left=-2), "window"), (dict(left=2 ** 30 + 1), "window"), (dict(causal=2), "causal"),
    (dict(scale=math.nan), "scale"), (dict(cap=-1.0), "cap"), (dict(cap=math.inf), "cap"), (dict(q=BUF + 8), "aligned"),
    (dict(q_stride=(252, 64)), "multiples of 8"), (dict(out=BUF * 5), "overlap"), (dict(out=BUF * 6), "overlap"),
    (dict(workspace_bytes=16), "workspace too small"), (dict(workspace=None), "workspace too small"),
    (dict(workspace=BUF + 4), "misaligned workspace"),
])
@pytest.mark.parametrize("name,make", CALLS[1:3])
def test_score_refusals(name, make, change, text):
    if name == "arthip_key_weights" and ("workspace" in str(change)):
        change = dict(change, tokens=100000, slots=4096, weights_stride=(8192, 4096), out_stride=(8192, 4096))
    _refused(getattr(_lib.lib(), name), make(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "null query"), (dict(out=None), "null query"), (dict(out=BUF + 2), "aligned"),
    (dict(out_stride=(0, 64)), "zero stride"), (dict(out_stride=(256, 0)), "zero stride"), (dict(lse=BUF + 2), "misaligned"),
    (dict(v_cache=None), "null v_cache"), (dict(v_cache_stride=(2048, 128, 4)), "multiples of 8"),
    (dict(out=BUF * 8), "overlap"),
])
def test_attention_refusals(change, text):
    _refused(_lib.lib().arthip_paged_attention, _attention(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(q_heads=0), "no query heads"), (dict(slots=-1), "slots"), (dict(batch=65536, k_heads=1024, q_heads=1024), "too large"),
    (dict(decay=math.inf), "decay"), (dict(out=None), "null output"), (dict(weights=None), "null weights"),
    (dict(out=BUF + 2), "misaligned"), (dict(lse=BUF + 1), "misaligned"), (dict(out_stride=(0, 100)), "zero stride"),
    (dict(out=BUF * 8, out_stride=(400, 100)), "in place"), (dict(out=BUF * 7), "overlap"), (dict(lse=None), "null queries"),
    (dict(q_stride=(-256, 64)), "strides of q"), (dict(q_heads=2, q_stride=(2 ** 24, 64)), "too far apart"),
])
def test_weights_refusals(change, text):
    _refused(_lib.lib().arthip_key_weights, _weights(**change), text)


@pytest.mark.parametrize("change,text", [
    (dict(keep=0), "keep"), (dict(keep=-5), "keep"), (dict(recent=-1), "recent"), (dict(recent=63), "recent"),
    (dict(first=-1), "recent"), (dict(slots=-1), "slots"), (dict(weights=None), "null weights"), (dict(kept=None), "null kept"),
    (dict(positions_out=BUF * 11), "without positions"), (dict(kept=BUF + 2), "misaligned"),
    (dict(v_cache=BUF * 5), "overlap"), (dict(new_len=BUF * 2), "overlap"), (dict(weights_out=BUF * 7), "overlap"),
    (dict(k_cache_stride=(2048, 0, 64)), "zero stride"), (dict(batch=65536, k_heads=1024), "too large"),
])
def test_evict_refusals(change, text):
    _refused(_lib.lib().arthip_cache_evict, _evict(**change), text)


def test_nothing_to_do():
    lib = _lib.lib()
    for name, make in CALLS:
        a = make(batch=0, tokens=0, pages=None, kv_len=None, q_offsets=None, k_cache=None)
        assert getattr(lib, name)(ctypes.byref(a), None) == 0, _lib.last_error()
        assert getattr(lib, name)(None, None) == 1 and "null" in _lib.last_error()
    assert lib.arthip_paged_attention(ctypes.byref(_attention(tokens=0, q=None, out=None, workspace=None)), None) == 0
    assert lib.arthip_paged_attention(ctypes.byref(_attention(q_heads=0, q=None, out=None, workspace=None)), None) == 0
    assert lib.arthip_cache_write(ctypes.byref(_write(tokens=0, k=None, v=None)), None) == 0
    assert lib.arthip_key_weights(ctypes.byref(_weights(slots=0, out=None, weights=None)), None) == 0


def test_evict_without_slots_still_writes():
    """new_len and kept are written whatever the slots: their buffers have to be there."""
    call = _lib.lib().arthip_cache_evict
    _refused(call, _evict(slots=0, weights=None, kept=None), "null kept")
    _refused(call, _evict(slots=0, kept=BUF + 2), "misaligned")
    _refused(call, _evict(slots=0, new_len=BUF * 2), "overlap")
    _refused(call, _evict(slots=0, batch=65536, k_heads=1024), "too large")


def test_workspaces():
    """Of sizes alone; none for calls that are refused."""
    lib = _lib.lib()
    attention = lambda **c: lib.arthip_paged_attention_workspace(ctypes.byref(_attention(**c)))  # noqa: E731
    weights = lambda **c: lib.arthip_key_weights_workspace(ctypes.byref(_weights(**c)))  # noqa: E731
    assert attention() > 0 and attention(workspace=None, q=None) == attention()
    assert attention(batch=100) > attention(batch=64)
    for change in (dict(tokens=0), dict(batch=0, tokens=0), dict(q_heads=3), dict(head_dim=300), dict(tokens=2 ** 31 - 1)):
        assert attention(**change) == 0
    assert weights() == 0 and weights(tokens=100000, slots=4096) > 0 and weights(q_heads=0) == 0
    assert lib.arthip_paged_attention_workspace(None) == 0 and lib.arthip_key_weights_workspace(None) == 0


def test_python_refusals_without_a_gpu():
    k = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    pages, kv_len = torch.zeros(1, 3, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 64, dtype=torch.float16)
    weights = torch.zeros(1, 2, 48)
    for call in (lambda: paged.cache_write(q[:, :2], q[:, :2], k, k.clone(), pages, kv_len),
                 lambda: paged.paged_attention(q, k, k.clone(), pages, kv_len),
                 lambda: paged.key_weights(q, k, pages, kv_len, None, q[:, :, 0].float(), weights),
                 lambda: paged.cache_evict(k, k.clone(), pages, kv_len, weights, 16)):
        with pytest.raises(EngineError, match="on a GPU"):
            call()
    with pytest.raises(EngineError, match="whole number"):
        paged.cache_evict(k, k, pages, kv_len, weights, 1.5)
    with pytest.raises(EngineError, match="must be a number"):
        paged.paged_attention(q, k, k, pages, kv_len, cap="x")
    with pytest.raises(EngineError, match="whole number"):
        paged.paged_attention(q, k, k, pages, kv_len, left=2 ** 40)


def test_structs_have_the_headers_sizes(tmp_path):
    """The ctypes mirrors against a C compiler's view of include/arthip.h."""
    import shutil
    import subprocess
    from pathlib import Path
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    names = {"arthip_pages": "Pages", "arthip_cache_write_args": "CacheWriteArgs",
             "arthip_paged_attention_args": "PagedAttentionArgs", "arthip_key_weights_args": "KeyWeightsArgs",
             "arthip_cache_evict_args": "CacheEvictArgs"}
    lines = []
    for c, py in names.items():
        for field, *_ in getattr(_lib, py)._fields_:
            lines.append(f'printf("%zu ", offsetof({c}, {field}));')
        lines.append(f'printf("%zu\\n", sizeof({c}));')
    src = tmp_path / "sizes.c"
    header = Path(__file__).resolve().parents[1] / "include" / "arthip.h"
    src.write_text(f'#include <stddef.h>\n#include <stdio.h>\n#include "{header}"\nint main(void) {{\n' + "\n".join(lines) +
                   "\nreturn 0;\n}\n")
    subprocess.run(["gcc", "-o", str(tmp_path / "sizes"), str(src)], check=True)
    got = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, py in zip(got, names.values()):
        t = getattr(_lib, py)
        want = [getattr(t, f).offset for f, *_ in t._fields_] + [ctypes.sizeof(t)]
        assert [int(x) for x in line.split()] == want, py


@pytest.mark.parametrize("change,text", [
    (dict(q_stride=(256, -64)), "strides of q"), (dict(q_stride=(2 ** 30 + 8, 64)), "strides of q"),
    (dict(q_stride=(256, 2 ** 62)), "strides of q"), (dict(q_stride=(64, 2 ** 29)), "too far apart"),
    (dict(q_stride=(2 ** 25, 64)), "too far apart"),
])
def test_weights_refuse_queries_past_32_bits(change, text):
    """34 tokens and two heads apart at most, as two query heads share a key head."""
    _refused(_lib.lib().arthip_key_weights, _weights(**change), text)


def test_the_key_weights_plan(tmp_path):
    """key_weights_plan, host code of the built library (tests/key_weights_plan.cc)."""
    import shutil
    import subprocess
    from pathlib import Path
    gxx = shutil.which("g++")
    if gxx is None or not Path("/opt/rocm/include/hip/hip_runtime.h").exists():
        pytest.skip("g++ or the HIP headers are not available")
    _lib.lib()
    here = Path(__file__).resolve().parent
    exe = tmp_path / "key_weights_plan"
    subprocess.run([gxx, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I",
                    str(here.parent / "arthip_amd" / "csrc"), str(here / "key_weights_plan.cc"), str(_lib.LIB_PATH),
                    f"-Wl,-rpath,{_lib.LIB_PATH.parent}", "-L/opt/rocm/lib", "-Wl,-rpath,/opt/rocm/lib", "-o", str(exe)],
                   check=True, capture_output=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
