"""The example block (examples/clip_attention.py), which runs the transformer operators
together with the package's convs, against the same network in float64 on the CPU."""

from __future__ import annotations

import importlib.util
import math
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

spec = importlib.util.spec_from_file_location(
    "clip_attention", Path(__file__).resolve().parents[1] / "examples" / "clip_attention.py")


def _reference(block, x, scenes):
    frames, h, w, c = x.shape

    def rms(v, weight):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * weight.double().cpu()

    def conv(v, layer):
        weight = torch.from_numpy(layer.weight.astype("float64"))
        return torch.nn.functional.conv2d(v.permute(0, 3, 1, 2), weight, padding=1).permute(0, 2, 3, 1)

    x = x.double().cpu()
    n = frames * h * w
    qkv = conv(rms(x, block.norms[0]), block.qkv).reshape(n, 3, 2, 16)
    q, k, v = qkv.unbind(1)
    grid = torch.stack(torch.meshgrid(*(torch.arange(s) for s in (frames, h, w)), indexing="ij")).reshape(3, n)
    angle = grid.double()[list(block.rope.axis)].T * torch.tensor(block.rope.freqs, dtype=torch.float64)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]

    def turn(t):
        a, b = t[..., :8], t[..., 8:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    s = torch.einsum("ihd,jhd->hij", turn(q), turn(k)) / 4
    s = 20 * torch.tanh(s / 20)
    frame = grid[0]
    s = s - block.slopes.double().cpu()[:, None, None] * (frame[:, None] - frame[None]).abs()
    scene = scenes.cpu()[frame]
    s = torch.where(scene[:, None] == scene[None], s, -math.inf)
    y = torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), v).reshape(frames, h, w, c)
    new = x + torch.tanh(block.gate.double().cpu()) * rms(conv(y, block.project), block.norms[1])
    return new, rms(new, block.norms[2])


@pytest.mark.parametrize("frames,h,w", [(3, 9, 13), (2, 16, 20), (1, 1, 1)])
def test_block_against_float64(frames, h, w):
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    torch.manual_seed(frames * h)
    block = example.ClipBlock(seed=3)
    buf, x = example.padded(frames, h, w)
    x.copy_(torch.randn(frames, h, w, 32, device="cuda"))
    scenes = torch.tensor([7, 7, 2][:frames], dtype=torch.int32, device="cuda")
    new, following = block(x, h, w, scenes)
    want = _reference(block, x, scenes)
    # Five tensors are rounded to fp16 on the way (h, qkv, the turned q and k, y, the
    # branch), each by 2^-11 of values of its own size, and the Winograd convs add a few
    # more; the norm after the branch brings that to values of size 1: 32 times 2^-11
    # of the values' root mean square bounds the whole, elementwise with a factor of 4.
    for got, ref in zip((new, following), want):
        err = (got.double().cpu() - ref).abs()
        size = ref.square().mean().sqrt()
        assert err.square().mean().sqrt() < 32 * 2 ** -11 * size
        assert err.max() < 4 * 32 * 2 ** -11 * size
    # The border of the padded buffers stays zero.
    assert not buf[:, 0].any() and not buf[:, :, 0].any()
