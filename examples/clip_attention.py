"""An attention block over the frames of a clip, on the conv engine's own activations.

The block stands between the convs of an upscaler: it takes 32-channel features of a
few frames in padded NHWC fp16 (arthip_padded_dims) and lets every patch see its own
scene, across frames:

    h  = norm(x)
    q, k, v = conv3x3(h), two heads of 16        (arthip_conv3x3_f16_nhwc, 32 -> 96)
    q, k turned by (frame, row, column)          (rope_axes)
    y  = attention within a scene, scores capped, nearer frames first  (attention)
    x' = x + tanh(gate) * norm(conv3x3(y)), h' = norm(x')              (gated_norm)

x' goes on as the residual stream, h' into the next layer's conv. Everything runs on
the current stream, on kernels of this package; torch holds the memory.

    python examples/clip_attention.py            # four 48 x 80 frames, two scenes
"""

from __future__ import annotations

import ctypes
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import torch  # noqa: E402

from arthip_amd import _lib, transformer  # noqa: E402
from arthip_amd.models import he_normal  # noqa: E402

C, HEADS, DIM = 32, 2, 16


class Conv:
    """A 3x3 conv on padded NHWC buffers, its filter packed once."""

    def __init__(self, weight: np.ndarray):
        self.m, self.c = weight.shape[:2]
        lib = _lib.lib()
        packed = np.zeros(lib.arthip_conv3x3_packed_halfs(self.m, self.c), np.uint16)
        bias = np.zeros(lib.arthip_conv3x3_bias_len(self.m), np.float32)
        rc = lib.arthip_conv3x3_pack(
            np.ascontiguousarray(weight).view(np.uint16).ctypes.data_as(ctypes.POINTER(ctypes.c_uint16)), None,
            self.m, self.c, packed.ctypes.data_as(ctypes.POINTER(ctypes.c_uint16)), packed.size,
            bias.ctypes.data_as(ctypes.POINTER(ctypes.c_float)), bias.size)
        if rc != 0:
            raise RuntimeError(_lib.last_error())
        self.weight = weight
        self.packed = torch.from_numpy(packed.view(np.float16)).cuda()
        self.bias = torch.from_numpy(bias).cuda()

    def __call__(self, x, h: int, w: int):
        out = torch.zeros(*x.shape[:3], self.m, dtype=torch.float16, device=x.device)
        rc = _lib.lib().arthip_conv3x3_f16_nhwc(
            x.data_ptr(), self.packed.data_ptr(), self.bias.data_ptr(), 0, None, None, out.data_ptr(),
            x.shape[0], h, w, self.c, self.m, torch.cuda.current_stream().cuda_stream)
        if rc != 0:
            raise RuntimeError(_lib.last_error())
        return out


def padded(frames: int, h: int, w: int, channels: int = C):
    """A zeroed activation buffer and the view of its pixels."""
    hp, wp = ctypes.c_int(), ctypes.c_int()
    _lib.lib().arthip_padded_dims(h, w, ctypes.byref(hp), ctypes.byref(wp))
    buf = torch.zeros(frames, hp.value, wp.value, channels, dtype=torch.float16, device="cuda")
    return buf, buf[:, 1:h + 1, 1:w + 1]


class ClipBlock:
    def __init__(self, seed: int = 0):
        rng = np.random.default_rng(seed)
        self.qkv = Conv(he_normal(rng, 3 * C, C))
        self.project = Conv(he_normal(rng, C, C))
        self.norms = [torch.from_numpy(1 + 0.1 * rng.standard_normal(C).astype(np.float32)).cuda() for _ in range(3)]
        self.gate = torch.from_numpy(rng.standard_normal(C).astype(np.float16)).cuda()
        self.slopes = torch.tensor([0.5, 0.125], device="cuda")  # a head, by the distance in frames
        self.rope = transformer.RopePlan((2, 3, 3), per_axis=True, theta=100.0)

    def __call__(self, x, h: int, w: int, scenes):
        """x: the pixels of a padded buffer [frames, h, w, 32]; scenes: int32 [frames].
        Returns (x', h') as such views; h' lies in a padded buffer, ready for a conv."""
        frames = x.shape[0]
        tokens = frames * h * w
        start, pixels = padded(frames, h, w)
        for f in range(frames):  # rows of a frame are batch items: the views keep their strides
            transformer.gated_norm(x[f], pre="rms", pre_weight=self.norms[0], h=pixels[f])
        qkv = self.qkv(start, h, w)[:, 1:h + 1, 1:w + 1].reshape(1, tokens, 3 * HEADS, DIM)
        q, k, v = qkv.split(HEADS, 2)

        t, y, col = torch.meshgrid(*(torch.arange(n, dtype=torch.int32, device="cuda") for n in (frames, h, w)),
                                   indexing="ij")
        pos = torch.stack([t, y, col]).reshape(3, tokens)
        transformer.rope_axes(q, k, pos, self.rope, q_out=q, k_out=k)
        scene = scenes.repeat_interleave(h * w)
        frame = t.reshape(-1).contiguous()
        mixed = transformer.attention(q, k, v, cap=20.0, docs=(scene, scene), codes=(frame, frame), slopes=self.slopes)

        buf, view = padded(frames, h, w)
        view.copy_(mixed.reshape(frames, h, w, C))
        branch = self.project(buf, h, w)[:, 1:h + 1, 1:w + 1]
        _, new = padded(frames, h, w)
        _, following = padded(frames, h, w)
        for f in range(frames):
            transformer.gated_norm(x[f], branch[f], post="rms", post_weight=self.norms[1], gate=self.gate,
                                   gate_act="tanh", pre="rms", pre_weight=self.norms[2], residual_out=new[f],
                                   h=following[f])
        return new, following


def main() -> None:
    frames, h, w = 4, 48, 80
    _, x = padded(frames, h, w)
    x.copy_(torch.randn(frames, h, w, C, device="cuda"))
    scenes = torch.tensor([0, 0, 0, 1], dtype=torch.int32, device="cuda")  # a cut before the last frame
    block = ClipBlock()
    new, following = block(x, h, w, scenes)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(20):
        block(x, h, w, scenes)
    end.record()
    end.synchronize()
    print(f"{frames} frames of {h}x{w}: x' {tuple(new.shape)} rms {new.float().pow(2).mean().sqrt():.3f}, "
          f"h' rms {following.float().pow(2).mean().sqrt():.3f}, {start.elapsed_time(end) / 20:.3f} ms a block")


if __name__ == "__main__":
    main()
