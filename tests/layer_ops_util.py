"""What the layer operators' tests share: tensors of any of their types on the device, pitched and offset ones,
and the half step of a type."""
import numpy as np
import torch

from conftest import sa3k

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TYPE = {"f32": sa3k.TYPE_F32, "f16": sa3k.TYPE_F16, "bf16": sa3k.TYPE_BF16}
U32 = 2.0 ** -24   # half a step of f32


def half_step(kind):
    return torch.finfo(TORCH[kind]).eps / 2


def draw(seed, shape, sd=1.0, mean=0.0, kind="f32"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * sd + mean).to(TORCH[kind])


def up(ctx, t):
    """a host tensor on the device"""
    t = t.contiguous()
    a = t.view(torch.int16).numpy().view(np.uint16) if t.element_size() == 2 else t.numpy()
    return ctx.upload(a)


def down(a, kind, shape=None):
    """a device array as a tensor of the type"""
    n = a.numpy()
    t = torch.from_numpy(n.view(np.int16)).view(TORCH[kind]) if kind != "f32" else torch.from_numpy(n)
    return t.reshape(shape) if shape is not None else t


class Pitched:
    """rows [rows][cols] in a wider device buffer, `off` elements into it, sentinel values around them"""

    SENTINEL = -77.0

    def __init__(self, ctx, t, ld, off=0):
        rows, cols = t.shape
        self.rows, self.cols, self.ld, self.off = rows, cols, ld, off
        self.kind = {v: k for k, v in TORCH.items()}[t.dtype]
        self.host = torch.full((off + rows * ld + 8,), self.SENTINEL, dtype=t.dtype)
        self.host[off:off + rows * ld].view(rows, ld)[:, :cols] = t
        self.buf = up(ctx, self.host)
        self.ptr = self.buf.ptr + off * t.element_size()

    def get(self):
        """the rows; checks that nothing around them was written"""
        now = down(self.buf, self.kind).clone()
        body = now[self.off:self.off + self.rows * self.ld].view(self.rows, self.ld)
        got = body[:, :self.cols].clone()
        body[:, :self.cols] = self.SENTINEL
        assert bool((now == self.SENTINEL).all()), "written outside the rows"
        return got
