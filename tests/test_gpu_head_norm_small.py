"""Head norms of very small heads without eps, whose mean square is no normal f32: against the formulas in 64 bits.

A square and a sum below 2^-126 are whole multiples of 2^-149: each of a head's D squares, D additions and the mean is off by half a step,
2^-150, so the mean by (2 D + 1) 2^-150 / D + 2^-150 < 2^-148, and r by half of 2^-148 / mean of itself, beside the rounding of the
result and 40 U of the head's largest (U = 2^-24)."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TORCH, TYPE, U32, down, draw, half_step, up

pytestmark = pytest.mark.gpu
SIZES = [1.0, 1e-17, 2e-19, 1e-19, 5e-20, 1e-20, 3e-21]


def inputs(kind, D):
    """[1][tokens][3 heads][D], each head of its own size"""
    x = draw(1, (1, len(SIZES), 3, D), 1.0, 0.0, "f32").double()
    x = x / x.square().mean(3, keepdim=True).sqrt()
    size = torch.tensor(SIZES, dtype=torch.float64)
    size = torch.stack([size, size.roll(1), size.roll(3)], 1)[None, :, :, None]
    return (x * size).to(TORCH[kind])


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("D", [24, 64, 128, 256])
def test_small_heads_without_eps(ctx, kind, D):
    x = inputs(kind, D)
    B, S, H, _ = x.shape
    n = sa3k.HeadNorm(ctx, TYPE[kind], B, S, H, H, D, 0, eps=0.0)
    el = np.uint16 if kind == "bf16" else np.float32
    y, yk = ctx.zeros(x.shape, el), ctx.zeros(x.shape, el)
    X = up(ctx, x)
    n.forward(X, X, None, None, y, yk)
    x64 = x.double()
    mean = x64.square().mean(3, keepdim=True)
    r = 1 / mean.sqrt()
    want, off = x64 * r, 2.0 ** -149 / mean
    tol = half_step(kind) * want.abs() + (40 * U32 + off) * want.abs().amax(3, keepdim=True)
    for o in (y, yk):
        got = down(o, kind, x.shape).double()
        assert bool(((got - want).abs() <= tol).all()), float((got - want).abs().max())
    dy = draw(2, x.shape, 1.0, 0.0, kind)
    dx, dk, dg = ctx.zeros(x.shape, el), ctx.zeros(x.shape, el), ctx.zeros(D)
    n.backward(X, X, up(ctx, dy), up(ctx, dy), None, None, dx, dk, dq_gain=dg)
    h = dy.double()
    m = (h * want).mean(3, keepdim=True)
    full = r * (h - want * m)
    # r is off by `off`, x r likewise and its mean; the mean's sum by 24 U of its absolute terms
    big = r * (h.abs() + want.abs() * (h * want).abs().mean(3, keepdim=True)).amax(3, keepdim=True)
    tol = half_step(kind) * full.abs() + (40 * U32 + 4 * off) * big
    for o in (dx, dk):
        got = down(o, kind, x.shape).double()
        assert bool(((got - full).abs() <= tol).all()), float(((got - full).abs() / big).max())
    terms = h * want
    err = (torch.from_numpy(dg.numpy()).double() - terms.sum((0, 1, 2))).abs()
    assert bool((err <= ((64 * U32 + off) * terms.abs()).sum((0, 1, 2))).all())
