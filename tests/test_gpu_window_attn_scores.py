"""Windowed attention where the running maximum moves: scores far apart in one row, by both forward kernels."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TORCH, TYPE, U32, down, half_step, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [1, 130])
def test_scores_past_2_27(ctx, kind, heads):
    """Two keys four blocks of 32 apart whose scores are 2^27 + 16 and 2^27 + 32 in base 2: the neighbours in f32. Both are exact
    (sums of whole numbers below 2^24, times 16), the second's weight is 1 and the first's 2^-16, every other key's 0. One head runs
    with the keys split, 130 by tiles. o is off by half a step of each weight and of itself."""
    D, sq, sk, a, b = 64, 3, 200, 3, 130
    scale = float(np.float32(11.090354919433594))
    assert np.float32(scale) * np.float32(1.4426950408889634) == 16
    q, k = torch.zeros((1, sq, heads, D)), torch.zeros((1, sk, heads, D))
    q[..., 0], q[..., 1] = 2048, 1
    k[:, a, :, 0], k[:, a, :, 1], k[:, b, :, 0], k[:, b, :, 1] = 4096, 1, 4096, 2
    g = torch.Generator().manual_seed(3)
    v = torch.randn((1, sk, heads, D), generator=g).to(TORCH[kind])
    sq_all = sq if heads == 1 else 40   # (more queries than the few that always split)
    q = q[:, :1].expand(1, sq_all, heads, D)
    attn = sa3k.WindowAttn(ctx, TYPE[kind], 1, heads, heads, sq_all, sk, D, scale=scale)
    o, lse = ctx.zeros((1, sq_all, heads, D), np.uint16), ctx.zeros((1, heads, sq_all))
    attn.forward(up(ctx, q.to(TORCH[kind])), up(ctx, k.to(TORCH[kind])), up(ctx, v), o, lse)
    va, vb = v[0, a].double(), v[0, b].double()
    want = (vb + 2.0 ** -16 * va) / (1 + 2.0 ** -16)
    tol = 2 * half_step(kind) * (vb.abs() + 2.0 ** -16 * va.abs()) + 64 * U32 * (va.abs() + vb.abs())
    got = down(o, kind).double()[0]
    assert bool(((got - want).abs() <= tol).all()), float((got - want).abs().max())
    assert np.array_equal(lse.numpy(), np.full((1, heads, sq_all), 2.0 ** 27 + 32, np.float32))
