"""gelu of negative z relative to itself: bf16 holds the values down to z = -13 as normal numbers.

The part of a normal distribution beyond |z| is off by at most 2^-19 of itself (the fit's 1.2e-6 in f32 arithmetic and two steps
of the hardware's exponential) and, for the exponential's argument, by 1.5 z^2 U (two products and a constant off by U each, of an
argument of z^2 / 2), U = 2^-24. y adds half a step. A slope adds two such parts of opposite sign, Phi(z) and z phi(z)."""
import math

import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TYPE, U32, down, half_step, up

pytestmark = pytest.mark.gpu


def tail_error(z):
    return 2.0 ** -19 + 1.5 * z * z * U32


@pytest.mark.parametrize("M", [8, 48])
def test_gelu_of_negative_values(ctx, M):
    N = 32
    # -12.9 .. 0, one a row of one column of x: z is exact
    x = -torch.linspace(0.001, 12.9, M, dtype=torch.float64).to(torch.bfloat16)[:, None]
    y = ctx.zeros((M, N), np.uint16)
    sa3k.linear_act_fwd(ctx, TYPE["bf16"], sa3k.ACT_GELU, up(ctx, x), up(ctx, torch.ones((N, 1), dtype=torch.bfloat16)), M, N, 1, y)
    z = x.double()
    want = z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    got = down(y, "bf16").double()
    rel = half_step("bf16") * (1 + tail_error(z)) + tail_error(z) + U32
    assert bool(((got - want).abs() <= rel * want.abs()).all()), float(((got - want) / want).abs().max())


def test_gelu_slope_of_negative_values(ctx):
    """dX = dz W with W = 1 in one column of one output: dz itself"""
    M = 208
    z = -torch.linspace(0.001, 12.9, M, dtype=torch.float64).to(torch.bfloat16)[:, None]
    dx = ctx.zeros((M, 1), np.uint16)
    one = torch.ones((M, 1), dtype=torch.bfloat16)
    sa3k.linear_act_bwd(ctx, TYPE["bf16"], sa3k.ACT_GELU, up(ctx, one), None, up(ctx, one[:1]), M, 1, 1, z=up(ctx, z), dx=dx)
    v = z.double()
    below, bell = 0.5 * torch.special.erfc(-v / math.sqrt(2)), torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
    want = below + v * bell
    e = (tail_error(v) + 4 * U32) * (below + v.abs() * bell)
    got = down(dx, "bf16").double()
    off = (got - want).abs() - (half_step("bf16") * (want.abs() + e) + e)
    assert bool((off <= 0).all()), (float(off.max()), float(v[off.argmax()]))
