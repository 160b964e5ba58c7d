"""The activations of the fused products where they saturate and beyond: huge values, infinities and NaN, which go through the
formulas as they stand. Forward through a product with K = 1 and weights of 1 (z is the row's one value in every column),
backward through the stored z; a NaN or an infinity stays in its row of dX."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TORCH, TYPE, U32, down, half_step, up

pytestmark = pytest.mark.gpu

ACTS = {"none": sa3k.ACT_NONE, "relu": sa3k.ACT_RELU, "silu": sa3k.ACT_SILU, "gelu": sa3k.ACT_GELU,
        "gelu_tanh": sa3k.ACT_GELU_TANH}
F64 = {"none": lambda z: z, "relu": lambda z: torch.where(z <= 0, torch.zeros_like(z), z), "silu": torch.nn.functional.silu,
       "gelu": torch.nn.functional.gelu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}
NAN, INF = float("nan"), float("inf")
VALUES = {"bf16": [NAN, INF, -INF, 3e38, -3e38, 1e36, -1e36, -1e33, 1e20, -1e20, 5e12, -5e12, -100.0, 100.0, -11.0, 11.0],
          "f16": [NAN, INF, -INF, 65504.0, -65504.0, 3e4, -3e4, 1000.0, -1000.0, -11.0, 11.0]}


def column(kind, M):
    """M rows, the values in turn and 0.5 between them"""
    v = VALUES[kind]
    return torch.tensor([v[i] if i < len(v) else 0.5 for i in range(M)], dtype=torch.float64).to(TORCH[kind])[:, None]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [16, 40])
def test_forward_of_extreme_values(ctx, kind, act, M):
    """y is z, 0, or the formula's NaN: half a step of y, 16 U of it for the factor, and 2^-25 for what underflows"""
    N = 24
    x = column(kind, M)
    y = ctx.zeros((M, N), np.uint16)
    sa3k.linear_act_fwd(ctx, TYPE[kind], ACTS[act], up(ctx, x), up(ctx, torch.ones((N, 1), dtype=TORCH[kind])), M, N, 1, y)
    want, got = F64[act](x.double()).expand(M, N), down(y, kind).double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), (x[:, 0], got[:, 0])
    assert torch.equal(torch.isinf(got), torch.isinf(want)), (x[:, 0], got[:, 0])
    fin = torch.isfinite(want)
    assert bool(((got - want).abs() <= (half_step(kind) + 16 * U32) * want.abs() + 2.0 ** -25)[fin].all()), (x[:, 0], got[:, 0])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("act", list(ACTS))
def test_backward_of_extreme_values(ctx, kind, act):
    """dz = dY act'(z): NaN where z is NaN, and at an infinite z of a smooth activation (0 times infinity in the slope);
    else the slope 0 or 1 to 32 U, rounded"""
    M, N = 40, 24
    z = column(kind, M)
    dy = torch.full((M, N), 1.5, dtype=TORCH[kind])
    dx = ctx.zeros((M, N), np.uint16)
    sa3k.linear_act_bwd(ctx, TYPE[kind], ACTS[act], up(ctx, dy), None, up(ctx, torch.eye(N).to(TORCH[kind])), M, N, N,
                        z=up(ctx, z.expand(M, N)), dx=dx)
    got = down(dx, kind).double()
    v = torch.where(torch.isnan(z.double()), torch.zeros(()).double(), z.double()).requires_grad_()
    F64[act](v).sum().backward()
    smooth = act in ("silu", "gelu", "gelu_tanh")
    nan = (torch.isnan(z) & (act != "none")) | (torch.isinf(z) & smooth)
    assert torch.equal(torch.isnan(got), nan.expand(M, N)), (z[:, 0], got[:, 0])
    want = (1.5 * v.grad).expand(M, N)
    ok = ~nan.expand(M, N)
    assert bool(((got - want).abs() <= (half_step(kind) + 48 * U32) * want.abs() + 48 * U32)[ok].all()), (z[:, 0], got[:, 0])


def test_few_rows_alone(ctx):
    """one row, as a step of one token is: the same values as among others"""
    for act in ("gelu_tanh", "gelu", "silu"):
        got = []
        for v in VALUES["bf16"]:
            y = ctx.zeros((1, 8), np.uint16)
            sa3k.linear_act_fwd(ctx, TYPE["bf16"], ACTS[act], up(ctx, torch.tensor([[v]], dtype=torch.bfloat16)),
                                up(ctx, torch.ones((8, 1), dtype=torch.bfloat16)), 1, 8, 1, y)
            got.append(down(y, "bf16").double()[0])
        want = F64[act](column("bf16", len(got)).double())[:, 0]
        for v, g, w in zip(VALUES["bf16"], got, want):
            same = torch.isnan(g) if bool(torch.isnan(w)) else (g - w).abs() <= 2.0 ** -8 * (1 + 2.0 ** -12) * w.abs() + 2.0 ** -25
            assert bool(same.all()) or bool((g == w).all()), (act, v, g, w)
