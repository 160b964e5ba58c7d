"""Windowed attention where the running maximum moves: scores far apart in one row, by both forward kernels, and the backward.
Tolerances as in test_gpu_window_attn.py, whose weights' error grows with the scores."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TORCH, TYPE, U32, down, half_step, up
from test_gpu_window_attn import Run, backward_reference, backward_tolerance, check_forward
from window_attn_ref import case, widened

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


# scores of a deviation of 11 (scale 1) to 46 (scale 4) in base 2, 16 and more with heads of 128: a row's maximum moves by more than
# the kernel lets pass several times, and what was summed before counts on
FAR = [
    case("far scores", h=2, sq=150, scale=1.0),
    case("far scores, causal window", h=2, sq=150, causal=True, left=40, sinks=1, scale=2.0),
    case("far scores, heads of 128", h=4, kv=2, d=128, sq=300, left=100, right=100, sinks=70, scale=1.0),
    case("far scores, hundreds", h=2, sq=200, causal=True, scale=4.0),
    case("far scores over a cache", b=2, h=8, kv=2, d=128, sq=1, sk=2000, causal=True, scale=1.0, layout="cache", ql=[1, 1],
         kl=[2000, 517]),
]
WIDE = [w for w in map(widened, FAR) if w]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("c", FAR + WIDE, ids=[c["name"] for c in FAR + WIDE])
def test_forward(ctx, c, kind):
    run = Run(ctx, c, kind, seed=41)
    o, lse = run.forward()
    check_forward(c, kind, o, lse, run.reference())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("c", FAR, ids=[c["name"] for c in FAR])
def test_backward(ctx, c, kind):
    """lse is held in f32: a weight is off by half a step of it on top, U |lse| in base 2"""
    run = Run(ctx, c, kind, seed=41)
    run.forward()
    r = run.reference()
    b = backward_reference(c, r, run.do)
    lse = float(r["lse"][torch.isfinite(r["lse"])].abs().max())
    extra = U32 * lse   # of each weight: ln 2 of it, and as much of ds
    p, sc = r["p"], c["scale"]
    more = (sc * extra * (b["ds"].abs() @ r["k"].abs()), b["fold"](b["T"](b["ds"].abs()) @ r["q"].abs()) * sc * extra,
            b["fold"](b["T"](p) @ b["do"].abs()) * extra)
    for name, got, want, tol, m, lens in zip(("dq", "dk", "dv"), run.backward(), b["grads"], backward_tolerance(c, kind, r, b), more,
                                             (c["ql"], c["kl"], c["kl"])):
        there = torch.stack([torch.arange(got.shape[2]) < n for n in lens])[:, None, :, None].expand_as(got)
        off = ((got - want).abs() - tol - m)[there]
        assert not bool(torch.isnan(off).any()) and float(off.max()) <= 0, (name, float(off.max()))
