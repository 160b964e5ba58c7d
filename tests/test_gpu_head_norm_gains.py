"""The gradients of the head norms' gains on the GPU: exact on whole numbers, and within what one lane adds otherwise.

Heads of +-1 (or +-2) have a mean square of 1 (or 4) exactly where head_dim is a power of two, and without eps r = 1 (or 1/2): x r is +-1,
the gradient's terms are whole, their sums stay below 2^24 and f32 holds them whatever the order. So a row, head or lane left out
or added twice shows. Positions are 0, whose turn is exact."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TYPE, U32, draw, up
from test_gpu_head_norm import CASES, heads, positions, rotated

pytestmark = pytest.mark.gpu

# batch, tokens, heads, kv, dim, rot, lengths: one to several parts a row, one to several rounds a workgroup
WHOLE = [(1, 1, 1, 1, 8, 0, None), (2, 2050, 3, 1, 64, 16, [2050, 77]), (1, 4, 70, 33, 128, 64, None), (1, 700, 25, 13, 64, 64, None),
         (3, 683, 16, 2, 128, 64, [683, 600, 1]), (1, 9000, 2, 1, 32, 32, None), (2, 1030, 7, 3, 256, 256, None), (1, 333, 97, 1, 16, 16, None),
         (1, 20000, 1, 1, 8, 0, None)]


def signs(seed, shape, size=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 2, shape, generator=g) * 2 - 1).float() * size


def run(ctx, kind, q, k, dq, dk, D, rot, base, eps, gains, pos, lens, near=False, old=None):
    B, S = q.shape[:2]
    el = np.uint16 if kind != "f32" else np.float32
    n = sa3k.HeadNorm(ctx, TYPE[kind], B, S, q.shape[2], k.shape[2], D, rot, neighbours=near, eps=eps, rope_base=base)
    dg = [up(ctx, torch.full((D,), 7.0) if old is None else o) for o in (old or (None, None))]
    n.backward(*[up(ctx, t) for t in (q, k, dq, dk)], *[None if g is None else up(ctx, g) for g in gains], ctx.zeros(q.shape, el),
               ctx.zeros(k.shape, el), dq_gain=dg[0], dk_gain=dg[1], pos=None if pos is None else ctx.upload(pos.numpy()),
               len=None if lens is None else ctx.upload(np.array(lens, np.int32)), accumulate=old is not None)
    return [torch.from_numpy(d.numpy()).double() for d in dg]


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("c", WHOLE, ids=lambda c: "x".join(map(str, c[:6])))
def test_exact_on_whole_numbers(ctx, kind, c):
    B, S, H, K, D, rot, lens = c
    t = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[kind]
    x = [signs(1, (B, S, H, D)), signs(2, (B, S, K, D), 2.0)]
    g = torch.Generator().manual_seed(3)
    dy = [torch.randint(-9, 10, (B, S, n, D), generator=g).float() for n in (H, K)]
    inside = torch.ones(B, S, dtype=torch.bool) if lens is None else torch.arange(S)[None] < torch.tensor(lens)[:, None]
    row = inside[:, :, None, None].double()
    want = [(d.double() * v.double().sign() * row).sum((0, 1, 2)) for v, d in zip(x, dy)]
    pos = torch.zeros((B, S), dtype=torch.int32)
    old = [torch.arange(D, dtype=torch.float32), -torch.arange(D, dtype=torch.float32)]
    for add in (None, old):
        got = run(ctx, kind, *[v.to(t) for v in (*x, *dy)], D, rot, 1e4, 0.0, (draw(5, (D,)), None), pos, lens, old=add)
        for i in range(2):
            assert torch.equal(got[i], want[i] + (0 if add is None else add[i].double()))


def additions(rows, H, K, D, kgroups=3, most=1024):
    """of one chain, for q and for k: a lane's rows and groups, the wave's heads, the waves, a sixteenth of the workgroups' rows, the
    sixteen; as the launch is laid out"""
    lanes = 4 if D <= 32 else 8 if D <= 64 else 16 if D <= 128 else 32
    per = kgroups * (64 // lanes)
    parts = [-(-H // per), -(-K // per)]
    blocks = -(-rows // 4)
    rounds = -(-blocks // max(1, most // sum(parts)))
    grid = -(-blocks // rounds)
    return [rounds * kgroups + 4 + 4 + -(-p * grid // 16) + 16 for p in parts]


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("c", [c for c in CASES if c[1] > 30] + [(2, 1088, 24, 24, 64, 32, False, None, None)], ids=lambda c: "x".join(map(str, c[:6])))
def test_within_a_lanes_additions(ctx, kind, c):
    """a term w x r is off by 16 U of itself and 3 U of its pair's larger w (turned back); every addition of its chain by U of the sum of
    absolute values (U = 2^-24). Where a 16-bit type takes r from the hardware's reciprocal root, 2 U more of the term"""
    B, S, H, K, D, rot, near, lens, how = c
    q, k, _ = heads(kind, c, 1, strange=False)
    dq, dk, _ = heads(kind, c, 11, strange=False)
    pos = positions(how, B, S)
    p64 = torch.arange(S).expand(B, -1) if pos is None else pos
    gains = [draw(5, (D,), 0.3, 1.0), draw(6, (D,), 0.3, 1.0)]
    got = run(ctx, kind, q, k, dq, dk, D, rot, 1e4, 1e-5, gains, pos, lens, near)
    inside = torch.ones(B, S, dtype=torch.bool) if lens is None else torch.arange(S)[None] < torch.tensor(lens)[:, None]
    row = inside[:, :, None, None].double()
    for i, (x, d) in enumerate(((q, dq), (k, dk))):
        x, d = x.double(), d.double() * row
        xh = x / (x.square().mean(3, keepdim=True) + 1e-5).sqrt()
        terms = rotated(d, p64, rot, near, 1e4, -1.0) * xh
        pair = (3 * U32 * 1.5 * d.abs().amax(3, keepdim=True) * xh.abs()).sum((0, 1, 2))
        chain = additions(B * S, H, K, D)[i]
        err = (got[i] - terms.sum((0, 1, 2))).abs()
        bound = (18 + chain) * U32 * terms.abs().sum((0, 1, 2)) + pair
        assert bool((err <= bound).all()), (i, float((err / bound).max()))
