"""Gated products with NaN in and around their tensors, and the activations at the end of the large tiles, on the GPU.

Inputs are small whole numbers, whose sums f32 holds exactly, so that every finite result must be the exact one rounded once. Pitch
gaps and the elements before and after each tensor are NaN: a product that lets one in shows it. A NaN inside reaches what the formulas
say, and nothing else."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from gated_shapes import BACKWARD, FORWARD
from layer_ops_util import TORCH, TYPE, U32, down, draw, half_step, up
from test_gpu_gated_linear import ACTS, F64, whole

pytestmark = pytest.mark.gpu
NAN = float("nan")


class InNan:
    """rows at a pitch in a buffer that is NaN before, between and behind them"""

    def __init__(self, ctx, t, gap, before=8):
        self.rows, self.cols = t.shape
        ld = self.cols + gap if gap else -(-self.cols // 8) * 8 + 8
        self.kind, self.ld, self.off = {v: k for k, v in TORCH.items()}[t.dtype], ld, before
        host = torch.full((before + self.rows * self.ld + 16,), NAN, dtype=t.dtype)
        host.as_strided(t.shape, (self.ld, 1), before).copy_(t)
        self.buf = up(ctx, host)
        self.ptr = self.buf.ptr + before * t.element_size()

    def get(self):
        now = down(self.buf, self.kind).clone()
        rows = now.as_strided((self.rows, self.cols), (self.ld, 1), self.off)
        got = rows.clone()
        rows.fill_(NAN)
        assert bool(now.isnan().all()), "written outside the rows"
        return got


def same(got, want):
    """the same numbers, NaN in the same places"""
    want = want.to(got.dtype)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


# M, N, K; the paths: few rows, two blocks of them, 128 and 256 wide tiles, whole and in splits (gated_shapes); odd: pitches and starts
# that no load of 16 bytes, and no dword, is aligned to
FORWARDS = [(1, 33, 40), (16, 100, 256), (5, 17, 7), (32, 304, 520), (17, 40, 1025), (64, 128, 64), (129, 257, 201), (300, 520, 1000),
            (396, 9688, 16), (417, 8435, 316), (155, 8511, 4009)]
BACKWARDS = [(1, 33, 40), (65, 768, 1032), (16, 195, 16), (158, 278, 130), (644, 18, 16), (131, 3914, 8405), (2321, 2250, 1695), (131, 8117, 149)]
assert {s for s in FORWARDS if s in FORWARD} and {s for s in BACKWARDS if s in BACKWARD}
# gap between rows (0: up to the next multiple of 8 and 8 more), elements before the first
LAYOUTS = {"aligned": (8, 8), "odd": (3, 1), "even": (2, 2), "eights": (0, 8)}


def product(a, b):
    """a . b^T in f64, NaN where a row's or a column's is"""
    return a.double() @ b.double().t()


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("M,N,K", FORWARDS)
def test_forward_among_nan(ctx, M, N, K, layout):
    gap, before = LAYOUTS[layout]
    kind = "bf16"
    x, w = whole(1, (M, K), 2, kind), [whole(2 + i, (N, K), 1 if K > 1500 else 2, kind) for i in range(2)]
    if layout != "even":   # a row of x, and one of each weight, hold a NaN: a row and two columns of the result do
        x[M // 2, K // 3] = NAN
        w[0][N // 3, K - 1] = NAN
        w[1][N - 1, 0] = NAN
    g, u = (product(torch.nan_to_num(x).float(), torch.nan_to_num(t).float()) for t in w)
    for t, s in ((g, w[0]), (u, w[1])):
        t[x.isnan().any(1)] = NAN
        t[:, s.isnan().any(1)] = NAN
    dev = [InNan(ctx, t, gap, before) for t in (x, *w)]
    out = [InNan(ctx, torch.zeros((M, N), dtype=TORCH[kind]), gap, before) for _ in range(3)]
    sa3k.gated_linear_fwd(ctx, TYPE[kind], ACTS["none"], *dev, M, N, K, out[0], gate=out[1], up=out[2], ldx=dev[0].ld, ldw=dev[1].ld,
                          ldy=out[0].ld, ldz=out[1].ld)
    same(out[1].get(), g)
    same(out[2].get(), u)
    same(out[0].get(), g * u)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("M,N,K", BACKWARDS)
def test_backward_among_nan(ctx, M, N, K, layout):
    """strange: a NaN in dY (a row of dX, a row of each weight's gradient), one in X (a column of the weights' gradients) and one in gate's
    weight (a column of dX)"""
    gap, before = LAYOUTS[layout]
    kind = "bf16"
    x, w, dy = whole(1, (M, K), 2, kind), [whole(2 + i, (N, K), 2, kind) for i in range(2)], whole(5, (M, N), 1, kind)
    g, u = whole(6, (M, N), 2, kind), whole(7, (M, N), 2, kind)
    strange = layout != "even"
    if strange:
        dy[M // 2, N // 3] = NAN
        x[M - 1, K // 2] = NAN
        w[0][N - 1, K - 1] = NAN
    clean = [torch.nan_to_num(t).float() for t in (dy, x, *w)]
    dg, du = clean[0] * u.float(), clean[0] * g.float()
    dx = (dg.double() @ clean[2].double()) + (du.double() @ clean[3].double())
    dw = [d.double().t() @ clean[1].double() for d in (dg, du)]
    db = [d.double().sum(0) for d in (dg, du)]
    if strange:
        dx[M // 2] = NAN
        dx[:, K - 1] = NAN
        for t in dw:
            t[N // 3] = NAN
            t[:, K // 2] = NAN
        for t in db:
            t[N // 3] = NAN
    ins = [InNan(ctx, t, gap, before) for t in (dy, g, u, x, *w)]
    ox = InNan(ctx, torch.zeros_like(x), gap, before)
    ow = [InNan(ctx, torch.zeros((N, K)), gap, before) for _ in range(2)]
    ob = [up(ctx, torch.full((N,), 7.0)) for _ in range(2)]
    sa3k.gated_linear_bwd(ctx, TYPE[kind], ACTS["none"], *ins, M, N, K, dx=ox, dw_gate=ow[0], dw_up=ow[1], db_gate=ob[0], db_up=ob[1],
                          dw_type=TYPE["f32"], lddy=ins[0].ld, ldz=ins[1].ld, ldx=ins[3].ld, ldw=ins[4].ld, lddx=ox.ld, lddw=ow[0].ld)
    same(ox.get(), dx)
    for o, t in zip(ow, dw):
        same(o.get(), t)
    for o, t in zip(ob, db):
        same(torch.from_numpy(o.numpy()), t)


# 256 wide tiles whose waves store by themselves, whose rows are staged through LDS, and in splits; 128 wide tiles in splits
ENDS = [(396, 9688, 16), (513, 6632, 325), (417, 8435, 316), (156, 8820, 3596), (300, 520, 1000)]


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M,N,K", ENDS)
def test_activations_at_every_end(ctx, M, N, K, act):
    """g = x and its columns again (rows of a unit matrix for gate's weight), u = a bias of 1, -2, 0 or 0.5 (up's weight zeros). act(g): the
    hardware's exp2 and reciprocal are off by 2 U each of a sigmoid, erf by 4 U of 1, so act(g) by 16 U (|act| + |g|), times u, and half
    a step of the result. With g and u stored or not."""
    kind = "bf16"
    x = draw(1, (M, K), 4.0, 0.0, kind)
    x[0, :16] = torch.tensor([0, -0.0, 1e-4, -1e-4, 30, -30, 100, -100, 8, -8, 12, -12, 3, -3, 0.5, -0.5]).to(TORCH[kind])
    at = torch.arange(N) % K
    wg = torch.zeros((N, K), dtype=TORCH[kind])
    wg[torch.arange(N), at] = 1
    c = torch.tensor([1.0, -2.0, 0.0, 0.5]).repeat(N // 4 + 1)[:N]
    X, WG, WU, C = up(ctx, x), up(ctx, wg), up(ctx, torch.zeros_like(wg)), up(ctx, c)
    g = x[:, at]
    want = F64[act](g.double()) * c.double()
    tol = 16 * U32 * (want.abs() + 2 * g.double().abs().clamp(max=30)) + (half_step(kind) + U32) * want.abs() + 2.0 ** -25
    for kept in (False, True):
        out = [ctx.zeros((M, N), np.uint16) for _ in range(3)]
        sa3k.gated_linear_fwd(ctx, TYPE[kind], ACTS[act], X, WG, WU, M, N, K, out[0], up_bias=C, gate=out[1] if kept else None,
                              up=out[2] if kept else None)
        assert bool(((down(out[0], kind).double() - want).abs() <= tol).all())
        if kept:
            assert torch.equal(down(out[1], kind), g + 0)
            assert torch.equal(down(out[2], kind), c.to(TORCH[kind]).expand(M, N))


@pytest.mark.parametrize("M,N,K", [(1, 40, 4616), (5, 333, 6001), (9, 8200, 5120), (16, 1024, 8192), (16, 88, 14344)])
def test_few_rows_on_tiles(ctx, M, N, K):
    """up to 16 rows of weights that the kernel for few rows would read slowly (gated.h: few_blocks)"""
    test_forward_among_nan(ctx, M, N, K, "aligned")
    test_forward_among_nan(ctx, M, N, K, "even")
