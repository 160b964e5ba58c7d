"""Gated products on the GPU, forward and backward, against the formulas in 64 bits.

Most inputs are small whole numbers: their sums stay below 2^24, so f32 holds them exactly whatever the order, and g, u and,
without an activation (or with relu), Y, dX and dW must be the exact value rounded once. The activations are then checked by
themselves over their range. Tolerances: U = 2^-24, hs = half a step of the type."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from gated_shapes import BACKWARD, DW_ALONE, DX_ALONE, FORWARD
from layer_ops_util import TORCH, TYPE, U32, Pitched, down, draw, half_step, up

pytestmark = pytest.mark.gpu

ACTS = {"none": sa3k.ACT_NONE, "relu": sa3k.ACT_RELU, "silu": sa3k.ACT_SILU, "gelu": sa3k.ACT_GELU,
        "gelu_tanh": sa3k.ACT_GELU_TANH}
F64 = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
       "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}
SHAPES = [(1, 1, 1), (1, 6, 40), (3, 17, 33), (5, 64, 7), (16, 100, 256), (17, 64, 1000), (32, 300, 520), (33, 40, 64),
          (64, 128, 64), (100, 130, 72), (129, 257, 201), (300, 264, 1000), (257, 520, 136), (40, 48, 4096), (1030, 904, 96),
          (65, 768, 1032), (2176, 192, 640)]


def whole(seed, shape, most=3, kind="f32"):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g).to(TORCH[kind])


def same(got, want):
    assert torch.equal(got, want.to(got.dtype)), float((got.double() - want.double()).abs().max())


def forward_case(ctx, kind, M, N, K, variant):
    """variant 0: plain and aligned; 1: everything, odd pitches, relu; 2: the weights as one tensor's halves, only u kept; 3: as 1
    with even pitches"""
    x = whole(1, (M, K), 2, kind)
    w = whole(2, (2 * N, K), 1 if K > 1500 else 2, kind)
    odd, full = variant == 1, variant in (1, 3)
    b = [whole(3 + i, (N,), 9) if full else None for i in range(2)]
    g, u = (x.float() @ t.float().t() + (c if full else 0) for t, c in zip((w[:N], w[N:]), b))
    act = "relu" if full else "none"
    want = F64[act](g) * u
    pad, off = ((1, 3, 2, 5), 1) if odd else ((0,) * 4, 0)
    dx = Pitched(ctx, x, K + pad[0], off)
    if variant == 2:
        both = Pitched(ctx, w, K)

        class Up:
            ptr = both.ptr + N * K * 2
        dw = [both, Up]
    else:
        dw = [Pitched(ctx, t, K + pad[1], off + 2 * i * odd) for i, t in enumerate((w[:N], w[N:]))]
    dy = Pitched(ctx, torch.zeros((M, N), dtype=TORCH[kind]), N + pad[2], off)
    kept = [Pitched(ctx, torch.zeros((M, N), dtype=TORCH[kind]), N + pad[3], off) for _ in range(2)]
    sa3k.gated_linear_fwd(ctx, TYPE[kind], ACTS[act], dx, dw[0], dw[1], M, N, K, dy, gate_bias=up(ctx, b[0]) if full else None,
                          up_bias=up(ctx, b[1]) if full else None, gate=kept[0] if full else None, up=kept[1] if variant else None,
                          ldx=dx.ld, ldw=K + pad[1], ldy=dy.ld, ldz=kept[0].ld)
    same(dy.get(), want)
    same(kept[0].get(), g if full else g * 0)
    same(kept[1].get(), u if variant else u * 0)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_forward_is_exact_on_whole_numbers(ctx, kind, M, N, K):
    for variant in range(3):
        forward_case(ctx, kind, M, N, K, variant)


@pytest.mark.parametrize("shape", list(FORWARD), ids=lambda s: "x".join(map(str, s)))
def test_forward_on_every_tile(ctx, shape):
    for variant in (0, 1, 2, 3):
        forward_case(ctx, "bf16", *shape, variant)
    forward_case(ctx, "f16", *shape, 3)


def backward_case(ctx, kind, M, N, K, variant):
    """variant 0: plain and aligned; 1: relu, odd pitches, f32 dW added to; 2: dX and one bias' gradient only; 3: the products only;
    4: dX only; 5: the weights' gradients only"""
    act = "relu" if variant == 1 else "none"
    x, w, dy = whole(1, (M, K), 2, kind), whole(2, (2 * N, K), 2, kind), whole(5, (M, N), 1, kind)
    g, u = whole(6, (M, N), 2, kind), whole(7, (M, N), 2, kind)
    f, s = (torch.relu(g.float()), (g > 0).float()) if variant == 1 else (g.float(), 1.0)
    dg, du = dy.float() * u.float() * s, dy.float() * f
    odd, some, bare, no_dx = variant == 1, variant in (2, 4), variant in (3, 4, 5), variant == 5
    pad, off = ((1, 3, 2, 5, 1, 2), 1) if odd else ((0,) * 6, 0)
    ddy, dG, dU, dxx = (Pitched(ctx, t, t.shape[1] + p, off) for t, p in ((dy, pad[0]), (g, pad[1]), (u, pad[1]), (x, pad[2])))
    dw = [Pitched(ctx, t, K + pad[3], off) for t in (w[:N], w[N:])]
    old = [whole(8 + i, (N, K), 5) for i in range(2)]
    oldb = [whole(10 + i, (N,), 5) for i in range(2)]
    ox = Pitched(ctx, torch.zeros_like(x), K + pad[4], off)
    ow = [Pitched(ctx, t if odd else torch.zeros((N, K), dtype=TORCH[kind]), K + pad[5], off) for t in old]
    ob = [up(ctx, t) for t in oldb]
    sa3k.gated_linear_bwd(ctx, TYPE[kind], ACTS[act], ddy, dG, dU, None if some else dxx, None if no_dx else dw[0],
                          None if no_dx else dw[1], M, N, K, dx=None if no_dx else ox,
                          dw_gate=None if some else ow[0], dw_up=None if some else ow[1], db_gate=None if some or bare else ob[0],
                          db_up=None if bare else ob[1], dw_type=TYPE["f32"] if odd else None, accumulate=odd, lddy=ddy.ld, ldz=dG.ld, ldx=dxx.ld,
                          ldw=dw[0].ld, lddx=ox.ld, lddw=ow[0].ld)
    if no_dx:
        assert not bool(ox.get().any())
    else:
        same(ox.get(), dg @ w[:N].float() + du @ w[N:].float())
    for i, d in enumerate((dg, du)):
        if bare or (some and i == 0):
            assert np.array_equal(ob[i].numpy(), oldb[i].numpy())
        else:
            assert np.array_equal(ob[i].numpy(), (d.double().sum(0) + (oldb[i].double() if odd else 0)).float().numpy())
        if some:
            assert not bool(ow[i].get().any())
        else:
            same(ow[i].get(), d.t() @ x.float() + (old[i] if odd else 0))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_backward_is_exact_on_whole_numbers(ctx, kind, M, N, K):
    for variant in range(4):
        backward_case(ctx, kind, M, N, K, variant)


def test_backward_of_many_rows(ctx):
    """more rows than the pass over dY, g and u has shares for, with and without column sums"""
    for variant in (0, 3):
        backward_case(ctx, "bf16", 40003, 24, 16, variant)


@pytest.mark.parametrize("shape", list(BACKWARD), ids=lambda s: "x".join(map(str, s)))
def test_backward_on_every_tile(ctx, shape):
    backward_case(ctx, "bf16", *shape, 0)
    backward_case(ctx, "f16", *shape, 1)


@pytest.mark.parametrize("variant,shape", [(v, s) for v, d in ((4, DX_ALONE), (5, DW_ALONE)) for s in d])
def test_backward_products_alone_on_every_tile(ctx, variant, shape):
    backward_case(ctx, "bf16", *shape, variant)
    backward_case(ctx, "f16", *shape, variant)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [7, 40])
def test_activations(ctx, kind, act, M):
    """g = x exactly (a product with the unit matrix), u = 1, -2 or 0 by a weight's diagonal, over the range of the activation. act(g): the
    hardware's exp2 and reciprocal are off by 2 U each of a sigmoid, erf by 4 U of 1, so act(g) by 16 U (|act| + |g|), times u, and half a
    step. A slope is at most 1.2 and made of up to four such factors with |g| <= 10 in front: off by 32 U (1 + |g|)."""
    N = 256
    x = draw(1, (M, N), 4.0, 0.0, kind)
    x[0, :16] = torch.tensor([0, -0.0, 1e-4, -1e-4, 30, -30, 100, -100, 8, -8, 12, -12, 3, -3, 0.5, -0.5]).to(TORCH[kind])
    y, gk = ctx.zeros((M, N), np.uint16), ctx.zeros((M, N), np.uint16)
    eye = torch.eye(N).to(TORCH[kind])
    c = torch.tensor([1.0, -2.0, 0.0, 0.5] * (N // 4))
    zero = torch.zeros((N, N), dtype=TORCH[kind])
    sa3k.gated_linear_fwd(ctx, TYPE[kind], ACTS[act], up(ctx, x), up(ctx, eye), up(ctx, zero), M, N, N, y, up_bias=up(ctx, c), gate=gk)
    assert torch.equal(down(gk, kind), x + 0)
    want = F64[act](x.double()) * c.double()
    tol = 16 * U32 * (want.abs() + 2 * x.double().abs().clamp(max=30)) + (half_step(kind) + U32) * want.abs() + 2.0 ** -25
    assert bool(((down(y, kind).double() - want).abs() <= tol).all())
    # backward: dX = dg (a unit matrix for gate's weight, zeros for up's), db = the column sums of both
    dy, u = draw(2, (M, N), 1.0, 0.0, kind), draw(3, (M, N), 1.0, 0.0, kind)
    dx, dbg, dbu = ctx.zeros((M, N), np.uint16), ctx.zeros(N), ctx.zeros(N)
    sa3k.gated_linear_bwd(ctx, TYPE[kind], ACTS[act], up(ctx, dy), up(ctx, x), up(ctx, u), None, up(ctx, eye), up(ctx, zero), M, N, N,
                          dx=dx, db_gate=dbg, db_up=dbu)
    v, uu = x.double().requires_grad_(), u.double().requires_grad_()
    (F64[act](v) * uu).backward(dy.double())
    big = 1 + x.double().abs().clamp(max=30)
    e = 32 * U32 * big * (dy.double() * u.double()).abs()
    # (dg rounded to the type, then the exact product with 1 rounded again: the same value)
    assert bool(((down(dx, kind).double() - v.grad).abs() <= e + half_step(kind) * (v.grad.abs() + e) + 2.0 ** -25).all())
    sums = lambda g, e: e.sum(0) + (M + 16) * U32 * g.abs().sum(0) + 1e-30  # noqa: E731
    assert bool(((torch.from_numpy(dbg.numpy()).double() - v.grad.sum(0)).abs() <= sums(v.grad, e)).all())
    e = 32 * U32 * big * dy.double().abs()
    assert bool(((torch.from_numpy(dbu.numpy()).double() - uu.grad.sum(0)).abs() <= sums(uu.grad, e)).all())


def test_backward_against_differences(ctx):
    """all gradients of a silu gate against central differences of sum(dy y) in 64 bits. dg and du are rounded to f16 for the products,
    outputs to f16 (dX) or f32: 2^-10 of the sums of absolute values, which for these sizes are below 40"""
    M, N, K = 40, 24, 16
    x, dy = draw(1, (M, K), 1.0, 0.0, "f16"), draw(3, (M, N), 1.0, 0.0, "f16")
    w = [draw(2 + i, (N, K), 0.5, 0.0, "f16") for i in (0, 7)]
    b = [draw(20 + i, (N,), 0.3) for i in range(2)]
    z = [(x.double() @ t.double().t() + c.double()).to(torch.float16) for t, c in zip(w, b)]
    dx, dw, db = ctx.zeros((M, K), np.uint16), [ctx.zeros((N, K)) for _ in w], [ctx.zeros(N) for _ in w]
    sa3k.gated_linear_bwd(ctx, TYPE["f16"], ACTS["silu"], up(ctx, dy), up(ctx, z[0]), up(ctx, z[1]), up(ctx, x), up(ctx, w[0]), up(ctx, w[1]),
                          M, N, K, dx=dx, dw_gate=dw[0], dw_up=dw[1], db_gate=db[0], db_up=db[1], dw_type=TYPE["f32"])
    base = [x.double(), w[0].double(), w[1].double(), b[0].double(), b[1].double()]

    def loss(p):
        return float((F64["silu"](p[0] @ p[1].t() + p[3]) * (p[0] @ p[2].t() + p[4]) * dy.double()).sum())

    got = [down(dx, "f16").double(), *[torch.from_numpy(t.numpy()).double() for t in dw + db]]
    for i, g in enumerate(got):
        for at in ((0,) * base[i].dim(), tuple(n - 1 for n in base[i].shape), tuple(n // 3 for n in base[i].shape)):
            hi, lo = [t.clone() for t in base], [t.clone() for t in base]
            hi[i][at] += 1e-4
            lo[i][at] -= 1e-4
            d = (loss(hi) - loss(lo)) / 2e-4
            assert abs(d - float(g[at])) <= 2.0 ** -9 * 40, (i, at)


@pytest.mark.parametrize("accumulate", [False, True])
def test_no_rows(ctx, accumulate):
    N, K = 24, 40
    old = [whole(i, (N, K)) for i in range(2)]
    dw, db = [up(ctx, t) for t in old], [up(ctx, t[:, 0]) for t in old]
    sa3k.gated_linear_fwd(ctx, TYPE["bf16"], ACTS["silu"], None, dw[0], dw[1], 0, N, K, None)
    sa3k.gated_linear_bwd(ctx, TYPE["bf16"], ACTS["silu"], None, None, None, None, None, None, 0, N, K, dw_gate=dw[0], dw_up=dw[1],
                          db_gate=db[0], db_up=db[1], dw_type=TYPE["f32"], accumulate=accumulate)
    for d, t in zip(dw + db, old + [t[:, 0] for t in old]):
        assert np.array_equal(d.numpy(), t.numpy() if accumulate else 0 * t.numpy())


def test_same_bits_every_time(ctx):
    M, N, K = 700, 1100, 520
    x, w, dy = draw(1, (M, K), 1.0, 0.0, "bf16"), draw(2, (2 * N, K), 0.04, 0.0, "bf16"), draw(3, (M, N), 1.0, 0.0, "bf16")
    X, W, DY = up(ctx, x), up(ctx, w), up(ctx, dy)
    Wu = W.view(N * K, (N, K))
    runs = []
    for _ in range(3):
        y, g, u, dx = (ctx.zeros(s, np.uint16) for s in ((M, N), (M, N), (M, N), (M, K)))
        dw, db = ctx.zeros((2 * N, K)), ctx.zeros(2 * N)
        sa3k.gated_linear_fwd(ctx, TYPE["bf16"], ACTS["gelu"], X, W, Wu, M, N, K, y, gate=g, up=u)
        sa3k.gated_linear_bwd(ctx, TYPE["bf16"], ACTS["gelu"], DY, g, u, X, W, Wu, M, N, K, dx=dx, dw_gate=dw,
                              dw_up=dw.view(N * K, (N, K)), db_gate=db, db_up=db.view(N, (N,)), dw_type=TYPE["f32"])
        runs.append([t.numpy() for t in (y, g, u, dx, dw, db)])
    for r in runs[1:]:
        assert all(np.array_equal(a, b) for a, b in zip(r, runs[0]))


def test_refusals(ctx):
    a = ctx.zeros(64, np.uint16)
    with pytest.raises(sa3k.Sa3kError, match="weights must not be null"):
        sa3k.gated_linear_fwd(ctx, TYPE["bf16"], 2, a, a, None, 2, 4, 4, a)
    with pytest.raises(sa3k.Sa3kError, match="both weights"):
        sa3k.gated_linear_bwd(ctx, TYPE["bf16"], 2, a, a, a, a, a, a, 2, 4, 4, dw_gate=a)
