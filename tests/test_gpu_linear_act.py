"""Products with bias, activation and residual on the GPU, forward and backward, against the formulas in 64 bits.

Most inputs are small whole numbers: their sums stay below 2^24, so f32 holds them exactly whatever the order, and z, and
without an activation (or with relu) y, dX and dW, must be the exact value rounded once. The activations are then checked by
themselves over their range. Tolerances: U = 2^-24, hs = half a step of the type."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TORCH, TYPE, U32, Pitched, down, draw, half_step, up

pytestmark = pytest.mark.gpu

ACTS = {"none": sa3k.ACT_NONE, "relu": sa3k.ACT_RELU, "silu": sa3k.ACT_SILU, "gelu": sa3k.ACT_GELU,
        "gelu_tanh": sa3k.ACT_GELU_TANH}
F64 = {"none": lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
       "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh")}

SHAPES = [(1, 1, 1), (1, 6, 40), (3, 17, 33), (5, 64, 7), (16, 100, 256), (17, 64, 1000), (32, 300, 520), (33, 40, 64),
          (64, 128, 64), (100, 130, 72), (129, 257, 201), (300, 264, 1000), (256, 256, 64), (257, 520, 136), (40, 48, 4096),
          (1030, 1800, 96), (2050, 2052, 80), (4100, 4360, 72), (2176, 192, 640), (65, 1536, 1032)]


def whole(seed, shape, most=3, kind="f32"):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g).to(TORCH[kind])


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_forward_is_exact_on_whole_numbers(ctx, kind, M, N, K):
    for variant in range(3):   # plain and aligned; everything, odd pitches; residual in place
        x, w = whole(1, (M, K), kind=kind), whole(2, (N, K), kind=kind)
        b, r = whole(3, (N,), 9) if variant else None, whole(4, (M, N), 9, kind) if variant else None
        z = x.double() @ w.double().t() + (b.double() if b is not None else 0)
        act = "relu" if variant == 1 else "none"
        want = (F64[act](z) + (r.double() if r is not None else 0)).to(TORCH[kind])
        pad = (0, 0, 0, 0, 0) if variant != 1 else (1, 3, 2, 5, 1)
        off = 1 if variant == 1 else 0
        dx, dw = Pitched(ctx, x, K + pad[0], off), Pitched(ctx, w, K + pad[1], off)
        dr = Pitched(ctx, r, N + pad[2], off) if variant else None
        dz = Pitched(ctx, torch.zeros_like(want), N + pad[3], off) if variant == 1 else None
        dy = dr if variant == 2 else Pitched(ctx, torch.zeros_like(want), N + pad[4], 3 * off)
        sa3k.linear_act_fwd(ctx, TYPE[kind], ACTS[act], dx, dw, M, N, K, dy, bias=up(ctx, b) if variant else None,
                            residual=dr, z=dz, ldx=dx.ld, ldw=dw.ld, ldr=dr.ld if dr else None, ldy=dy.ld,
                            ldz=dz.ld if dz else None)
        assert torch.equal(dy.get(), want), variant
        if dz:
            assert torch.equal(dz.get(), z.to(TORCH[kind]))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_backward_is_exact_on_whole_numbers(ctx, kind, M, N, K):
    for variant in range(3):   # plain and aligned; relu, odd pitches, f32 dW added to; only some gradients
        act = "relu" if variant == 1 else "none"
        x, w, dy = whole(1, (M, K), kind=kind), whole(2, (N, K), kind=kind), whole(5, (M, N), 2, kind)
        z = whole(6, (M, N), 1, kind)
        dz = dy.double() * (z > 0 if variant == 1 else 1)
        pad, off = ((1, 3, 2, 5, 1, 2), 1) if variant == 1 else ((0,) * 6, 0)
        dxx, dw_, ddy, dzz = (Pitched(ctx, t, t.shape[1] + p, off) for t, p in zip((x, w, dy, z), pad))
        f32 = variant == 1
        old_w, old_b = whole(7, (N, K), 5), whole(8, (N,), 5)
        ox = Pitched(ctx, torch.zeros_like(x), K + pad[4], off)
        ow = Pitched(ctx, old_w if f32 else torch.zeros_like(w), K + pad[5], off)
        ob = up(ctx, old_b)
        some = variant == 2
        sa3k.linear_act_bwd(ctx, TYPE[kind], ACTS[act], ddy, None if some else dxx, dw_, M, N, K, z=dzz if act == "relu" else None,
                            dx=ox, dw=None if some else ow, db=None if some else ob, dw_type=TYPE["f32"] if f32 else None,
                            accumulate=f32, lddy=ddy.ld, ldz=dzz.ld, ldx=dxx.ld, ldw=dw_.ld, lddx=ox.ld, lddw=ow.ld)
        assert torch.equal(ox.get(), (dz @ w.double()).to(TORCH[kind])), variant
        if some:
            assert np.array_equal(ob.numpy(), old_b.numpy()) and not bool(ow.get().any())
            continue
        want = dz.t() @ x.double() + (old_w.double() if f32 else 0)
        assert torch.equal(ow.get(), want.to(ow.get().dtype)), variant
        assert np.array_equal(ob.numpy(), (dz.sum(0) + (old_b.double() if f32 else 0)).float().numpy())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [7, 40])
def test_activations(ctx, kind, act, M):
    """z = x exactly (a product with the unit matrix), over the range of the activation. act(z): the hardware's exp2 and
    reciprocal are off by 2 U each of a sigmoid, erf by 4 U of 1, so y by 16 U (|y| + |z|) and half a step; a slope is at most 1.2
    and made of up to four such factors with |z| <= 10 in front: off by 32 U (1 + |z|)."""
    N = 256
    x = draw(1, (M, N), 4.0, 0.0, kind)
    x[0, :16] = torch.tensor([0, -0.0, 1e-4, -1e-4, 30, -30, 100, -100, 8, -8, 12, -12, 3, -3, 0.5, -0.5]).to(TORCH[kind])
    if kind == "bf16":
        x[1, :4] = torch.tensor([1e18, -1e18, 3e30, -3e30]).to(TORCH[kind])
    y, z = ctx.zeros((M, N), np.uint16), ctx.zeros((M, N), np.uint16)
    eye = torch.eye(N).to(TORCH[kind])
    sa3k.linear_act_fwd(ctx, TYPE[kind], ACTS[act], up(ctx, x), up(ctx, eye), M, N, N, y, z=z)
    assert torch.equal(down(z, kind), x + 0)
    want = F64[act](x.double())
    tol = 16 * U32 * (want.abs() + x.double().abs().clamp(max=30)) + half_step(kind) * want.abs() + 2.0 ** -25
    assert bool(((down(y, kind).double() - want).abs() <= tol).all())
    dy = draw(2, (M, N), 1.0, 0.0, kind)
    dx, db = ctx.zeros((M, N), np.uint16), ctx.zeros(N)
    sa3k.linear_act_bwd(ctx, TYPE[kind], ACTS[act], up(ctx, dy), None, up(ctx, eye), M, N, N, z=up(ctx, x), dx=dx, db=db)
    v = x.double().clamp(-1e4, 1e4).requires_grad_()   # (every slope is constant out there)
    F64[act](v).backward(dy.double())
    # dz rounded to the type, then the exact product with 1 rounded again: the same value
    e = 32 * U32 * (1 + x.double().abs().clamp(max=30)) * dy.double().abs()
    assert bool(((down(dx, kind).double() - v.grad).abs() <= e + half_step(kind) * (v.grad.abs() + e) + 2.0 ** -25).all())
    assert bool(((torch.from_numpy(db.numpy()).double() - v.grad.sum(0)).abs() <= e.sum(0) + (M + 16) * U32 * v.grad.abs().sum(0) + 1e-30).all())


def test_backward_against_differences(ctx):
    """dx of a gelu product against central differences of sum(dy y) in 64 bits"""
    M, N, K = 40, 24, 16
    x, w, dy = draw(1, (M, K), 1.0, 0.0, "f16"), draw(2, (N, K), 0.5, 0.0, "f16"), draw(3, (M, N), 1.0, 0.0, "f16")
    z = (x.double() @ w.double().t()).to(torch.float16)
    dx, dw = ctx.zeros((M, K), np.uint16), ctx.zeros((N, K))
    sa3k.linear_act_bwd(ctx, TYPE["f16"], ACTS["gelu"], up(ctx, dy), up(ctx, x), up(ctx, w), M, N, K, z=up(ctx, z), dx=dx, dw=dw,
                        dw_type=TYPE["f32"])
    loss = lambda a, b: float((F64["gelu"](a @ b.t()) * dy.double()).sum())  # noqa: E731
    a, b = x.double(), w.double()
    hs = half_step("f16")
    # z and dz are each rounded once: a slope moves by at most 0.8 hs |z| (gelu'' < 0.8), dz by hs of itself
    zz = a @ b.t()
    e = dy.double().abs() * (0.8 * hs * zz.abs() + 1.2 * hs)
    for i, j in ((0, 0), (7, 5), (39, 15)):
        d = torch.zeros_like(a)
        d[i, j] = 1e-4
        num = (loss(a + d, b) - loss(a - d, b)) / 2e-4
        tol = float(e[i] @ b[:, j].abs())
        assert abs(float(down(dx, "f16")[i, j]) - num) <= tol + hs * (abs(num) + tol) + 1e-6
    for i, j in ((0, 0), (23, 3)):
        d = torch.zeros_like(b)
        d[i, j] = 1e-4
        num = (loss(a, b + d) - loss(a, b - d)) / 2e-4
        assert abs(float(dw.numpy()[i, j]) - num) <= float(e[:, i] @ a[:, j].abs()) + 1e-5


@pytest.mark.parametrize("odd", ["x", "w", "dy"])
def test_one_operand_off_its_alignment(ctx, odd):
    """only one operand has rows that the wide loads cannot take: exact on whole numbers, forward and backward"""
    M, N, K = 140, 72, 104
    x, w, dy = whole(1, (M, K), kind="f16"), whole(2, (N, K), kind="f16"), whole(3, (M, N), 2, "f16")
    px, pw, pd = (Pitched(ctx, t, t.shape[1] + (3 if n == odd else 0), 1 if n == odd else 0)
                  for n, t in (("x", x), ("w", w), ("dy", dy)))
    y, dx, dw = (ctx.zeros(s, np.uint16) for s in ((M, N), (M, K), (N, K)))
    sa3k.linear_act_fwd(ctx, TYPE["f16"], ACTS["none"], px, pw, M, N, K, y, ldx=px.ld, ldw=pw.ld)
    sa3k.linear_act_bwd(ctx, TYPE["f16"], ACTS["none"], pd, px, pw, M, N, K, dx=dx, dw=dw, lddy=pd.ld, ldx=px.ld, ldw=pw.ld)
    X, W, D = x.double(), w.double(), dy.double()
    for got, want in ((y, X @ W.t()), (dx, D @ W), (dw, D.t() @ X)):
        assert torch.equal(down(got, "f16"), want.to(torch.float16))


def test_long_sums(ctx):
    """random values over a long K, split over workgroups: K U of the terms' absolute sum at most"""
    M, N, K = 70, 90, 20000
    x, w = draw(1, (M, K), 1.0, 0.0, "bf16"), draw(2, (N, K), 1.0, 0.0, "bf16")
    y = ctx.zeros((M, N), np.uint16)
    sa3k.linear_act_fwd(ctx, TYPE["bf16"], ACTS["none"], up(ctx, x), up(ctx, w), M, N, K, y)
    want, mag = x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t()
    assert bool(((down(y, "bf16").double() - want).abs() <= half_step("bf16") * want.abs() + K * U32 * mag).all())


def test_garbage_around_the_operands(ctx):
    """NaN behind every row and past the last one never reaches a result"""
    for M, N, K in ((5, 20, 40), (50, 40, 72), (140, 100, 200), (50, 44, 70)):
        x, w, dy = whole(1, (M, K), kind="bf16"), whole(2, (N, K), kind="bf16"), whole(3, (M, N), kind="bf16")
        Pitched.SENTINEL = float("nan")
        try:
            px, pw, pd = Pitched(ctx, x, K + 16, 8), Pitched(ctx, w, K + 8, 16), Pitched(ctx, dy, N + 12 + N % 8, 8)
        finally:
            Pitched.SENTINEL = -77.0
        y, dx, dw, db = (ctx.zeros(s, np.uint16) for s in ((M, N), (M, K), (N, K), (2 * N,)))
        sa3k.linear_act_fwd(ctx, TYPE["bf16"], ACTS["none"], px, pw, M, N, K, y, ldx=px.ld, ldw=pw.ld)
        sa3k.linear_act_bwd(ctx, TYPE["bf16"], ACTS["none"], pd, px, pw, M, N, K, dx=dx, dw=dw, db=db, lddy=pd.ld, ldx=px.ld,
                            ldw=pw.ld)
        X, W, D = x.double(), w.double(), dy.double()
        for got, want in ((y, X @ W.t()), (dx, D @ W), (dw, D.t() @ X)):
            assert torch.equal(down(got, "bf16"), want.to(torch.bfloat16)), (M, N, K)


def test_no_rows(ctx):
    N, K = 70, 48
    w = up(ctx, whole(1, (N, K), kind="bf16"))
    sa3k.linear_act_fwd(ctx, TYPE["bf16"], ACTS["gelu"], None, w, 0, N, K, None)
    dw, db = up(ctx, torch.full((N, K), 3.0)), up(ctx, torch.full((N,), 4.0))
    args = (ctx, TYPE["bf16"], ACTS["gelu"], None, None, w, 0, N, K)
    sa3k.linear_act_bwd(*args, dw=dw, db=db, dw_type=TYPE["f32"], accumulate=True)
    assert (dw.numpy() == 3).all() and (db.numpy() == 4).all()
    sa3k.linear_act_bwd(*args, dw=dw, db=db, dw_type=TYPE["f32"])
    assert not dw.numpy().any() and not db.numpy().any()


def test_same_bits_every_time(ctx):
    M, N, K = 700, 264, 520
    x, w, dy = (up(ctx, draw(i, s, 1.0, 0.0, "bf16")) for i, s in ((1, (M, K)), (2, (N, K)), (3, (M, N))))
    seen = set()
    for _ in range(4):
        out = [ctx.zeros(s, t) for s, t in (((M, K), np.uint16), ((N, K), np.float32), ((N,), np.float32))]
        sa3k.linear_act_bwd(ctx, TYPE["bf16"], ACTS["silu"], dy, x, w, M, N, K, z=dy, dx=out[0], dw=out[1], db=out[2],
                            dw_type=TYPE["f32"])
        seen.add(b"".join(o.numpy().tobytes() for o in out))
    assert len(seen) == 1


def test_rows_past_32_bits(ctx):
    """row pitches of 2^21: the last rows lie past 2^32 bytes"""
    M, N, K, ld = 1040, 24, 64, (1 << 21) + 8
    x, w = whole(1, (M, K), kind="f16"), whole(2, (N, K), kind="f16")
    buf = ctx.empty(((M - 1) * ld + K,), np.uint16)
    for i in range(M):
        ctx.copy_into(buf.view(i * ld, (K,)), x[i].view(torch.int16).numpy().view(np.uint16))
    y, dw = ctx.zeros((M, N), np.uint16), ctx.zeros((N, K))
    sa3k.linear_act_fwd(ctx, TYPE["f16"], ACTS["none"], buf, up(ctx, w), M, N, K, y, ldx=ld)
    want = x.double() @ w.double().t()
    assert torch.equal(down(y, "f16"), want.half())
    dy = whole(3, (M, N), kind="f16")
    sa3k.linear_act_bwd(ctx, TYPE["f16"], ACTS["none"], up(ctx, dy), buf, None, M, N, K, dw=dw, dw_type=TYPE["f32"], ldx=ld)
    assert np.array_equal(dw.numpy(), (dy.double().t() @ x.double()).float().numpy())
    buf.free()


def test_refusals(ctx):
    z = ctx.zeros(4096, np.uint16)
    ok = dict(type=TYPE["bf16"], act=ACTS["gelu"], x=z, w=z, M=4, N=8, K=8, y=z)
    for change, code in ((dict(type=TYPE["f32"]), 4), (dict(act=9), 1), (dict(K=0), 1), (dict(ldx=7), 1), (dict(x=None), 1)):
        with pytest.raises(sa3k.Sa3kError) as e:
            sa3k.linear_act_fwd(ctx, **{**ok, **change})
        assert e.value.code == code, change
    with pytest.raises(sa3k.Sa3kError):
        sa3k.linear_act_bwd(ctx, TYPE["bf16"], ACTS["gelu"], z, z, z, 4, 8, 8, dx=z)   # no z for the activation
