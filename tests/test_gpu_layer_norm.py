"""Layer norm on the GPU, forward and backward, against the formulas in 64 bits.

Tolerances. A row's sums are f32 in at most 32 steps in a lane, 6 over a wave and 8 over waves: n = 46 steps,
each off by at most U = 2^-24 of the partial sum, so mean is off by at most 48 U mean|s| (with the division), a
difference to it by that and U |s - mean|. The sum of squares is off by 48 U of itself and twice the difference's
error; rstd by half of that and 4 U for the root and the division. With A = max|s| rstd (what a row's values are worth
in units of its deviation) xh is off by at most 64 U (A + |xh| (1 + A)) < 64 U (1 + A)(1 + |xh|): a row far
from zero loses that much in any f32 arithmetic. Each output adds half a step of its own type."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TYPE, U32, Pitched, down, draw, half_step, up

pytestmark = pytest.mark.gpu
EPS = 1e-5

SHAPES = [(1, 1), (1, 16), (3, 7), (5, 513), (5, 1536), (33, 1025), (9, 2048), (7, 2049), (4, 4097), (3, 8192),
          (2, 8193), (2, 16384), (2100, 40), (4500, 9)]


def reference(x, r, gamma, beta, kind):
    s = (x.double() + r.double()).to(x.dtype) if r is not None else x
    d = s.double()
    mean = d.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((d - mean).square().mean(1, keepdim=True) + EPS)
    xh = (d - mean) * rstd
    g = gamma.double() if gamma is not None else torch.ones(x.shape[1], dtype=torch.float64)
    b = beta.double() if beta is not None else torch.zeros(x.shape[1], dtype=torch.float64)
    A = d.abs().amax(1, keepdim=True) * rstd
    err = 64 * U32 * (1 + A) * (1 + xh.abs())   # of xh
    return s, mean[:, 0], rstd[:, 0], xh, xh * g + b, err


def close(got, want, tol, what):
    bad = (got.double() - want).abs() - tol
    assert not bool(torch.isnan(got.double()).any()), what
    assert float(bad.max()) <= 0, (what, float(bad.max()), int(bad.argmax()))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(ctx, kind, rows, cols):
    for res in (False, True):
        x, r = draw(rows + cols, (rows, cols), 1.5, 0.3, kind), draw(7, (rows, cols), 0.5, 0.0, kind) if res else None
        gamma, beta = draw(1, (cols,), 0.1, 1.0), draw(2, (cols,), 0.1)
        dx = Pitched(ctx, x, cols + 3, 1)
        dr = Pitched(ctx, r, cols) if res else None
        dy, ds = Pitched(ctx, torch.zeros_like(x), cols + 1, 3), Pitched(ctx, torch.zeros_like(x), cols + 2)
        mean, rstd = ctx.zeros(rows), ctx.zeros(rows)
        sa3k.layer_norm_fwd(ctx, TYPE[kind], dx, rows, cols, up(ctx, gamma), up(ctx, beta), EPS, dy, mean=mean, rstd=rstd,
                            residual=dr, sum=ds if res else None, ldx=cols + 3, ldy=cols + 1, ldsum=cols + 2)
        s, wm, wr, xh, wy, err = reference(x, r, gamma, beta, kind)
        close(dy.get(), wy, half_step(kind) * (wy.abs() + err) + err * gamma.double().abs() + 4 * U32 * wy.abs() + 1e-7, "y")
        if kind == "f16":   # 2^-25: half a step of its smallest values, covered by the 1e-7 above
            assert 2.0 ** -25 < 1e-7
        close(torch.from_numpy(mean.numpy()), wm, 48 * U32 * s.double().abs().mean(1) + 1e-30, "mean")
        A = s.double().abs().amax(1) * wr
        close(torch.from_numpy(rstd.numpy()), wr, 64 * U32 * (1 + A) * wr, "rstd")
        if res:
            # the sum of two values of the type is exact in f32 for these inputs or rounded once more there
            close(ds.get(), x.double() + r.double(), (half_step(kind) + U32) * (x.double() + r.double()).abs(), "sum")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(ctx, kind, rows, cols):
    for ds_given in (False, True):
        x, dy = draw(rows + cols, (rows, cols), 1.5, 0.3, kind), draw(8, (rows, cols), 1.0, 0.0, kind)
        ds = draw(9, (rows, cols), 1.0, 0.0, kind) if ds_given else None
        gamma = draw(1, (cols,), 0.1, 1.0)
        _, mean, rstd, xh, _, err = reference(x, None, gamma, None, kind)
        mean, rstd = mean.float(), rstd.float()
        dx = Pitched(ctx, torch.zeros_like(x), cols + 5, 1)
        dxx, ddy = Pitched(ctx, x, cols + 1), Pitched(ctx, dy, cols + 2, 1)
        dds = Pitched(ctx, ds, cols + 1, 1) if ds_given else None
        dg, db = up(ctx, draw(3, (cols,))), up(ctx, draw(4, (cols,)))
        sa3k.layer_norm_bwd(ctx, TYPE[kind], ddy, dxx, rows, cols, up(ctx, gamma), up(ctx, mean), up(ctx, rstd), dx,
                            dsum=dds, dgamma=dg, dbeta=db, accumulate=ds_given, lddx=cols + 5, ldx=cols + 1,
                            lddy=cols + 2, lddsum=cols + 1)
        D, r = dy.double(), rstd.double()[:, None]
        h = D * gamma.double()
        m0, m1 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
        want = r * (h - m0 - xh * m1) + (ds.double() if ds_given else 0)
        # h and the means are off by 64 U of their absolute sums, xh by err
        habs, hx = h.abs().mean(1, keepdim=True), (h * xh).abs().mean(1, keepdim=True)
        e = r * (64 * U32 * (h.abs() + habs + xh.abs() * hx) + err * hx + xh.abs() * (h.abs() * err).mean(1, keepdim=True))
        close(dx.get(), want, half_step(kind) * want.abs() + 2 * e + 4 * U32 * want.abs() + 1e-7, "dx")
        # a column's sum takes at most rows + 140 steps (a lane's rows, the waves, the workgroups)
        n = (rows + 140) * U32
        wg, wb = (D * xh).sum(0), D.sum(0)
        if ds_given:
            wg, wb = wg + draw(3, (cols,)).double(), wb + draw(4, (cols,)).double()
        close(torch.from_numpy(dg.numpy()), wg, n * ((D * xh).abs().sum(0) + 1) + (D.abs() * err).sum(0) + 4 * U32 * wg.abs(), "dgamma")
        close(torch.from_numpy(db.numpy()), wb, n * (D.abs().sum(0) + 1) + 4 * U32 * wb.abs(), "dbeta")


def test_backward_against_differences(ctx):
    """dx of the formula against central differences of the forward in 64 bits, at a few places"""
    rows, cols = 3, 37
    x, dy, gamma = draw(5, (rows, cols), 1.5, 0.3), draw(6, (rows, cols)), draw(1, (cols,), 0.1, 1.0)

    def loss(v):
        d = v - v.mean(1, keepdim=True)
        return (d / torch.sqrt(d.square().mean(1, keepdim=True) + EPS) * gamma.double() * dy.double()).sum()

    _, mean, rstd, _, _, _ = reference(x, None, gamma, None, "f32")
    dx = ctx.zeros((rows, cols))
    sa3k.layer_norm_bwd(ctx, TYPE["f32"], up(ctx, dy), up(ctx, x), rows, cols, up(ctx, gamma), up(ctx, mean.float()),
                        up(ctx, rstd.float()), dx)
    got = dx.numpy()
    for i, j in [(0, 0), (1, 17), (2, 36)]:
        e = torch.zeros((rows, cols), dtype=torch.float64)
        e[i, j] = 1e-5
        num = float(loss(x.double() + e) - loss(x.double() - e)) / 2e-5
        # the difference is off by its third-order term, under 1e-9 here, and 64-bit noise over the step, under 1e-9
        assert abs(got[i, j] - num) < 1e-8 + 400 * U32 * 4


def test_in_place_and_null_vectors(ctx):
    rows, cols = 13, 200
    x, r = draw(1, (rows, cols), kind="bf16"), draw(2, (rows, cols), kind="bf16")
    ref, y = up(ctx, x), ctx.zeros((rows, cols), np.uint16)
    sa3k.layer_norm_fwd(ctx, TYPE["bf16"], ref, rows, cols, None, None, EPS, y, residual=up(ctx, r))
    a, b = up(ctx, x), up(ctx, r)
    sa3k.layer_norm_fwd(ctx, TYPE["bf16"], a, rows, cols, None, None, EPS, a, residual=b, sum=b)
    assert np.array_equal(a.numpy(), y.numpy())
    s, mean, rstd, xh, want, err = reference(x, r, None, None, "bf16")
    assert torch.equal(down(b, "bf16"), s)
    close(down(y, "bf16"), want, half_step("bf16") * (want.abs() + err) + err + 4 * U32 * want.abs(), "y")
    # the backward with dx over each of its inputs
    dy, ds = draw(3, (rows, cols), kind="bf16"), draw(4, (rows, cols), kind="bf16")
    mean, rstd = up(ctx, mean.float()), up(ctx, rstd.float())
    out = ctx.zeros((rows, cols), np.uint16)
    sa3k.layer_norm_bwd(ctx, TYPE["bf16"], up(ctx, dy), b, rows, cols, None, mean, rstd, out, dsum=up(ctx, ds))
    for which in range(3):
        t = [up(ctx, dy), up(ctx, s), up(ctx, ds)]
        sa3k.layer_norm_bwd(ctx, TYPE["bf16"], t[0], t[1], rows, cols, None, mean, rstd, t[which], dsum=t[2])
        assert np.array_equal(t[which].numpy(), out.numpy()), which


def test_same_bits_every_time(ctx):
    rows, cols = 5000, 130
    x, dy = up(ctx, draw(1, (rows, cols), kind="f16")), up(ctx, draw(2, (rows, cols), kind="f16"))
    mean, rstd, dx = ctx.zeros(rows), up(ctx, torch.ones(rows)), ctx.zeros((rows, cols), np.uint16)
    seen = set()
    for _ in range(4):
        dg, db = ctx.zeros(cols), ctx.zeros(cols)
        sa3k.layer_norm_bwd(ctx, TYPE["f16"], dy, x, rows, cols, None, mean, rstd, dx, dgamma=dg, dbeta=db)
        seen.add(dg.numpy().tobytes() + db.numpy().tobytes() + dx.numpy().tobytes())
    assert len(seen) == 1


def test_one_gradient_only(ctx):
    rows, cols = 70, 33
    x, dy = up(ctx, draw(1, (rows, cols))), up(ctx, draw(2, (rows, cols)))
    mean, rstd, dx = ctx.zeros(rows), up(ctx, torch.ones(rows)), ctx.zeros((rows, cols))
    dg, db, only_g, only_b = (up(ctx, torch.full((cols,), 5.0)) for _ in range(4))
    call = lambda **k: sa3k.layer_norm_bwd(ctx, TYPE["f32"], dy, x, rows, cols, None, mean, rstd, dx, **k)  # noqa: E731
    call(dgamma=dg, dbeta=db)
    call(dgamma=only_g)
    call(dbeta=only_b)
    assert np.array_equal(dg.numpy(), only_g.numpy()) and np.array_equal(db.numpy(), only_b.numpy())


def test_no_rows(ctx):
    cols = 300
    dg, db = up(ctx, torch.full((cols,), 5.0)), up(ctx, torch.full((cols,), 6.0))
    sa3k.layer_norm_fwd(ctx, TYPE["bf16"], None, 0, cols, None, None, EPS, None)
    sa3k.layer_norm_bwd(ctx, TYPE["bf16"], None, None, 0, cols, None, None, None, None, dgamma=dg, dbeta=db, accumulate=True)
    assert (dg.numpy() == 5).all() and (db.numpy() == 6).all()
    sa3k.layer_norm_bwd(ctx, TYPE["bf16"], None, None, 0, cols, None, None, None, None, dgamma=dg, dbeta=db)
    assert not dg.numpy().any() and not db.numpy().any()


def test_offsets_past_32_bits(ctx):
    """rows 2^26 elements apart: the last ones lie past 2^31 elements and 2^32 bytes"""
    rows, cols, ld = 36, 64, 1 << 26
    x = draw(3, (rows, cols), kind="bf16")
    buf = ctx.empty(((rows - 1) * ld + cols,), np.uint16)
    for i in range(rows):
        ctx.copy_into(buf.view(i * ld, (cols,)), x[i].view(torch.int16).numpy().view(np.uint16))
    y, z = ctx.zeros((rows, cols), np.uint16), ctx.zeros((rows, cols), np.uint16)
    sa3k.layer_norm_fwd(ctx, TYPE["bf16"], buf, rows, cols, None, None, EPS, y, ldx=ld)
    sa3k.layer_norm_fwd(ctx, TYPE["bf16"], up(ctx, x), rows, cols, None, None, EPS, z)
    assert np.array_equal(y.numpy(), z.numpy())
    buf.free()


def test_infinities_stay_in_their_row(ctx):
    x = draw(3, (5, 64), kind="f16")
    x[2, 7], x[3, 9] = float("inf"), float("nan")
    y = ctx.zeros((5, 64), np.uint16)
    sa3k.layer_norm_fwd(ctx, TYPE["f16"], up(ctx, x), 5, 64, None, None, EPS, y)
    bad = torch.isnan(down(y, "f16")).any(1)
    assert bad.tolist() == [False, False, True, True, False]


def test_constant_rows(ctx):
    """no deviation: y is the offset (eps keeps rstd finite)"""
    x = torch.full((4, 1536), 3.0)
    y, beta = ctx.zeros((4, 1536)), draw(2, (1536,))
    sa3k.layer_norm_fwd(ctx, TYPE["f32"], up(ctx, x), 4, 1536, None, up(ctx, beta), EPS, y)
    # the mean of equal values is off by at most 48 U of 3, and rstd is 1 / sqrt(1e-5)
    assert np.abs(y.numpy() - beta.numpy()).max() <= 48 * U32 * 3 * 317


def test_refusals(ctx):
    a = ctx.zeros((8, 8))
    ok = dict(type=TYPE["f32"], x=a, rows=8, cols=8, gamma=None, beta=None, eps=EPS, y=a)
    for change, code in ((dict(type=8), 4), (dict(cols=0), 1), (dict(rows=-1), 1), (dict(cols=16385), 4), (dict(ldx=7), 1),
                         (dict(eps=float("nan")), 1), (dict(x=None), 1), (dict(sum=a), 1),
                         (dict(y=a.view(0, (8, 8), np.uint8).view(1, (8, 8))), 1)):
        with pytest.raises(sa3k.Sa3kError) as e:
            sa3k.layer_norm_fwd(ctx, **{**ok, **change})
        assert e.value.code == code, change
