"""Global norm and clip of many gradient tensors on the GPU, against the formula in 64 bits.

Tolerances. U = 2^-24, hs = half a step of the type. The average is one rounding in f32 (U of a value, and of the norm), squares and sums
are f64: the norm is off by U, with less than a thousandth of it for the sums. The factor is rounded to f32 (U) from a norm off by U; a
result has the average's and its product's rounding besides: 4 U, then its type's half step (f16: or 2^-25)."""
import numpy as np
import pytest
import torch

from conftest import rng, sa3k
from layer_ops_util import TORCH, TYPE, U32, down, draw, half_step, up

pytestmark = pytest.mark.gpu
SENTINEL = -77.0


class Grads:
    """tensors [(elements, type, output: None in place, "same" or "f32")] in a buffer a type, gaps of sentinels between them"""

    def __init__(self, ctx, specs, gap=3, sd=0.02, seed=1):
        self.ctx, self.specs = ctx, specs
        self.values = [draw(seed + i, (n,), sd, 0.0, t) for i, (n, t, _) in enumerate(specs)]
        self.buf, self.at = [], []
        for (n, t, o), v in zip(specs, self.values):
            host = torch.full((gap + n + 5,), SENTINEL, dtype=TORCH[t])
            host[gap:gap + n] = v
            ot = t if o != "f32" else "f32"
            out = None if o is None else up(ctx, torch.full((1 + n + 5,), SENTINEL, dtype=TORCH[ot]))
            self.buf.append((up(ctx, host), out, ot))
        self.gap = gap
        el = lambda t: 4 if t == "f32" else 2  # noqa: E731
        self.list = sa3k.Tensors(ctx, [(g.ptr + gap * el(t), n, TYPE[t], None if out is None else out.ptr + el(ot), TYPE[ot])
                                       for (n, t, _), (g, out, ot) in zip(specs, self.buf)])

    def results(self):
        """outputs; everything around them, and gradients that are only read, stay as they were"""
        got = []
        for (n, t, o), (g, out, ot), v in zip(self.specs, self.buf, self.values):
            src = down(g, t)
            edge = torch.cat([src[:self.gap], src[self.gap + n:]])
            assert bool((edge == SENTINEL).all())
            if out is None:
                got.append(src[self.gap:self.gap + n])
                continue
            assert torch.equal(src[self.gap:self.gap + n].view(torch.uint8), v.view(torch.uint8))
            dst = down(out, ot)
            assert bool((torch.cat([dst[:1], dst[1 + n:]]) == SENTINEL).all())
            got.append(dst[1:1 + n])
        return got


def expected(values, count, most):
    s = [v.double() / count for v in values]
    norm = float(torch.sqrt(sum((x.square().sum() for x in s), torch.zeros((), dtype=torch.float64))))
    f = most / (norm + 1e-6) if most > 0 and norm > most else 1.0
    return norm, f, [x * f for x in s]


LISTS = [
    [(1, "f32", None)], [(7, "bf16", None), (8193, "f32", "same")], [(16384, "f16", "same"), (16384, "bf16", "f32"), (8192, "f32", None)],
    [(20000, "bf16", "f32"), (1, "f16", "f32"), (3, "f32", "same"), (0, "bf16", None), (65537, "f16", None)],
    [(n, t, o) for n in (1, 2, 15, 255, 1000, 4099) for t in ("f32", "f16", "bf16") for o in (None, "same", "f32")],
    [(300 + i, "f32", None) for i in range(300)], [(3000001, "bf16", "f32"), (2500003, "f32", "same")],
]


@pytest.mark.parametrize("count,most", [(1, 1.0), (4, 0.5), (1, 1e9), (3, 0.0), (5, 1e9), (1, -1.0)])
@pytest.mark.parametrize("specs", LISTS, ids=lambda s: f"{len(s)}x{s[0][0]}")
def test_clip(ctx, specs, count, most):
    g = Grads(ctx, specs, gap=1 + count)
    stat = ctx.zeros(2, np.float64)
    norm, f, want = expected(g.values, count, most)
    assert abs(norm - most) > 1e-3 * norm   # (no case where a rounding decides)
    got_norm = g.list.clip(count, most, stat=stat, want_norm=True)
    st = stat.numpy()
    assert st[0] == got_norm and abs(got_norm - norm) <= 1.01 * U32 * norm + 1e-300
    assert abs(st[1] - f) <= 2.1 * U32 * f and (f < 1 or st[1] == 1.0)
    for (n, t, o), y, w in zip(specs, g.results(), want):
        ot = "f32" if o == "f32" else t
        tol = (4 * U32 + half_step(ot)) * w.abs() + (2.0 ** -25 if ot == "f16" else 2.0 ** -149)
        assert bool(((y.double() - w).abs() <= tol).all()), (n, t, o)
        if count == 1 and f == 1:
            assert torch.equal(y, g.values[specs.index((n, t, o))].to(y.dtype))
    g.list.destroy()


def test_against_the_flat_arena(ctx):
    """tensors that lie end to end in one arena: what sa3k_average_and_clip does there, but for the order of the norm's sum"""
    sizes = [1536 * 32, 1536, 77, 4096 * 5, 1, 130000]
    flat = draw(1, (sum(sizes),), 0.3)
    a, b = up(ctx, flat), up(ctx, flat)
    at = np.cumsum([0] + sizes)
    t = sa3k.Tensors(ctx, [(a.ptr + 4 * int(o), n, TYPE["f32"], None, TYPE["f32"]) for o, n in zip(at, sizes)])
    norm = t.clip(3, 1.0, want_norm=True)
    import ctypes as C
    ref = C.c_double()
    ctx.check(ctx.lib.sa3k_average_and_clip(ctx.h, b.ptr, flat.numel(), 3, 1.0, C.byref(ref)))
    assert abs(norm - ref.value) <= 1e-13 * norm
    x, y = a.numpy(), b.numpy()
    assert bool((np.abs(x - y) <= 2 * U32 * np.abs(y)).all())   # (a factor one step apart at the most)
    t.destroy()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_finite(ctx, bad):
    """as sa3k_average_and_clip: a NaN norm clips nothing, an infinite one by 0"""
    g = Grads(ctx, [(100, "f32", None), (50, "bf16", "f32")])
    v = g.values[0].clone()
    v[3] = bad
    ctx.copy_into(g.buf[0][0].view(g.gap, (100,)), v.numpy())
    norm = g.list.clip(1, 1.0, want_norm=True)
    x, y = g.results()
    if np.isnan(bad):
        assert np.isnan(norm) and torch.equal(y, g.values[1].float()) and bool(torch.isnan(x[3])) and torch.equal(x[4:], v[4:])
    else:
        assert np.isinf(norm) and bool((y == 0).all()) and bool(torch.isnan(x[3])) and bool((x[4:] == 0).all())


def test_large_values_do_not_overflow(ctx):
    """squares past the range of f32"""
    v = torch.full((1000,), 3e38)
    a = up(ctx, v)
    t = sa3k.Tensors(ctx, [(a.ptr, 1000, TYPE["f32"], None, TYPE["f32"])])
    norm = t.clip(1, 1.0, want_norm=True)
    want = float(v[0].double()) * 1000 ** 0.5
    assert abs(norm - want) <= 1e-12 * want
    assert bool((np.abs(a.numpy() - 1000 ** -0.5) <= 4 * U32).all())
    t.destroy()


def test_empty_list_and_repeats(ctx):
    t = sa3k.Tensors(ctx, [])
    stat = ctx.zeros(2, np.float64)
    assert t.clip(1, 1.0, stat=stat, want_norm=True) == 0.0 and list(stat.numpy()) == [0.0, 1.0]
    t.destroy()
    v = draw(1, (5000,), 1.0)
    a, o = up(ctx, v), [ctx.zeros(5000) for _ in range(2)]
    t = sa3k.Tensors(ctx, [(a.ptr, 5000, TYPE["f32"], x.ptr, TYPE["f32"]) for x in o])   # one gradient, twice in the norm
    norm = t.clip(1, 0.0, want_norm=True)
    assert abs(norm - float(v.double().norm()) * 2 ** 0.5) <= 1e-7 * norm
    assert all(np.array_equal(x.numpy(), v.numpy()) for x in o)
    runs = [t.clip(1, 0.0, want_norm=True) for _ in range(3)]
    assert runs == [norm] * 3
    t.destroy()


def test_two_lists_in_turn(ctx):
    """lists share nothing: each one's norm is its own, whatever ran in between without a wait"""
    a, b = Grads(ctx, [(50000, "f32", "same")], seed=1), Grads(ctx, [(70000, "bf16", "f32")], seed=9)
    sa, sb = ctx.zeros(2, np.float64), ctx.zeros(2, np.float64)
    for _ in range(20):
        a.list.clip(1, 1.0, stat=sa)
        b.list.clip(2, 1.0, stat=sb)
    na, fa, _ = expected(a.values, 1, 1.0)
    nb, fb, _ = expected(b.values, 2, 1.0)
    assert abs(sa.numpy()[0] - na) <= 1.01 * U32 * na and abs(sb.numpy()[0] - nb) <= 1.01 * U32 * nb
    a.results()
    b.results()


def test_into_the_optimizer(ctx):
    """clipped into one f32 arena, which sa3k_adamw_clip then takes without a clip of its own: its update with the clip over the same
    gradients in f32, but for a factor one step apart"""
    sizes, hp = [4096, 1536, 99], (1e-2, 0.9, 0.999, 1e-8, 0.01, 1.0)
    n = sum(sizes)
    grads = [draw(5 + i, (k,), 0.5, 0.0, "bf16") for i, k in enumerate(sizes)]
    dev = [up(ctx, g) for g in grads]
    arena = ctx.zeros(n)
    at = np.cumsum([0] + sizes)
    t = sa3k.Tensors(ctx, [(d.ptr, k, TYPE["bf16"], arena.ptr + 4 * int(o), TYPE["f32"]) for d, k, o in zip(dev, sizes, at)])
    p = rng(1).normal(0, 0.1, n).astype(np.float32)
    z = np.zeros(n, np.float32)
    one = [ctx.upload(x) for x in (p, z, z)]
    two = [ctx.upload(x) for x in (p, z, z)]
    t.clip(2, 1.0)
    ctx.adamw_clip(one[0], arena, one[1], one[2], hp[:5] + (0.0,), 1, 1)
    flat = up(ctx, torch.cat([g.float() for g in grads]))
    ctx.adamw_clip(two[0], flat, two[1], two[2], hp, 1, 2)
    for a, b in zip(one, two):
        a, b = a.numpy(), b.numpy()
        assert np.max(np.abs(a - b)) <= 1e-6 * np.max(np.abs(b))
    t.destroy()


def test_refusals(ctx):
    a = ctx.zeros(64)
    with pytest.raises(sa3k.Sa3kError, match="meets"):
        sa3k.Tensors(ctx, [(a.ptr, 8, TYPE["f32"], None, TYPE["f32"]), (a.ptr + 4, 8, TYPE["f32"], None, TYPE["f32"])])
    t = sa3k.Tensors(ctx, [(a.ptr, 8, TYPE["f32"], None, TYPE["f32"])])
    with pytest.raises(sa3k.Sa3kError, match="empty"):
        t.clip(0, 1.0)
    with pytest.raises(sa3k.Sa3kError, match="number"):
        t.clip(1, float("nan"))
    t.destroy()
