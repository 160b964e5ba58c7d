"""Head norms with rotation on the GPU, forward and backward, against the formulas in 64 bits.

Tolerances. U = 2^-24, hs = half a step of the type. The sum of squares: at most 13 additions (8 in a lane, 5 across) and a product each,
so 14 U of itself, 7 U of r; r, gain and their products 5 U, sine and cosine 3 U, the turn 2 U: 17 U of a pair's two values, taken as
24 U of the head's largest, and half a step of the result (f16: or 2^-25, half the step of its smallest values)."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TORCH, TYPE, U32, down, draw, half_step, up

pytestmark = pytest.mark.gpu
SENTINEL = -77.0


class At:
    """an address in a buffer"""

    def __init__(self, buf, off, el):
        self.buf, self.ptr = buf, buf.ptr + off * el


class View:
    """[B][S][H][D] somewhere in a buffer of sentinels"""

    def __init__(self, ctx, t, strides=None, off=0, size=None, kind="bf16"):
        self.kind, self.shape, self.off = kind, tuple(t.shape), off
        B, S, H, D = self.shape
        self.st = strides or (S * H * D, H * D, D)
        size = size or off + sum(s * (n - 1) for s, n in zip(self.st, self.shape[:3])) + D + 8
        host = torch.full((size,), SENTINEL, dtype=TORCH[kind])
        host.as_strided(self.shape, (*self.st, 1), off).copy_(t)
        self.buf = up(ctx, host)
        self.ptr = self.buf.ptr + off * host.element_size()

    def get(self, clean=True):
        now = down(self.buf, self.kind).clone()
        v = now.as_strided(self.shape, (*self.st, 1), self.off)
        got = v.clone()
        if clean:
            v.fill_(SENTINEL)
            assert bool((now == SENTINEL).all()), "written outside the rows"
        return got


def rotated(x, pos, rot, near, base, sign=1.0):
    """x [B][S][H][D] in 64 bits turned by pos [B][S]"""
    y = x.clone()
    if rot == 0:
        return y
    a = pos.double()[:, :, None, None] * base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    cs, sn = torch.cos(a), sign * torch.sin(a)
    p, q = (slice(0, rot, 2), slice(1, rot, 2)) if near else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., p] = x[..., p] * cs - x[..., q] * sn
    y[..., q] = x[..., q] * cs + x[..., p] * sn
    return y


def forward(x, gain, pos, rot, near, base, eps):
    n = x / (x.square().mean(3, keepdim=True) + eps).sqrt() * (1 if gain is None else gain.double())
    return rotated(n, pos, rot, near, base)


def tolerance(kind, y, scale):
    """scale: a head's largest value before the result"""
    return half_step(kind) * y.abs() + 24 * U32 * scale + (2.0 ** -25 if kind == "f16" else 0)


# batch, tokens, heads, kv, dim, rot, near, lengths, positions
CASES = [
    (1, 1, 1, 1, 8, 0, False, None, None), (1, 1, 3, 1, 32, 32, False, None, "far"), (2, 5, 5, 2, 64, 32, False, [5, 0], None),
    (3, 7, 24, 24, 64, 64, True, [7, 3, 1], "far"), (2, 130, 8, 2, 128, 128, False, None, "far"),
    (1, 33, 7, 3, 80, 48, False, [20], "far"), (1, 9, 4, 1, 96, 96, True, None, None), (2, 3, 2, 1, 256, 256, False, [3, 2], "far"),
    (1, 17, 3, 3, 256, 16, True, None, "far"), (2, 2050, 3, 1, 64, 16, False, [2050, 77], None), (1, 8200, 1, 1, 16, 16, True, None, "far"),
    (1, 4, 70, 33, 128, 64, False, None, "end"), (1, 3, 2, 2, 24, 16, False, None, None), (4, 1030, 2, 1, 256, 256, True, None, None),
]


def positions(how, B, S, seed=9):
    if how is None:
        return None
    if how == "end":   # the range of the type's ends
        p = torch.tensor([2 ** 31 - 1, -2 ** 31, -1, 2 ** 30 + 7], dtype=torch.int32)
        return p.repeat(B * S // 4 + 1)[:B * S].view(B, S)
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-100000, 1 << 24, (B, S), generator=g, dtype=torch.int32)


def heads(kind, c, seed, strange=True):
    """q, k, v of a case with NaN and infinities past the lengths"""
    B, S, H, K, D, _, _, lens, _ = c
    out = [draw(seed + i, (B, S, n, D), 1.5, 0.3, kind) for i, n in enumerate((H, K, K))]
    if strange and lens is not None:
        for b, n in enumerate(lens):
            for t in out:
                t[b, n:] = float("nan")
                t[b, n + 1:n + 2] = float("inf")
    return out


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("c", CASES, ids=lambda c: "x".join(map(str, c[:6])))
def test_forward(ctx, kind, c):
    B, S, H, K, D, rot, near, lens, how = c
    base, eps = 1e4, 1e-6
    q, k, v = heads(kind, c, 1)
    gq, gk = draw(5, (D,), 0.3, 1.0), draw(6, (D,), 0.3, 1.0)
    pos = positions(how, B, S)
    p64 = torch.arange(S).expand(B, -1) if pos is None else pos
    inside = torch.ones(B, S, dtype=torch.bool) if lens is None else torch.arange(S)[None] < torch.tensor(lens)[:, None]
    W = (H + 2 * K) * D
    for variant in range(3):   # in a projection's output; odd strides and starts without gains; in place
        odd = variant == 1
        g = (None, None) if odd else (gq, gk)
        if odd:
            src = [View(ctx, t, (S * (n * (D + 3) + 5) + 1, n * (D + 3) + 5, D + 3), off=1 + i, kind=kind)
                   for i, (t, n) in enumerate(((q, H), (k, K), (v, K)))]
            dst = [View(ctx, torch.full_like(t, SENTINEL), (n * S * (D + 1) + 3, D + 1, S * (D + 1)), off=3 - i, kind=kind)
                   for i, (t, n) in enumerate(((q, H), (k, K), (v, K)))]
        else:
            hold = up(ctx, torch.cat([q, k, v], 2))
            el = q.element_size()
            src = [At(hold, o * D, el) for o in (0, H, H + K)]
            for s in src:
                s.st = (S * W, W, D)
            dst = src if variant == 2 else [View(ctx, torch.full_like(t, SENTINEL), kind=kind) for t in (q, k, v)]
        n = sa3k.HeadNorm(ctx, TYPE[kind], B, S, H, K, D, rot, neighbours=near, eps=eps, rope_base=base,
                          **{f"{a}_{b}strides": t.st for b, ts in (("", src), ("out_", dst)) for a, t in zip("qkv", ts)})
        use_v = variant != 2
        n.forward(src[0], src[1], *[None if x is None else up(ctx, x) for x in g], dst[0], dst[1], v=src[2] if use_v else None,
                  v_out=dst[2] if use_v else None, pos=None if pos is None else ctx.upload(pos.numpy()),
                  len=None if lens is None else ctx.upload(np.array(lens, np.int32)))
        if variant == 2:
            all_ = down(hold, kind, (B, S, H + 2 * K, D))
            got = [all_[:, :, :H], all_[:, :, H:H + K], all_[:, :, H + K:]]
        else:
            got = [d.get() for d in dst]
        for i, (x, y) in enumerate(zip((q, k, v), got)):
            rest = x if variant == 2 else torch.full_like(x, SENTINEL)
            assert torch.equal(y[~inside].view(torch.uint8), rest[~inside].view(torch.uint8)), "a row behind a sequence was written"
            if i == 2:
                assert torch.equal(y[inside], x[inside])
                continue
            x = torch.where(inside[:, :, None, None], x, torch.zeros_like(x)).double()
            want = forward(x, g[i], p64, rot, near, base, eps)
            big = forward(x, g[i], p64, 0, near, base, eps).abs().amax(3, keepdim=True)
            ok = (y.double() - want).abs() <= tolerance(kind, want, big)
            assert bool(ok[inside].all()), (variant, i, float((y.double() - want)[inside].abs().max()))


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("c", CASES, ids=lambda c: "x".join(map(str, c[:6])))
def test_backward(ctx, kind, c):
    """dx: w 3 U, h 4 U, r 12 U, the mean of D products 20 U of their absolute mean: 40 U of r (|h| + |x r| mean |h x r|) by the head's
    largest. dgain: a term is off by 16 U of itself and every addition by U of the sum of absolute values; a thread adds at most
    N terms one after the other, then 6 + 4 + 16 and the workgroups' in turn: 16 + N + 50 U of it, N the terms there are."""
    B, S, H, K, D, rot, near, lens, how = c
    base, eps = 1e4, 1e-5
    q, k, _ = heads(kind, c, 1)
    dq, dk, _ = heads(kind, c, 11)
    gains = [draw(5, (D,), 0.3, 1.0), draw(6, (D,), 0.3, 1.0)]
    pos = positions(how, B, S)
    p64 = torch.arange(S).expand(B, -1) if pos is None else pos
    inside = torch.ones(B, S, dtype=torch.bool) if lens is None else torch.arange(S)[None] < torch.tensor(lens)[:, None]
    row = inside[:, :, None, None]
    lay = lambda n, p: (S * (n * (D + p) + 5) + 1, n * (D + p) + 5, D + p)  # noqa: E731
    for variant in range(3):   # dense; odd strides, without gains, sums added to; in place over dy
        odd = variant == 1
        g = [None, None] if odd else gains
        st = lambda n, p: lay(n, p) if odd else None  # noqa: E731
        src = [View(ctx, t, st(n, 3), off=i * odd, kind=kind) for i, (t, n) in enumerate(((q, H), (k, K)))]
        dy = [View(ctx, t, st(n, 1), off=i * odd, kind=kind) for i, (t, n) in enumerate(((dq, H), (dk, K)))]
        dst = dy if variant == 2 else [View(ctx, torch.full_like(t, SENTINEL), st(n, 3), off=1, kind=kind) for t, n in ((q, H), (k, K))]
        old = [draw(20 + i, (D,), 1.0) for i in range(2)]
        dg = [up(ctx, o) for o in old]
        n = sa3k.HeadNorm(ctx, TYPE[kind], B, S, H, K, D, rot, neighbours=near, eps=eps, rope_base=base, q_strides=src[0].st,
                          k_strides=src[1].st, q_out_strides=dy[0].st, k_out_strides=dy[1].st)
        n.backward(src[0], src[1], dy[0], dy[1], *[None if x is None else up(ctx, x) for x in g], dst[0], dst[1], dq_gain=dg[0],
                   dk_gain=dg[1], pos=None if pos is None else ctx.upload(pos.numpy()),
                   len=None if lens is None else ctx.upload(np.array(lens, np.int32)), accumulate=odd)
        for i, (x, d) in enumerate(((q, dq), (k, dk))):
            y = dst[i].get()
            rest = d if variant == 2 else torch.full_like(x, SENTINEL)
            assert torch.equal(y[~inside].view(torch.uint8), rest[~inside].view(torch.uint8)), "a row behind a sequence was written"
            x, d = (torch.where(row, t, torch.zeros_like(t)).double() for t in (x, d))
            gain = torch.ones(D, dtype=torch.float64) if g[i] is None else g[i].double()
            r = 1 / (x.square().mean(3, keepdim=True) + eps).sqrt()
            w = rotated(d, p64, rot, near, base, -1.0)
            h, xh = w * gain, x * r
            want = r * (h - xh * (h * xh).mean(3, keepdim=True))
            big = r * ((d.abs().amax(3, keepdim=True) * 1.5 * gain.abs().max()) + xh.abs() * (h * xh).abs().mean(3, keepdim=True))
            ok = (y.double() - want).abs() <= tolerance(kind, want, big * 40 / 24)
            assert bool(ok[inside].all()), (variant, i, float((y.double() - want)[inside].abs().max()))
            terms = w * xh
            want = terms.sum((0, 1, 2)) + (old[i].double() if odd else 0)
            most = (d.abs().amax() * 1.5 * xh.abs()).sum((0, 1, 2)) * 0 + terms.abs().sum((0, 1, 2)) + old[i].double().abs()
            # (a turned-back w is off by 3 U of its pair's larger value, not of itself)
            pair = (3 * U32 * 1.5 * d.abs().amax(3, keepdim=True) * xh.abs()).sum((0, 1, 2))
            err = (torch.from_numpy(dg[i].numpy()).double() - want).abs()
            assert bool((err <= (66 + int(inside.sum()) * x.shape[2]) * U32 * most + pair + 1e-30).all()), (variant, i, float(err.max()))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("S,K,D", [(1, 8, 128), (3, 2, 64), (2, 5, 80)])
def test_slots(ctx, kind, S, K, D):
    """new tokens into head-major caches: rows out of range and negative ones stay out, everything else in the caches stays as it was"""
    B, H, C = 4, 2 * K, 21
    c = (B, S, H, K, D, D // 16 * 16, False, None, None)
    q, k, v = heads(kind, c, 1)
    g = torch.Generator().manual_seed(3)
    slot = torch.stack([torch.randperm(C, generator=g)[:S] for _ in range(B)]).to(torch.int32)
    slot[1, 0], slot[2, S - 1], slot[3, 0] = -1, C, 2 ** 31 - 1
    pos = slot.clamp(0, C)
    yk, yv = (View(ctx, torch.full((B, C, K, D), SENTINEL, dtype=TORCH[kind]), (K * C * D, D, C * D), kind=kind) for _ in range(2))
    yq = View(ctx, torch.zeros_like(q), kind=kind)
    n = sa3k.HeadNorm(ctx, TYPE[kind], B, S, H, K, D, c[5], cache_tokens=C, k_out_strides=yk.st, v_out_strides=yv.st)
    n.forward(up(ctx, q), up(ctx, k), None, None, yq, yk, v=up(ctx, v), v_out=yv, pos=ctx.upload(pos.numpy()),
              slot=ctx.upload(slot.numpy()))
    wk = torch.full((B, C, K, D), SENTINEL, dtype=torch.float64)
    wv = wk.clone()
    fk = forward(k.double(), None, pos, c[5], False, 1e4, 1e-6)
    for b in range(B):
        for t in range(S):
            if 0 <= slot[b, t] < C:
                wk[b, slot[b, t]], wv[b, slot[b, t]] = fk[b, t], v[b, t].double()
    assert torch.equal(yv.get().double(), wv)
    gk = yk.get().double()
    assert torch.equal(gk == SENTINEL, wk == SENTINEL)
    assert bool(((gk - wk).abs() <= tolerance(kind, wk, 12.0)).all())
    want = forward(q.double(), None, pos, c[5], False, 1e4, 1e-6)
    assert bool(((yq.get().double() - want).abs() <= tolerance(kind, want, want.abs().amax(3, keepdim=True) * 1.5)).all())


def test_cache_rows_past_32_bits(ctx):
    """samples' caches 2^31 elements apart, and a row far into one"""
    B, S, H, K, D, C = 2, 1, 2, 1, 64, 1 << 20
    far = (1 << 31) + 64
    q, k, v = heads("bf16", (B, S, H, K, D, 0, False, None, None), 1)
    big = ctx.empty(far + C * D + 64, np.uint16)
    slot = torch.tensor([[C - 1], [C - 1]], dtype=torch.int32)
    n = sa3k.HeadNorm(ctx, TYPE["bf16"], B, S, H, K, D, 0, cache_tokens=C, k_out_strides=(far, D, D), v_out_strides=(far, D, D))
    n.forward(None, None, None, None, None, None, v=up(ctx, v), v_out=big, slot=ctx.upload(slot.numpy()))
    for b in range(B):
        got = down(big.view(b * far + (C - 1) * D, (D,)), "bf16")
        assert torch.equal(got, v[b, 0, 0])
    big.free()


def test_same_bits_every_time_and_against_differences(ctx):
    """the same bits in every run; dx and dgain against central differences of sum(dy y) in 64 bits"""
    B, S, H, K, D, rot = 2, 40, 3, 1, 64, 32
    c = (B, S, H, K, D, rot, False, None, None)
    q, k, _ = heads("f32", c, 1)
    dq, dk, _ = heads("f32", c, 11)
    gain = draw(5, (D,), 0.3, 1.0)
    n = sa3k.HeadNorm(ctx, TYPE["f32"], B, S, H, K, D, rot)
    pos = torch.arange(S).expand(B, -1)
    runs = []
    for _ in range(3):
        o, p = ctx.zeros(q.shape), ctx.zeros(k.shape)
        a, b = ctx.zeros(D), ctx.zeros(D)
        n.backward(up(ctx, q), up(ctx, k), up(ctx, dq), up(ctx, dk), up(ctx, gain), up(ctx, gain), o, p, dq_gain=a, dk_gain=b)
        runs.append([t.numpy() for t in (o, p, a, b)])
    for r in runs[1:]:
        assert all(np.array_equal(x, y) for x, y in zip(r, runs[0]))
    loss = lambda x, g: float((forward(x, g, pos, rot, False, 1e4, 1e-6) * dq.double()).sum())  # noqa: E731
    x, e = q.double(), 1e-4
    for at in ((0, 0, 0, 0), (1, 39, 2, 63), (0, 17, 1, 20)):
        d = torch.zeros_like(x)
        d[at] = e
        diff = (loss(x + d, gain) - loss(x - d, gain)) / (2 * e)
        assert abs(diff - runs[0][0][at]) <= 1e-5 * (1 + abs(diff))
    for i in (0, 33, 63):
        d = torch.zeros(D, dtype=torch.float64)
        d[i] = e
        diff = (loss(x, gain.double() + d) - loss(x, gain.double() - d)) / (2 * e)
        assert abs(diff - runs[0][2][i]) <= 1e-4 * (1 + abs(diff))


@pytest.mark.parametrize("accumulate", [False, True])
def test_no_tokens(ctx, accumulate):
    n = sa3k.HeadNorm(ctx, TYPE["bf16"], 2, 0, 4, 2, 64, 32)
    old = draw(1, (64,), 1.0)
    dg = [up(ctx, old), up(ctx, old)]
    n.forward(None, None, None, None, None, None)
    n.backward(None, None, None, None, None, None, None, None, dq_gain=dg[0], dk_gain=dg[1], accumulate=accumulate)
    for d in dg:
        assert np.array_equal(d.numpy(), old.numpy() if accumulate else np.zeros(64, np.float32))


def test_refusals(ctx):
    n = sa3k.HeadNorm(ctx, TYPE["bf16"], 1, 2, 4, 2, 64, 40)
    a = ctx.zeros(4096, np.uint16)
    with pytest.raises(sa3k.Sa3kError, match="multiple of 16"):
        n.forward(a, None, None, None, a, None)
    n = sa3k.HeadNorm(ctx, TYPE["bf16"], 1, 2, 4, 2, 64, 32)
    with pytest.raises(sa3k.Sa3kError, match="all null"):
        n.forward(None, None, None, None, None, None)
    with pytest.raises(sa3k.Sa3kError, match="outputs' gradients"):
        n.backward(a, None, None, None, None, None, a, None)
