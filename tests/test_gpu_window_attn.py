"""Windowed attention on the GPU, forward and backward, against the formulas in 64 bits.

Tolerances. U = 2^-24, hs = half a step of the type. A score is a sum of D products: off by at most D U of the
sum of their absolute values, S in units of the exponent, so a weight by w = 1.5 D U S (with the exponent's own rounding)
and 4 U for the hardware's exp. Rounding the weights for the product with v adds hs of each (f16: or 2^-25, half the step
of its smallest values, of a largest weight of at least 1), the sums 64 U, the result half a step of itself."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TORCH, TYPE, U32, down, draw, half_step, up
from window_attn_ref import CASES, case, forward, widened

pytestmark = pytest.mark.gpu
SENTINEL = 9.0


class Run:
    """a case's inputs in its layout, with garbage past the lengths"""

    def __init__(self, ctx, c, kind, seed=1):
        self.ctx, self.c, self.kind = ctx, c, kind
        B, H, K, D, sq, sk = c["batch"], c["heads"], c["kv"], c["dim"], c["sq"], c["sk"]
        self.q, self.k, self.v = (draw(seed + i, (B, n, h, D), 1.0, 0.0, kind) for i, (n, h) in
                                  enumerate(((sq, H), (sk, K), (sk, K))))
        self.do = draw(seed + 3, (B, sq, H, D), 1.0, 0.0, kind)
        for b in range(B):   # NaN, infinities and large values where nothing is read
            for t, n in ((self.q, c["ql"][b]), (self.do, c["ql"][b]), (self.k, c["kl"][b]), (self.v, c["kl"][b])):
                t[b, n:] = float("nan")
                t[b, n + 1:n + 2] = float("inf")
        es = 2
        if c["layout"] == "packed":
            W = (H + 2 * K) * D
            self.hold = up(ctx, torch.cat([self.q, self.k, self.v], 2))
            self.dhold = up(ctx, torch.full((B, sq, H + 2 * K, D), SENTINEL, dtype=TORCH[kind]))
            st = dict(q_strides=(sq * W, W, D), k_strides=(sq * W, W, D), v_strides=(sq * W, W, D))
            at = lambda hold: [hold.ptr, hold.ptr + H * D * es, hold.ptr + (H + K) * D * es]  # noqa: E731
            self.p, self.dp = at(self.hold), at(self.dhold)
        else:
            cache = c["layout"] == "cache"
            lay = (lambda t: t.transpose(1, 2)) if cache else (lambda t: t)
            self.hold = [up(ctx, self.q), up(ctx, lay(self.k)), up(ctx, lay(self.v))]
            self.dhold = [up(ctx, torch.full_like(lay(t) if i else t, SENTINEL)) for i, t in
                          enumerate((self.q, self.k, self.v))]
            st = dict(k_strides=(sk * K * D, D, sk * D), v_strides=(sk * K * D, D, sk * D)) if cache else {}
            self.p, self.dp = [a.ptr for a in self.hold], [a.ptr for a in self.dhold]
        self.attn = sa3k.WindowAttn(ctx, TYPE[kind], B, H, K, sq, sk, D, left=c["left"], right=c["right"], sinks=c["sinks"],
                                    causal=c["causal"], scale=c["scale"], **st)
        self.o = up(ctx, torch.full((B, sq, H, D), SENTINEL, dtype=TORCH[kind]))
        self.lse = up(ctx, torch.full((B, H, sq), SENTINEL))
        self.ql = ctx.upload(np.array(c["ql"], np.int32)) if c["lens"] else None
        self.kl = ctx.upload(np.array(c["kl"], np.int32)) if c["lens"] else None

    @staticmethod
    def at(ptr):
        class A:
            pass
        a = A()
        a.ptr = ptr
        return a

    def forward(self):
        q, k, v = map(self.at, self.p)
        self.attn.forward(q, k, v, self.o, self.lse, self.ql, self.kl)
        c = self.c
        return (down(self.o, self.kind).double().transpose(1, 2), torch.from_numpy(self.lse.numpy()).double())

    def backward(self):
        q, k, v = map(self.at, self.p)
        dq, dk, dv = map(self.at, self.dp)
        self.attn.backward(q, k, v, self.o, self.lse, up(self.ctx, self.do), dq, dk, dv, self.ql, self.kl)
        c = self.c
        if c["layout"] == "packed":
            t = down(self.dhold, self.kind).double()
            H, K = c["heads"], c["kv"]
            return [x.transpose(1, 2) for x in (t[:, :, :H], t[:, :, H:H + K], t[:, :, H + K:])]
        got = [down(a, self.kind).double() for a in self.dhold]
        return [got[0].transpose(1, 2)] + [g if c["layout"] == "cache" else g.transpose(1, 2) for g in got[1:]]

    def reference(self):
        return forward(self.c, self.q.double(), self.k.double(), self.v.double())


def weight_error(c, r):
    """of a weight, relative"""
    return 1.5 * c["dim"] * U32 * float(r["s_abs"].max() if r["s_abs"].numel() else 0) * 1.4427 + 4 * U32


def check_forward(c, kind, o, lse, r):
    hs, w = half_step(kind), weight_error(c, r)
    rows = r["rows"].expand_as(r["o"])
    tol = r["absv"] * (hs + 2 * w + 64 * U32) + hs * r["o"].abs() + (2.0 ** -25 * r["allv"] if kind == "f16" else 0) + 1e-7
    off = (o - r["o"]).abs() - tol
    assert float(off[rows].max() if rows.any() else -1) <= 0, (c["name"], float(off[rows].max()))
    assert bool((o[~rows] == SENTINEL).all()), "rows past a sample's length were written"
    there, want = rows[..., 0], r["lse"]
    assert torch.equal(torch.isinf(lse) & there, torch.isinf(want) & there) and bool((lse[~there] == SENTINEL).all())
    fin = there & ~torch.isinf(want)
    ltol = 1.4427 * (w + c["sk"] * U32) + 4 * U32 * want.abs() + 2.0 ** -20
    assert bool(((lse - want).abs()[fin] <= ltol[fin]).all()), float((lse - want).abs()[fin].max())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("c", CASES, ids=[c["name"] for c in CASES])
def test_forward(ctx, c, kind):
    run = Run(ctx, c, kind)
    o, lse = run.forward()
    check_forward(c, kind, o, lse, run.reference())


WIDE = [w for w in map(widened, CASES) if w]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("c", WIDE, ids=[c["name"] for c in WIDE])
def test_forward_by_tiles(ctx, c, kind):
    run = Run(ctx, c, kind, seed=21)
    o, lse = run.forward()
    check_forward(c, kind, o, lse, run.reference())


def test_lengths_are_clamped(ctx):
    c = case("clamped", b=2, sq=40, sk=70, ql=[40, 40], kl=[70, 0], layout="split")
    run, want = Run(ctx, c, "bf16"), None
    want = [t.clone() for t in run.forward()]
    run.ql, run.kl = ctx.upload(np.array([41, 1 << 30], np.int32)), ctx.upload(np.array([71, -5], np.int32))
    got = run.forward()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_shared_keys_and_far_offsets(ctx):
    """one cache for the batch (sample stride 0), its heads 2^32 bytes apart"""
    B, H, D, sk = 3, 4, 64, 130
    far = 1 << 31
    q, k, v = draw(1, (B, 1, H, D), kind="bf16"), draw(2, (1, sk, 2, D), kind="bf16"), draw(3, (1, sk, 2, D), kind="bf16")
    buf = ctx.empty((far + 2 * sk * D,), np.uint16)
    bits = lambda t: t.contiguous().view(torch.int16).numpy().view(np.uint16)  # noqa: E731
    for h in range(2):
        ctx.copy_into(buf.view(h * far, (sk, D)), bits(k[0, :, h]))
        ctx.copy_into(buf.view(h * far + sk * D, (sk, D)), bits(v[0, :, h]))
    c = case("shared", b=B, h=H, kv=2, d=D, sq=1, sk=sk, causal=True, layout="split")
    a = sa3k.WindowAttn(ctx, TYPE["bf16"], B, H, 2, 1, sk, D, causal=True, k_strides=(0, D, far), v_strides=(0, D, far))
    o, lse = ctx.zeros((B, 1, H, D), np.uint16), ctx.zeros((B, H, 1))
    a.forward(up(ctx, q), buf, buf.view(sk * D, (1,)), o, lse)
    r = forward(c, q.double(), k.double().expand(B, -1, -1, -1), v.double().expand(B, -1, -1, -1))
    check_forward(c, "bf16", down(o, "bf16").double().transpose(1, 2), torch.from_numpy(lse.numpy()).double(), r)
    buf.free()


def test_large_scores(ctx):
    """scores of hundreds: one key takes a row; nothing overflows"""
    c = case("large", h=2, d=64, sq=150, sk=150, causal=True, left=40, sinks=1, scale=8.0, layout="split")
    run = Run(ctx, c, "bf16")
    o, lse = run.forward()
    assert bool(torch.isfinite(o).all()) and bool(torch.isfinite(lse).all())
    r = run.reference()
    w = weight_error(c, r)
    assert bool(((lse - r["lse"]).abs() <= 1.4427 * (w + 150 * U32) + 8 * U32 * r["lse"].abs() + 1e-5).all())


def test_no_samples_or_queries(ctx):
    for kw in (dict(batch=0, q_tokens=4), dict(batch=2, q_tokens=0)):
        a = sa3k.WindowAttn(ctx, TYPE["bf16"], kw["batch"], 2, 1, kw["q_tokens"], 8, 64)
        a.forward(None, None, None, None) if kw["batch"] == 0 else a.forward(None, ctx.zeros(2048), ctx.zeros(2048), None)


def backward_reference(c, r, do):
    """gradients in 64 bits, and what their terms' absolute values add up to"""
    g = c["heads"] // c["kv"]
    rows = r["rows"]
    do = torch.where(rows, do.double().transpose(1, 2), torch.zeros((), dtype=torch.float64))
    p, q, k, v, sc = r["p"], r["q"], r["k"], r["v"], c["scale"]
    dp = do @ v.transpose(2, 3)
    delta = (do * r["o"]).sum(3, keepdim=True)
    ds = p * (dp - delta)
    fold = lambda t: t.view(t.shape[0], c["kv"], g, *t.shape[2:]).sum(2)  # noqa: E731
    T = lambda t: t.transpose(2, 3)  # noqa: E731
    # |dP| and |delta| as sums of absolute values: what the rounding of o and the f32 sums are relative to
    dpa = do.abs() @ v.abs().transpose(2, 3)
    da = (do * r["o"]).abs().sum(3, keepdim=True)
    return dict(grads=(sc * ds @ k, fold(T(ds) @ q) * sc, fold(T(p) @ do)), ds=ds, dpa=dpa, da=da, do=do, fold=fold, T=T)


def backward_tolerance(c, kind, r, b):
    """A weight is off by wr = w + (lse's own error) of itself; ds by hs of itself for its rounding, wr of p |dP - delta|, and
    p (D U dpa + hs da): f32 sums of D products, o rounded in delta. p is rounded once (f16: or by 2^-25, as ds). Each
    gradient adds 64 U of its terms for its sum and half a step of itself."""
    hs, w = half_step(kind), weight_error(c, r)
    wr = 2 * w + (c["sk"] + 64) * U32
    p, sc, T, fold = r["p"], c["scale"], b["T"], b["fold"]
    tiny = 2.0 ** -25 if kind == "f16" else 0.0
    e = b["ds"].abs() * (hs + wr + 64 * U32) + p * (c["dim"] * U32 * b["dpa"] + (hs + c["dim"] * U32) * b["da"]) + tiny * r["ok"]
    ep = p * (hs + wr + 64 * U32) + tiny * r["ok"]
    q, k, do = r["q"].abs(), r["k"].abs(), b["do"].abs()
    tol = (sc * e @ k, fold(T(e) @ q) * sc, fold(T(ep) @ do))
    return [t + hs * (g.abs() + t) + tiny + 1e-12 for t, g in zip(tol, b["grads"])]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("c", CASES, ids=[c["name"] for c in CASES])
def test_backward(ctx, c, kind):
    run = Run(ctx, c, kind, seed=11)
    run.forward()
    r = run.reference()
    b = backward_reference(c, r, run.do)
    for name, got, want, tol, lens in zip(("dq", "dk", "dv"), run.backward(), b["grads"], backward_tolerance(c, kind, r, b),
                                          (c["ql"], c["kl"], c["kl"])):
        there = torch.stack([torch.arange(got.shape[2]) < n for n in lens])[:, None, :, None].expand_as(got)
        assert bool((got[~there] == SENTINEL).all()), (name, "rows past a sample's length were written")
        off = ((got - want).abs() - tol)[there]
        assert not bool(torch.isnan(off).any()), name
        assert not off.numel() or float(off.max()) <= 0, (name, float(off.max()), float((got - want).abs()[there].max()))


def test_backward_same_bits_every_time(ctx):
    c = case("twice", b=2, h=8, kv=1, d=64, sq=400, left=50, sinks=70, causal=True)
    run = Run(ctx, c, "bf16")
    run.forward()
    seen = {b"".join(t.contiguous().numpy().tobytes() for t in run.backward()) for _ in range(4)}
    assert len(seen) == 1


def test_backward_against_differences(ctx):
    """a few entries of dq, dk and dv against central differences of the loss sum(dO o) in 64 bits"""
    c = case("differences", h=2, kv=1, d=64, sq=40, left=9, sinks=2, causal=True, layout="split")
    run = Run(ctx, c, "f16")
    run.forward()
    grads = run.backward()
    r = run.reference()
    tol = backward_tolerance(c, "f16", r, backward_reference(c, r, run.do))
    x = [run.q.double(), run.k.double(), run.v.double()]

    def loss(y):
        return float((forward(c, *y)["o"].transpose(1, 2) * run.do.double()).sum())

    for t, (b, i, h, d) in ((0, (0, 0, 1, 3)), (0, (0, 33, 0, 60)), (1, (0, 1, 0, 5)), (1, (0, 20, 0, 0)), (2, (0, 0, 0, 9)),
                            (2, (0, 39, 0, 63))):
        y = [[a.clone() for a in x] for _ in range(2)]
        for side, sign in enumerate((1, -1)):
            y[side][t][b, i, h, d] += sign * 1e-4
        num = (loss(y[0]) - loss(y[1])) / 2e-4
        # third-order term: below 1e-8 x the third derivative (some tens here)
        assert abs(float(grads[t][b, h, i, d]) - num) <= float(tol[t][b, h, i, d]) + 1e-6, (t, i)


def test_refusals(ctx):
    z = ctx.zeros(4096, np.uint16)
    for kw, code in ((dict(head_dim=32), 4), (dict(kv_heads=3), 1), (dict(type=0), 4), (dict(scale=0.0), 1), (dict(sinks=-1), 1)):
        args = dict(type=TYPE["bf16"], batch=1, heads=2, kv_heads=1, q_tokens=2, k_tokens=2, head_dim=64)
        args.update(kw)
        with pytest.raises(sa3k.Sa3kError) as e:
            sa3k.WindowAttn(ctx, **args).forward(z, z, z, z)
        assert e.value.code == code, kw
