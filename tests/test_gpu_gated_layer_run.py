"""The operators of a gated layer together, as a layer uses them: training, and single tokens over a cache.

Training: norm -> q/k/v product -> head norms with rotation in place -> windowed attention -> out product onto the residual -> norm ->
gated product -> down product onto the residual; all gradients back through the same operators, then clipped as one list into an f32
arena. Against autograd in 64 bits over the same weights. Every step rounds its outputs once (half a step of f16, 2^-11 relative), 14
outputs lie on the longest way there and back, and no step makes a relative error of its input more than about four times larger
(the norms divide by a deviation near 1, the softmax's scores are of order 1): 14 x 4 x 2^-11 = 0.028 of each tensor's norm.

Single tokens: a prompt in one call, then token by token with k and v into their cache rows. What both give for the same token
may differ by the roundings on the way from q, k and v to its result: q and k off by one step of bf16 at a rounding's border (2^-7
of a value that is one in a hundred of its kind), weights rounded in another order (2^-8) and the result (2^-8): 2^-6 of its norm."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_util import TYPE, down, draw, up
from window_attn_ref import case, visible

pytestmark = pytest.mark.gpu
EPS, QK_EPS, BASE = 1e-5, 1e-6, 1e4


def rel(got, want):
    want = want.detach()
    return float((got.double() - want).norm() / want.norm())


def turned(x, pos, rot):
    """x [B][H][S][D] in 64 bits, halves of the first rot elements paired"""
    a = pos.double()[:, None] * BASE ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    p, q = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([p * a.cos() - q * a.sin(), q * a.cos() + p * a.sin(), x[..., rot:]], -1)


@pytest.mark.parametrize("kv,causal", [(4, False), (2, True)])
def test_gated_layer_forward_and_backward(ctx, kv, causal):
    B, S, H, D, F, R = 2, 150, 4, 64, 328, 32
    E, M, W = H * D, B * S, (H + 2 * kv) * D
    t = TYPE["f16"]
    h = lambda seed, shape, sd=1.0, mean=0.0: draw(seed, shape, sd, mean, "f16")  # noqa: E731
    x, dy = h(1, (M, E)), h(2, (M, E))
    w = {"qkv": h(3, (W, E), E ** -0.5), "out": h(4, (E, E), E ** -0.5), "gate": h(5, (F, E), E ** -0.5), "up": h(6, (F, E), E ** -0.5),
         "down": h(7, (E, F), F ** -0.5)}
    g = {k: draw(30 + i, (n,), 0.1, 1.0) for i, (k, n) in enumerate((("g1", E), ("g2", E), ("gq", D), ("gk", D)))}
    b = {k: draw(40 + i, (F,), 0.1) for i, k in enumerate(("gate_b", "up_b"))}

    # ---- the framework
    dev = {k: up(ctx, v) for d in (w, g, b) for k, v in d.items()}
    f16 = lambda *shape: ctx.zeros(shape, np.uint16)  # noqa: E731
    X, DY = up(ctx, x), up(ctx, dy)
    n1, raw, qkv, a, x1, n2, hid, zg, zu, y = (f16(M, E), f16(M, W), f16(M, W), f16(M, E), f16(M, E), f16(M, E), f16(M, F), f16(M, F),
                                               f16(M, F), f16(M, E))
    st = [ctx.zeros(M) for _ in range(4)]
    lse = ctx.zeros((B, H, S))
    lay = (S * W, W, D)
    rope = sa3k.HeadNorm(ctx, t, B, S, H, kv, D, R, eps=QK_EPS, rope_base=BASE, q_strides=lay, k_strides=lay, v_strides=lay,
                         q_out_strides=lay, k_out_strides=lay, v_out_strides=lay)
    attn = sa3k.WindowAttn(ctx, t, B, H, kv, S, S, D, left=32, right=32, sinks=5, causal=causal, q_strides=lay, k_strides=lay,
                           v_strides=lay)
    parts = lambda r: (r, r.view(E, (1,)), r.view(E + kv * D, (1,)))  # noqa: E731
    none, silu = sa3k.ACT_NONE, sa3k.ACT_SILU
    sa3k.layer_norm_fwd(ctx, t, X, M, E, dev["g1"], None, EPS, n1, mean=st[0], rstd=st[1])
    sa3k.linear_act_fwd(ctx, t, none, n1, dev["qkv"], M, W, E, raw)
    (rq, rk, rv), (q, k, v) = parts(raw), parts(qkv)
    rope.forward(rq, rk, dev["gq"], dev["gk"], q, k, v=rv, v_out=v)
    attn.forward(q, k, v, a, lse)
    sa3k.linear_act_fwd(ctx, t, none, a, dev["out"], M, E, E, x1, residual=X)
    sa3k.layer_norm_fwd(ctx, t, x1, M, E, dev["g2"], None, EPS, n2, mean=st[2], rstd=st[3])
    sa3k.gated_linear_fwd(ctx, t, silu, n2, dev["gate"], dev["up"], M, F, E, hid, gate_bias=dev["gate_b"], up_bias=dev["up_b"], gate=zg,
                          up=zu)
    sa3k.linear_act_fwd(ctx, t, none, hid, dev["down"], M, E, F, y, residual=x1)
    dhid, dn, dx1, da, dqkv, dn1, dx = f16(M, F), f16(M, E), f16(M, E), f16(M, E), f16(M, W), f16(M, E), f16(M, E)
    dw = {k: f16(*v.shape) for k, v in w.items()}
    dv = {k: ctx.zeros(n.shape) for d in (g, b) for k, n in d.items()}
    sa3k.linear_act_bwd(ctx, t, none, DY, hid, dev["down"], M, E, F, dx=dhid, dw=dw["down"])
    sa3k.gated_linear_bwd(ctx, t, silu, dhid, zg, zu, n2, dev["gate"], dev["up"], M, F, E, dx=dn, dw_gate=dw["gate"], dw_up=dw["up"],
                          db_gate=dv["gate_b"], db_up=dv["up_b"])
    sa3k.layer_norm_bwd(ctx, t, dn, x1, M, E, dev["g2"], st[2], st[3], dx1, dsum=DY, dgamma=dv["g2"])
    sa3k.linear_act_bwd(ctx, t, none, dx1, a, dev["out"], M, E, E, dx=da, dw=dw["out"])
    dq, dk, dvv = parts(dqkv)
    attn.backward(q, k, v, a, lse, da, dq, dk, dvv)
    rope.backward(rq, rk, dq, dk, dev["gq"], dev["gk"], dq, dk, dq_gain=dv["gq"], dk_gain=dv["gk"])   # over the attention's
    sa3k.linear_act_bwd(ctx, t, none, dqkv, n1, dev["qkv"], M, W, E, dx=dn1, dw=dw["qkv"])
    sa3k.layer_norm_bwd(ctx, t, dn1, X, M, E, dev["g1"], st[0], st[1], dx, dsum=dx1, dgamma=dv["g1"])
    names = [*w, *g, *b]
    sizes = [{**w, **g, **b}[k].numel() for k in names]
    arena, at = ctx.zeros(sum(sizes)), np.cumsum([0] + sizes)
    grads = sa3k.Tensors(ctx, [({**dw, **dv}[k].ptr, n, t if k in w else TYPE["f32"], arena.ptr + 4 * int(o), TYPE["f32"])
                               for k, n, o in zip(names, sizes, at)])
    norm = grads.clip(B, 1.0, want_norm=True)

    # ---- 64 bits
    leaf = {k: v.double().requires_grad_() for d in (w, g, b) for k, v in d.items()}
    xx = x.double().requires_grad_()
    ln = lambda v, k: torch.nn.functional.layer_norm(v, (E,), leaf[k], None, EPS)  # noqa: E731
    rms = lambda v, k: v / (v.square().mean(-1, keepdim=True) + QK_EPS).sqrt() * leaf[k]  # noqa: E731
    u = (ln(xx, "g1") @ leaf["qkv"].t()).view(B, S, H + 2 * kv, D).transpose(1, 2)
    pos = torch.arange(S)
    qq, kk = turned(rms(u[:, :H], "gq"), pos, R), turned(rms(u[:, H:H + kv], "gk"), pos, R).repeat_interleave(H // kv, 1)
    c = case("layer", b=B, h=H, kv=kv, sq=S, left=32, right=32, sinks=5, causal=causal)
    s = (qq @ kk.transpose(2, 3)) * D ** -0.5
    p = torch.softmax(s.masked_fill(~visible(c, S, S), float("-inf")), 3)
    o = (p @ u[:, H + kv:].repeat_interleave(H // kv, 1)).transpose(1, 2).reshape(M, E)
    xa = xx + o @ leaf["out"].t()
    nn = ln(xa, "g2")
    hh = torch.nn.functional.silu(nn @ leaf["gate"].t() + leaf["gate_b"]) * (nn @ leaf["up"].t() + leaf["up_b"])
    yy = xa + hh @ leaf["down"].t()
    yy.backward(dy.double())

    tol = 0.028
    assert rel(down(y, "f16", (M, E)), yy) <= tol and rel(down(dx, "f16", (M, E)), xx.grad) <= tol
    want = {k: leaf[k].grad / B for k in names}
    total = float(torch.sqrt(sum(v.square().sum() for v in want.values())))
    assert abs(norm - total) <= tol * total
    got = arena.numpy()
    for k, n, o in zip(names, sizes, at):
        assert rel(torch.from_numpy(got[o:o + n]).view(want[k].shape), want[k] / (total + 1e-6)) <= 2 * tol, k   # (the norm's besides)
    assert abs(float(np.linalg.norm(got.astype(np.float64))) - 1.0) <= 1e-5
    grads.destroy()


def test_tokens_one_by_one_over_a_cache(ctx):
    B, H, kv, D, R, C = 3, 4, 2, 64, 64, 96
    P, T = [40, 1, 33], 5   # prompts, and tokens after them
    t, kind = TYPE["bf16"], "bf16"
    S = max(P) + T
    W = (H + 2 * kv) * D
    raw = draw(1, (B, S, H + 2 * kv, D), 1.2, 0.0, kind)
    gq, gk = up(ctx, draw(2, (D,), 0.2, 1.0)), up(ctx, draw(3, (D,), 0.2, 1.0))
    lay, cache = (S * W, W, D), (kv * C * D, D, C * D)
    f16 = lambda *shape: ctx.zeros(shape, np.uint16)  # noqa: E731
    el = 2

    class At:
        def __init__(self, buf, off):
            self.buf, self.ptr = buf, buf.ptr + off * el

    # all tokens at once, causal, into dense tensors
    src = up(ctx, raw)
    q, k, v, o = f16(B, S, H, D), f16(B, S, kv, D), f16(B, S, kv, D), f16(B, S, H, D)
    lens = ctx.upload(np.array([p + T for p in P], np.int32))
    full = sa3k.HeadNorm(ctx, t, B, S, H, kv, D, R, q_strides=lay, k_strides=lay, v_strides=lay)
    full.forward(src, At(src, H * D), gq, gk, q, k, v=At(src, (H + kv) * D), v_out=v, len=lens)
    sa3k.WindowAttn(ctx, t, B, H, kv, S, S, D, causal=True).forward(q, k, v, o, None, lens, lens)
    want = down(o, kind, (B, S, H, D))
    # the prompts into the caches, in one call; then a token a sample at a time
    kc, vc = f16(B, kv, C, D), f16(B, kv, C, D)
    slot = np.tile(np.arange(S, dtype=np.int32), (B, 1))
    for b, p in enumerate(P):
        slot[b, p:] = -1
    pre = sa3k.HeadNorm(ctx, t, B, S, H, kv, D, R, cache_tokens=C, k_strides=lay, v_strides=lay, k_out_strides=cache, v_out_strides=cache)
    pre.forward(None, At(src, H * D), None, gk, None, kc, v=At(src, (H + kv) * D), v_out=vc, slot=ctx.upload(slot))
    step = sa3k.HeadNorm(ctx, t, B, 1, H, kv, D, R, cache_tokens=C, q_strides=(W, W, D), k_strides=(W, W, D), v_strides=(W, W, D),
                         k_out_strides=cache, v_out_strides=cache)
    one = sa3k.WindowAttn(ctx, t, B, H, kv, 1, C, D, causal=True, k_strides=cache, v_strides=cache)
    q1, o1 = f16(B, 1, H, D), f16(B, 1, H, D)
    for i in range(T):
        new = up(ctx, torch.stack([raw[b, p + i] for b, p in enumerate(P)]))
        at = np.array([[p + i] for p in P], np.int32)
        pos = ctx.upload(at)
        step.forward(new, At(new, H * D), gq, gk, q1, kc, v=At(new, (H + kv) * D), v_out=vc, pos=pos, slot=pos)
        one.forward(q1, kc, vc, o1, None, None, ctx.upload(at.ravel() + 1))
        got = down(o1, kind, (B, H, D))
        for b, p in enumerate(P):
            assert rel(got[b], want[b, p + i].double()) <= 2.0 ** -6, (i, b)
