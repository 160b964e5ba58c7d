"""The layer operators together, as a layer uses them, and beside the attention that the framework had.

One pre-norm layer, forward and backward: norm -> q/k/v product -> windowed attention over the heads in the product's output ->
out product onto the residual -> norm -> up product with gelu -> down product onto the residual. All gradients against
autograd in 64 bits over the same weights. Every step rounds its outputs once (half a step of f16, 2^-11 relative), 12 outputs lie
on the longest way there and back, and no step makes a relative error of its input more than about four times larger
(the norms divide by a deviation near 1, the softmax's scores are of order 1): 12 x 4 x 2^-11 = 0.023 of each tensor's norm."""
import numpy as np
import pytest
import torch

from conftest import bf16_bits, bf16_round, rng, sa3k
from layer_ops_util import TYPE, down, draw, up
from window_attn_ref import case, visible

pytestmark = pytest.mark.gpu
EPS = 1e-5


def rel(got, want):
    want = want.detach()
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("kv,causal", [(4, False), (2, True)])
def test_layer_forward_and_backward(ctx, kv, causal):
    B, S, H, D, F = 2, 150, 4, 64, 512
    E, M, W = H * D, B * S, (H + 2 * kv) * D
    c = case("layer", b=B, h=H, kv=kv, sq=S, left=32, right=32, sinks=5, causal=causal)
    t = TYPE["f16"]
    h = lambda seed, shape, sd=1.0, mean=0.0: draw(seed, shape, sd, mean, "f16")  # noqa: E731
    x, dy = h(1, (M, E)), h(2, (M, E))
    w = {"qkv": h(3, (W, E), E ** -0.5), "out": h(4, (E, E), E ** -0.5), "up": h(5, (F, E), E ** -0.5), "down": h(6, (E, F), F ** -0.5)}
    b = {k: draw(20 + i, (v.shape[0],), 0.1) for i, (k, v) in enumerate(w.items())}
    g = {k: draw(30 + i, (E,), 0.1, 1.0) for i, k in enumerate(("g1", "g2"))}
    o = {k: draw(40 + i, (E,), 0.1) for i, k in enumerate(("o1", "o2"))}

    # ---- the framework
    dev = {k: up(ctx, v) for d in (w, b, g, o) for k, v in ((n + ("_b" if d is b else ""), v) for n, v in d.items())}
    f16 = lambda *shape: ctx.zeros(shape, np.uint16)  # noqa: E731
    X, DY = up(ctx, x), up(ctx, dy)
    n1, qkv, a, x1, n2, hid, z, y = f16(M, E), f16(M, W), f16(M, E), f16(M, E), f16(M, E), f16(M, F), f16(M, F), f16(M, E)
    st = [ctx.zeros(M) for _ in range(4)]
    lse = ctx.zeros((B, H, S))
    attn = sa3k.WindowAttn(ctx, t, B, H, kv, S, S, D, left=32, right=32, sinks=5, causal=causal, q_strides=(S * W, W, D),
                           k_strides=(S * W, W, D), v_strides=(S * W, W, D))
    parts = lambda r: (r, r.view(E, (1,)), r.view(E + kv * D, (1,)))  # noqa: E731
    none, gelu = sa3k.ACT_NONE, sa3k.ACT_GELU
    sa3k.layer_norm_fwd(ctx, t, X, M, E, dev["g1"], dev["o1"], EPS, n1, mean=st[0], rstd=st[1])
    sa3k.linear_act_fwd(ctx, t, none, n1, dev["qkv"], M, W, E, qkv, bias=dev["qkv_b"])
    attn.forward(*parts(qkv), a, lse)
    sa3k.linear_act_fwd(ctx, t, none, a, dev["out"], M, E, E, x1, bias=dev["out_b"], residual=X)
    sa3k.layer_norm_fwd(ctx, t, x1, M, E, dev["g2"], dev["o2"], EPS, n2, mean=st[2], rstd=st[3])
    sa3k.linear_act_fwd(ctx, t, gelu, n2, dev["up"], M, F, E, hid, bias=dev["up_b"], z=z)
    sa3k.linear_act_fwd(ctx, t, none, hid, dev["down"], M, E, F, y, bias=dev["down_b"], residual=x1)
    dhid, dn, dx1, da, dqkv, dn1, dx = f16(M, F), f16(M, E), f16(M, E), f16(M, E), f16(M, W), f16(M, E), f16(M, E)
    dw = {k: ctx.zeros(v.shape) for k, v in w.items()}
    db = {k: ctx.zeros(v.shape) for k, v in b.items()}
    dg = {k: ctx.zeros(E) for k in ("g1", "g2", "o1", "o2")}
    f32 = dict(dw_type=TYPE["f32"], accumulate=True)
    sa3k.linear_act_bwd(ctx, t, none, DY, hid, dev["down"], M, E, F, dx=dhid, dw=dw["down"], db=db["down"], **f32)
    sa3k.linear_act_bwd(ctx, t, gelu, dhid, n2, dev["up"], M, F, E, z=z, dx=dn, dw=dw["up"], db=db["up"], **f32)
    sa3k.layer_norm_bwd(ctx, t, dn, x1, M, E, dev["g2"], st[2], st[3], dx1, dsum=DY, dgamma=dg["g2"], dbeta=dg["o2"],
                        accumulate=True)
    sa3k.linear_act_bwd(ctx, t, none, dx1, a, dev["out"], M, E, E, dx=da, dw=dw["out"], db=db["out"], **f32)
    attn.backward(*parts(qkv), a, lse, da, *parts(dqkv))
    sa3k.linear_act_bwd(ctx, t, none, dqkv, n1, dev["qkv"], M, W, E, dx=dn1, dw=dw["qkv"], db=db["qkv"], **f32)
    sa3k.layer_norm_bwd(ctx, t, dn1, X, M, E, dev["g1"], st[0], st[1], dx, dsum=dx1, dgamma=dg["g1"], dbeta=dg["o1"],
                        accumulate=True)

    # ---- 64 bits
    leaf = {k: v.double().requires_grad_() for d in (w, g, o) for k, v in d.items()}
    bias = {k: v.double().requires_grad_() for k, v in b.items()}
    xx = x.double().requires_grad_()
    ln = lambda v, i: torch.nn.functional.layer_norm(v, (E,), leaf[f"g{i}"], leaf[f"o{i}"], EPS)  # noqa: E731
    lin = lambda v, k: v @ leaf[k].t() + bias[k]  # noqa: E731
    u = lin(ln(xx, 1), "qkv").view(B, S, H + 2 * kv, D).transpose(1, 2)
    q, k, v = u[:, :H], u[:, H:H + kv].repeat_interleave(H // kv, 1), u[:, H + kv:].repeat_interleave(H // kv, 1)
    s = (q @ k.transpose(2, 3)) * D ** -0.5
    p = torch.softmax(s.masked_fill(~visible(c, S, S), float("-inf")), 3)
    r1 = xx + lin((p @ v).transpose(1, 2).reshape(M, E), "out")
    want = r1 + lin(torch.nn.functional.gelu(lin(ln(r1, 2), "up")), "down")
    want.backward(dy.double())

    TOL = 12 * 4 * 2.0 ** -11
    assert rel(down(y, "f16"), want) <= TOL
    assert rel(down(dx, "f16"), xx.grad) <= TOL
    for name in w:
        assert rel(torch.from_numpy(dw[name].numpy()), leaf[name].grad) <= TOL, name
        assert rel(torch.from_numpy(db[name].numpy()), bias[name].grad) <= TOL, name
    for name in dg:
        assert rel(torch.from_numpy(dg[name].numpy()), leaf[name].grad) <= TOL, name


@pytest.mark.parametrize("window", [0, 64])
def test_beside_the_differential_attention(ctx, window):
    """without first tokens, a branch of sa3k_diff_attn_fwd is this attention over head-major tensors: both are within half a
    step of their rounded weights and half a step of the result of the same values (bf16: 4 x 2^-8 of the largest v)"""
    B, H, S = 2, 3, 200
    r = rng(4)
    X = [bf16_round(r.normal(0, 1, (B * H, S, 64)).astype(np.float32)) for _ in range(5)]
    q1, k1, q2, k2, v = (ctx.upload(bf16_bits(x)) for x in X)
    _, o1, o2, l1, l2 = sa3k.attn_fwd(ctx, q1, k1, q2, k2, v, B, H, S, S, window)
    st = (H * S * 64, 64, S * 64)
    side = window // 2 if window else -1
    a = sa3k.WindowAttn(ctx, TYPE["bf16"], B, H, H, S, S, 64, left=side, right=side, q_strides=st, k_strides=st, v_strides=st,
                        o_strides=st)
    o, lse = ctx.zeros((B * H, S, 64), np.uint16), ctx.zeros((B * H, S))
    for q, k, want, wl in ((q1, k1, o1, l1), (q2, k2, o2, l2)):
        a.forward(q, k, v, o, lse)
        d = (down(o, "bf16").double() - down(want, "bf16").double()).abs().max()
        assert float(d) <= 4 * 2.0 ** -8 * np.abs(X[4]).max()
        # one of the two sums its weights as rounded: half a step of the sum, 1.44 x 2^-8 of the base-2 logarithm
        assert np.abs(lse.numpy() - wl.numpy()).max() <= 1.4427 * 2.0 ** -8
