"""Products on every tile, split and pairing that the plan knows (layer_ops_shapes.py; which shape takes which is checked on the CPU):
exact on whole numbers, whose sums stay below 2^24 so that f32 holds them in any order. bf16 runs plainly laid out, f16 at odd
pitches with everything the epilogue has, dW in f32 and added to."""
import numpy as np
import pytest
import torch

from conftest import sa3k
from layer_ops_shapes import BACKWARD, FORWARD
from layer_ops_util import TORCH, TYPE, Pitched, up

pytestmark = pytest.mark.gpu


def whole(seed, shape, most=3, kind="f32"):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g, dtype=torch.int8).to(TORCH[kind])


def place(ctx, t, pad):
    return Pitched(ctx, t, t.shape[1] + pad, 1 if pad else 0)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", list(FORWARD))
def test_forward(ctx, M, N, K, kind):
    odd = kind == "f16"
    x, w, b, r = whole(1, (M, K), 3, kind), whole(2, (N, K), 3, kind), whole(3, (N,), 9), whole(4, (M, N), 9, kind)
    px, pw, pr, pz, py = (place(ctx, t, p if odd else 0) for t, p in
                          ((x, 3), (w, 1), (r, 5), (torch.zeros_like(r), 1), (torch.zeros_like(r), 2)))
    sa3k.linear_act_fwd(ctx, TYPE[kind], sa3k.ACT_RELU, px, pw, M, N, K, py, bias=up(ctx, b), residual=pr, z=pz, ldx=px.ld,
                        ldw=pw.ld, ldr=pr.ld, ldz=pz.ld, ldy=py.ld)
    z = x.float() @ w.float().t() + b
    assert torch.equal(pz.get(), z.to(TORCH[kind]))
    assert torch.equal(py.get(), (torch.relu(z) + r.float()).to(TORCH[kind]))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("M,N,K", list(BACKWARD))
def test_backward(ctx, M, N, K, kind):
    odd = kind == "f16"
    x, w, dy, z = whole(1, (M, K), 3, kind), whole(2, (N, K), 3, kind), whole(5, (M, N), 2, kind), whole(6, (M, N), 1, kind)
    act = sa3k.ACT_RELU if odd else sa3k.ACT_NONE
    dz = dy.float() * (z > 0 if odd else 1)
    old_w, old_b = whole(7, (N, K), 5, "f32" if odd else kind), whole(8, (N,), 5)
    px, pw, pd, pz, ox, ow = (place(ctx, t, p if odd else 0) for t, p in
                              ((x, 1), (w, 3), (dy, 2), (z, 5), (torch.zeros_like(x), 1), (old_w, 2)))
    ob = up(ctx, old_b)
    sa3k.linear_act_bwd(ctx, TYPE[kind], act, pd, px, pw, M, N, K, z=pz if odd else None, dx=ox, dw=ow, db=ob,
                        dw_type=TYPE["f32"] if odd else None, accumulate=odd, lddy=pd.ld, ldz=pz.ld, ldx=px.ld, ldw=pw.ld,
                        lddx=ox.ld, lddw=ow.ld)
    assert torch.equal(ox.get(), (dz @ w.float()).to(TORCH[kind]))
    want = dz.t() @ x.float()
    assert torch.equal(ow.get(), want + old_w if odd else want.to(TORCH[kind]))
    assert np.array_equal(ob.numpy(), (dz.sum(0) + (old_b if odd else 0)).numpy())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_one_gradient_alone(ctx, kind):
    """dX or dW by itself on 256 x 256 tiles"""
    M, N, K = 1313, 1739, 9179
    x, w, dy = whole(1, (M, K), 3, kind), whole(2, (N, K), 3, kind), whole(5, (M, N), 2, kind)
    dx, dw, px, pw, pd = ctx.zeros((M, K), np.uint16), ctx.zeros((N, K)), up(ctx, x), up(ctx, w), up(ctx, dy)
    sa3k.linear_act_bwd(ctx, TYPE[kind], sa3k.ACT_NONE, pd, None, pw, M, N, K, dx=dx)
    sa3k.linear_act_bwd(ctx, TYPE[kind], sa3k.ACT_NONE, pd, px, None, M, N, K, dw=dw, dw_type=TYPE["f32"])
    got = torch.from_numpy(dx.numpy().view(np.int16)).view(TORCH[kind])
    assert torch.equal(got, (dy.float() @ w.float()).to(TORCH[kind]))
    assert torch.equal(torch.from_numpy(dw.numpy()), dy.float().t() @ x.float())
