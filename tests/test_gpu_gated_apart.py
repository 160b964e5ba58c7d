"""Gated products on the GPU refuse outputs that meet another tensor, and leave everything as it was."""
import numpy as np
import pytest

from conftest import sa3k
from layer_ops_util import TYPE, draw, up

pytestmark = pytest.mark.gpu
M, N, K = 40, 64, 64


def test_outputs_that_meet(ctx):
    t, a = TYPE["bf16"], sa3k.ACT_SILU
    x, wg, wu, dy, g, u = (up(ctx, draw(1 + i, s, 1.0, kind="bf16")) for i, s in enumerate(((M, K), (N, K), (N, K), (M, N), (M, N), (M, N))))
    y, dw = ctx.zeros((M, N), np.uint16), ctx.zeros((2 * N, K), np.uint16)
    held = (x, wg, wu, dy, g, u, y, dw)
    before = [h.numpy() for h in held]

    def fwd(y, gate=None, up_=None):
        with pytest.raises(sa3k.Sa3kError, match="meets"):
            sa3k.gated_linear_fwd(ctx, t, a, x, wg, wu, M, N, K, y, gate=gate, up=up_)

    def bwd(**out):
        with pytest.raises(sa3k.Sa3kError, match="meets"):
            sa3k.gated_linear_bwd(ctx, t, a, dy, g, u, x, wg, wu, M, N, K, **out)

    fwd(g, gate=g)
    fwd(u, up_=u)
    fwd(x)
    fwd(y, gate=wg)
    fwd(y, gate=x)
    bwd(dx=x)
    bwd(dx=dy)
    bwd(dx=y, dw_gate=dw, dw_up=wu)
    bwd(dx=dw, dw_gate=dw, dw_up=dw.view(N * K, (N, K)))
    for h, b in zip(held, before):
        assert np.array_equal(h.numpy(), b)
    # rows in turns of one buffer are apart: g, u and Y side by side
    row = ctx.zeros((M, 3 * N), np.uint16)
    sa3k.gated_linear_fwd(ctx, t, a, x, wg, wu, M, N, K, row.view(2 * N, (1,)), gate=row, up=row.view(N, (1,)), ldy=3 * N, ldz=3 * N)
    own = [ctx.zeros((M, N), np.uint16) for _ in range(3)]
    sa3k.gated_linear_fwd(ctx, t, a, x, wg, wu, M, N, K, own[2], gate=own[0], up=own[1])
    got = row.numpy()
    for i, o in enumerate(own):
        assert np.array_equal(got[:, i * N:(i + 1) * N], o.numpy())
