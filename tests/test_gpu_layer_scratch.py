"""The layer operators' scratch is their own: a DiT's captured steps replay to the eager step's bits after calls of the layer
operators, on the same context, that need far more scratch than the DiT's products do."""
import numpy as np
import pytest

from conftest import sa3k
from layer_ops_util import TYPE, draw, up
from test_gpu_dit import CFG, HP, db, make_gpu, upload_inputs

pytestmark = pytest.mark.gpu


def run_layer_ops(ctx, rows):
    """each operator that takes scratch, needing more of it the more rows there are"""
    t, n, D = TYPE["bf16"], 520, 64
    h = lambda seed, *shape: up(ctx, draw(seed, shape, 0.5, kind="bf16"))  # noqa: E731
    new = lambda *shape: ctx.zeros(shape, np.uint16)  # noqa: E731
    x, dy, w = h(1, rows, n), h(2, rows, n), h(3, n, n)
    mean, rstd, dgamma, dbeta, bias = ctx.zeros(rows), ctx.zeros(rows), ctx.zeros(n), ctx.zeros(n), ctx.zeros(n)
    y, z, dx, dw = new(rows, n), new(rows, n), new(rows, n), new(n, n)
    sa3k.layer_norm_fwd(ctx, t, x, rows, n, None, None, 1e-5, y, mean=mean, rstd=rstd)
    sa3k.layer_norm_bwd(ctx, t, dy, x, rows, n, None, mean, rstd, dx, dgamma=dgamma, dbeta=dbeta)
    sa3k.linear_act_fwd(ctx, t, sa3k.ACT_GELU, x, w, rows, n, n, y, z=z)
    sa3k.linear_act_bwd(ctx, t, sa3k.ACT_GELU, dy, x, w, rows, n, n, z=z, dx=dx, dw=dw, db=bias)
    H = 8
    q, k, v, dO = (h(4 + i, rows, H, D) for i in range(4))
    a = sa3k.WindowAttn(ctx, t, 1, H, H, rows, rows, D, left=64, right=64, sinks=32)
    o, dq, dk, dv, lse = new(rows, H, D), new(rows, H, D), new(rows, H, D), new(rows, H, D), ctx.zeros((1, H, rows))
    a.forward(q, k, v, o, lse)
    a.backward(q, k, v, o, lse, dO, dq, dk, dv)
    few = sa3k.WindowAttn(ctx, t, 1, H, H, 1, rows, D)
    few.forward(q, k, v, o, lse)
    ctx.sync()


@pytest.fixture
def fresh():
    """a context whose workspaces no other test has grown"""
    c = sa3k.Context(0)
    yield c
    c.close()


def test_captured_dit_steps_after_layer_operators(fresh):
    ctx = fresh
    tensors, adapters, inputs = db.random_dit(45, CFG, "full")
    upl, _ = upload_inputs(ctx, inputs)
    models = []
    try:
        for graphs in (False, True):
            d = make_gpu(ctx, CFG, tensors, adapters, "full", sa3k.TYPE_F16)
            d.set_graphs(graphs)
            models.append(d)
        for step in range(1, 5):
            got = []
            for d in models:
                loss = [d.accumulate(upl["x_t"], upl["target"], upl["t"], upl["cross"], upl["glob"]) for _ in range(2)]
                g = d.arena(1).numpy()
                d.apply_adamw(HP, step)
                got.append((*loss, g, d.arena(0).numpy()))
            for a, b in zip(*got):
                assert np.array_equal(a, b), f"a replayed step differs from the eager one at step {step}"
            run_layer_ops(ctx, 1024 * step)   # grows the layer operators' scratch between the replays
        assert models[1].graphs() == 1, "the step was not captured"
    finally:
        for d in models:
            d.destroy()
