"""The gated layer's operators beside others on one GPU: a DiT's captured steps replay to the eager step's bits after calls of
theirs, on the same context, that grow the layer operators' scratch; and calls of two contexts in turns give the bits that one
context alone gives."""
import numpy as np
import pytest

from conftest import sa3k
from layer_ops_util import TYPE, draw, up
from test_gpu_dit import CFG, HP, db, make_gpu, upload_inputs

pytestmark = pytest.mark.gpu


class Layer:
    """each operator of a gated layer, needing more scratch the more rows there are"""

    def __init__(self, ctx, rows):
        self.ctx, self.rows, self.n, self.k, self.D = ctx, rows, 333, 265, 64
        h = lambda seed, *shape: up(ctx, draw(seed, shape, 0.5, kind="bf16"))  # noqa: E731
        self.x, self.wg, self.wu, self.dy = h(1, rows, self.k), h(2, self.n, self.k), h(3, self.n, self.k), h(4, rows, self.n)
        self.q, self.kk, self.dq, self.dk = (h(5 + i, 1, rows, hh, self.D) for i, hh in enumerate((6, 2, 6, 2)))
        self.gain = up(ctx, draw(9, (self.D,), 0.1, 1.0))

    def run(self):
        """every output; the calls are queued, nothing is waited for"""
        c, t, R, n, k, D = self.ctx, TYPE["bf16"], self.rows, self.n, self.k, self.D
        new = lambda *shape: c.zeros(shape, np.uint16)  # noqa: E731
        y, g, u, dx, dwg, dwu = new(R, n), new(R, n), new(R, n), new(R, k), new(n, k), new(n, k)
        db = [c.zeros(n), c.zeros(n)]
        sa3k.gated_linear_fwd(c, t, sa3k.ACT_SILU, self.x, self.wg, self.wu, R, n, k, y, gate=g, up=u)
        sa3k.gated_linear_bwd(c, t, sa3k.ACT_SILU, self.dy, g, u, self.x, self.wg, self.wu, R, n, k, dx=dx, dw_gate=dwg, dw_up=dwu,
                              db_gate=db[0], db_up=db[1])
        rope = sa3k.HeadNorm(c, t, 1, R, 6, 2, D, D)
        qo, ko, gq, gk, dg = new(1, R, 6, D), new(1, R, 2, D), new(1, R, 6, D), new(1, R, 2, D), [c.zeros(D), c.zeros(D)]
        rope.forward(self.q, self.kk, self.gain, self.gain, qo, ko)
        rope.backward(self.q, self.kk, self.dq, self.dk, self.gain, self.gain, gq, gk, dq_gain=dg[0], dk_gain=dg[1])
        outs = [c.zeros(n * k), c.zeros(n * k), c.zeros(D)]
        t32 = TYPE["f32"]
        self.list = sa3k.Tensors(c, [(dwg.ptr, n * k, t, outs[0].ptr, t32), (dwu.ptr, n * k, t, outs[1].ptr, t32),
                                     (dg[0].ptr, D, t32, outs[2].ptr, t32)])
        self.list.clip(2, 0.5)
        return [y, g, u, dx, dwg, dwu, *db, qo, ko, gq, gk, *dg, *outs]

    def done(self):
        self.list.destroy()


@pytest.fixture
def two():
    """contexts whose workspaces no other test has grown"""
    c = [sa3k.Context(0), sa3k.Context(0)]
    yield c
    for x in c:
        x.close()


def test_captured_dit_steps_after_gated_layers(two):
    ctx = two[0]
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
            layer = Layer(ctx, 1023 * step)   # grows the layer operators' scratch between the replays
            layer.run()
            ctx.sync()
            layer.done()
        assert models[1].graphs() == 1, "the step was not captured"
    finally:
        for d in models:
            d.destroy()


def test_two_contexts_in_turns(two):
    sizes = (700, 1400)
    alone = []
    for c, rows in zip(two, sizes):
        layer = Layer(c, rows)
        alone.append([o.numpy().copy() for o in layer.run()])
        layer.done()
    layers = [Layer(c, rows) for c, rows in zip(two, sizes)]
    for c in two:
        c.sync()
    for _ in range(3):
        outs = [layer.run() for layer in layers]   # both contexts' streams are busy at once
        for o, want in zip(outs, alone):
            for a, b in zip(o, want):
                assert np.array_equal(a.numpy(), b)
        for layer in layers:
            layer.done()


def test_a_list_is_its_contexts_own(two):
    a = two[0].zeros(64)
    t = sa3k.Tensors(two[0], [(a.ptr, 64, TYPE["f32"], None, TYPE["f32"])])
    t.ctx = two[1]
    for call in (lambda: t.clip(1, 1.0), t.destroy):
        with pytest.raises(sa3k.Sa3kError, match="another context"):
            call()
    t.ctx = two[0]
    assert t.clip(1, 1.0, want_norm=True) == 0.0
    t.destroy()
