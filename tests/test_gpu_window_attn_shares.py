"""The attention's backward where only the key tiles with first tokens are shared out over workgroups: gradients against 64 bits,
the same bits every time, nothing written past a sample's lengths. Tolerances as in test_gpu_window_attn.py."""
import pytest
import torch

from layer_ops_shapes import FIRST_SHARED
from test_gpu_window_attn import SENTINEL, Run, backward_reference, backward_tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("c", FIRST_SHARED, ids=[c["name"] for c in FIRST_SHARED])
def test_backward(ctx, c, kind):
    run = Run(ctx, c, kind, seed=31)
    run.forward()
    r = run.reference()
    b = backward_reference(c, r, run.do)
    got = run.backward()
    for name, g, want, tol, lens in zip(("dq", "dk", "dv"), got, b["grads"], backward_tolerance(c, kind, r, b),
                                        (c["ql"], c["kl"], c["kl"])):
        there = torch.stack([torch.arange(g.shape[2]) < n for n in lens])[:, None, :, None].expand_as(g)
        assert bool((g[~there] == SENTINEL).all()), name
        off = ((g - want).abs() - tol)[there]
        assert not bool(torch.isnan(off).any()) and float(off.max()) <= 0, (name, float(off.max()))
    for again in range(2):
        assert all(torch.equal(a, b) for a, b in zip(got, run.backward())), again
