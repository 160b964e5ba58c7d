"""A call that fails leaves nothing behind: the next one succeeds."""
import ctypes as C

import numpy as np
import pytest

from conftest import sa3k

pytestmark = pytest.mark.gpu


def test_calls_after_an_allocation_that_failed(ctx):
    rows, cols = 4, 64
    x = ctx.upload(np.arange(rows * cols, dtype=np.float32).reshape(rows, cols))
    y = ctx.zeros((rows, cols))
    out = C.c_void_p()
    assert ctx.lib.sa3k_malloc(ctx.h, 1 << 46, C.byref(out)) == 3 and not out.value   # 64 TiB: more than any card has
    sa3k.layer_norm_fwd(ctx, sa3k.TYPE_F32, x, rows, cols, None, None, 1e-5, y)
    ctx.sync()
    assert abs(float(y.numpy().mean())) < 1e-5
