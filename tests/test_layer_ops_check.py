"""The layer operators' argument checks and the rules that pick a variant (csrc/layer_ops.h), which are host
arithmetic: compiled with g++ and checked without a GPU."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import PKG, ROOT, sa3k

INVALID, UNSUPPORTED = 1, 4


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("layer_ops") / "liblayer_ops.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "layer_ops_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return C.CDLL(out)


NORM_P = ("x", "r", "dy", "y", "sum", "gamma", "beta", "mean", "rstd", "dgamma", "dbeta")


def norm(host, bwd=False, type=sa3k.TYPE_BF16, rows=4, cols=64, eps=1e-5, accumulate=0, ld=None, **p):
    at = dict(x=64, y=64)
    if bwd:
        at.update(dy=64, mean=64, rstd=64)
    at.update(p)
    f = host.norm
    f.argtypes = [C.c_int, C.c_int64, C.c_int64, C.c_float, C.c_int, C.c_int, C.POINTER(C.c_int64), C.POINTER(C.c_int64)]
    lds = dict(x=cols, r=cols, dy=cols, y=cols, sum=cols)
    lds.update(ld or {})
    return f(type, rows, cols, eps, accumulate, int(bwd), (C.c_int64 * 11)(*[at.get(n, 0) for n in NORM_P]),
             (C.c_int64 * 5)(*[lds[n] for n in ("x", "r", "dy", "y", "sum")]))


def test_norm_accepts(host):
    assert norm(host) == 0 and norm(host, bwd=True) == 0
    assert norm(host, r=64, sum=128) == 0
    assert norm(host, x=66, ld=dict(x=65)) == 0            # any element may start a row
    assert norm(host, rows=0, x=0, y=0) == 0               # no rows: nothing is touched
    assert norm(host, bwd=True, rows=0, x=0, y=0, dy=0, mean=0, rstd=0, dgamma=64) == 0
    assert norm(host, cols=16384) == 0 and norm(host, eps=0.0) == 0


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=sa3k.TYPE_Q8_0)), (UNSUPPORTED, dict(cols=16385)), (INVALID, dict(cols=0)),
    (INVALID, dict(cols=-4)), (INVALID, dict(rows=-1)), (INVALID, dict(rows=1 << 31)), (INVALID, dict(eps=-1e-5)),
    (INVALID, dict(eps=float("nan"))), (INVALID, dict(eps=float("inf"))), (INVALID, dict(x=0)), (INVALID, dict(y=0)),
    (INVALID, dict(sum=64)), (INVALID, dict(ld=dict(x=63))), (INVALID, dict(ld=dict(y=1 << 31))), (INVALID, dict(x=65)),
    (INVALID, dict(type=sa3k.TYPE_F32, y=66)), (INVALID, dict(gamma=66)), (INVALID, dict(mean=2)),
    (INVALID, dict(r=64, ld=dict(r=0))),
])
def test_norm_forward_refuses(host, want, change):
    assert norm(host, **change) == want


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=7)), (INVALID, dict(dy=0)), (INVALID, dict(x=0)), (INVALID, dict(y=0)), (INVALID, dict(mean=0)),
    (INVALID, dict(rstd=0)), (INVALID, dict(accumulate=2)), (INVALID, dict(ld=dict(dy=10))), (INVALID, dict(dgamma=65)),
    (INVALID, dict(dbeta=2)), (INVALID, dict(dy=33)),
])
def test_norm_backward_refuses(host, want, change):
    assert norm(host, bwd=True, **change) == want
