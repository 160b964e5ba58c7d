"""The gated products' argument checks (csrc/gated.h) and the variants that their GPU tests' shapes take, which are host
arithmetic: compiled with g++ and checked without a GPU."""
import ctypes as C
import heapq
import os
import subprocess

import pytest

from conftest import PKG, ROOT, sa3k
from gated_shapes import BACKWARD, DW_ALONE, DX_ALONE, FORWARD

INVALID, UNSUPPORTED = 1, 4
P = ("X", "Wg", "Wu", "dY", "G", "U", "Y", "Go", "Uo", "dX", "dWg", "dWu", "bg", "bu", "dbg", "dbu")
LD = ("x", "w", "dy", "z", "y", "dx", "dw")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("gated") / "libgated.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "gated_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    lib = C.CDLL(out)
    lib.gated.argtypes = [C.c_int, C.c_int] + [C.POINTER(C.c_int64)] * 3 + [C.c_int] * 3
    lib.plans.argtypes = [C.c_int64] * 3 + [C.POINTER(C.c_int)]
    lib.span.argtypes, lib.span.restype = [C.c_int64, C.c_double] * 2 + [C.c_int64], C.c_double
    return lib


def check(host, bwd=False, type=sa3k.TYPE_BF16, act=2, M=4, N=24, K=16, dw_type=None, accumulate=0, ld=None, **p):
    at = dict(Wg=64, Wu=128, X=192)
    at.update(dict(dY=256, G=320, U=384, dX=448, dWg=512, dWu=8192) if bwd else dict(Y=256))
    at.update(p)
    lds = dict(x=K, w=K, dy=N, z=N, y=N, dx=K, dw=K)
    lds.update(ld or {})
    return host.gated(type, act, (C.c_int64 * 3)(M, N, K), (C.c_int64 * 16)(*[at.get(n, 0) for n in P]),
                      (C.c_int64 * 7)(*[lds[n] for n in LD]), type if dw_type is None else dw_type, accumulate, int(bwd))


def test_accepts(host):
    assert check(host) == 0 and check(host, bwd=True) == 0
    assert check(host, Go=64, Uo=8192, bg=64, bu=68) == 0 and check(host, Go=64) == 0
    assert check(host, X=194, ld=dict(x=17)) == 0
    assert check(host, M=0, X=0, Y=0) == 0 and check(host, bwd=True, M=0, X=0, dY=0, G=0, U=0) == 0
    assert check(host, bwd=True, dX=0, dWg=0, dWu=0, dbg=64) == 0 and check(host, bwd=True, dX=0, Wg=0, Wu=0) == 0
    assert check(host, bwd=True, dWg=0, dWu=0, X=0) == 0
    assert check(host, bwd=True, dw_type=sa3k.TYPE_F32, accumulate=1) == 0
    assert check(host, N=(1 << 21) - 64, K=1, M=1) == 0


def test_gates_outputs_and_ups_lie_apart(host):
    """N 24, K 16: rows that take turns in one tensor are apart, rows that share an element are not"""
    f, b, f32 = dict(Go=1024), dict(bwd=True, dWg=1024), dict(bwd=True, dWg=1024, dw_type=sa3k.TYPE_F32)
    for want, kw in ((INVALID, dict(f, Uo=1024)), (INVALID, dict(f, Uo=1024 + 2 * 95)), (0, dict(f, Uo=1024 + 2 * 96)),
                     (0, dict(f, Uo=1024 + 2 * 24, ld=dict(z=48))), (INVALID, dict(f, Uo=1024 + 2 * 23, ld=dict(z=48))),
                     (0, dict(f, Uo=1024 - 2 * 24, ld=dict(z=48))), (INVALID, dict(f, Uo=1024 - 2 * 25, ld=dict(z=48))),
                     (INVALID, dict(b, dWu=1024)), (0, dict(b, dWu=1024 + 32, ld=dict(dw=32))), (0, dict(b, dWu=1024 + 768)),
                     (INVALID, dict(b, dWu=1024 + 766)), (0, dict(f32, dWu=1024 + 1536)), (INVALID, dict(f32, dWu=1024 + 1532)),
                     (INVALID, dict(b, dbg=64, dbu=64)), (INVALID, dict(b, dbg=64, dbu=64 + 92)), (0, dict(b, dbg=64, dbu=64 + 96))):
        assert check(host, **kw) == want, kw
    assert check(host, M=1, Go=1024, Uo=1024 + 48, ld=dict(z=30)) == 0


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=sa3k.TYPE_F32)), (INVALID, dict(act=5)), (INVALID, dict(act=-1)), (INVALID, dict(M=-1)),
    (INVALID, dict(M=1 << 31)), (INVALID, dict(N=0)), (INVALID, dict(K=0)), (INVALID, dict(N=(1 << 21) - 63)), (INVALID, dict(K=1 << 22)),
    (INVALID, dict(ld=dict(x=15))), (INVALID, dict(ld=dict(w=15))), (INVALID, dict(ld=dict(y=23))), (INVALID, dict(Go=64, ld=dict(z=23))),
    (INVALID, dict(ld=dict(w=1 << 22))), (INVALID, dict(X=193)), (INVALID, dict(Wu=129)), (INVALID, dict(Y=257)), (INVALID, dict(Uo=65)),
    (INVALID, dict(bg=66)), (INVALID, dict(bu=2)), (INVALID, dict(Wg=0)), (INVALID, dict(Wu=0)), (INVALID, dict(X=0)), (INVALID, dict(Y=0)),
    (UNSUPPORTED, dict(M=1 << 30, N=1 << 20)),
])
def test_forward_refuses(host, want, change):
    assert check(host, **change) == want


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=sa3k.TYPE_Q8_0)), (INVALID, dict(dY=0)), (INVALID, dict(G=0)), (INVALID, dict(U=0)), (INVALID, dict(X=0)),
    (INVALID, dict(Wg=0)), (INVALID, dict(Wu=0)), (INVALID, dict(dWg=0)), (INVALID, dict(dWu=0)), (INVALID, dict(accumulate=2)),
    (INVALID, dict(accumulate=1)), (INVALID, dict(dw_type=sa3k.TYPE_F16)), (INVALID, dict(dw_type=sa3k.TYPE_F32, dWg=514)),
    (INVALID, dict(dbg=66)), (INVALID, dict(dbu=2)), (INVALID, dict(ld=dict(dx=15))), (INVALID, dict(ld=dict(dw=15))),
    (INVALID, dict(ld=dict(dy=23))), (INVALID, dict(ld=dict(z=23))), (INVALID, dict(dX=449)),
])
def test_backward_refuses(host, want, change):
    assert check(host, bwd=True, **change) == want


def test_shapes_take_their_variants(host):
    o = (C.c_int * 11)()
    for (M, N, K), want in FORWARD.items():
        host.plans(M, N, K, o)
        assert (o[0], o[1] > 1) == want, (M, N, K, list(o))
    for (M, N, K), want in BACKWARD.items():
        host.plans(M, N, K, o)
        assert (bool(o[2]), o[3], o[4] > 1, o[5], o[6] > 1) == want, (M, N, K, list(o))
    for shapes, at in ((DX_ALONE, 7), (DW_ALONE, 9)):
        for (M, N, K), want in shapes.items():
            host.plans(M, N, K, o)
            assert (o[at], o[at + 1] > 1) == want, (M, N, K, list(o))


@pytest.mark.parametrize("slots", [32, 64])
@pytest.mark.parametrize("nx,tx,nw,tw", [(1, 5.0, 1, 3.0), (32, 5.0, 32, 3.0), (27, 76.0, 36, 55.0), (40, 10.0, 1, 100.0), (5, 100.0, 115, 7.0),
                                         (125, 3.5, 5, 2.25), (63, 1.0, 65, 1.0), (64, 9.0, 65, 8.0), (3, 1000.0, 2500, 1.0), (7, 0.5, 64, 90.0)])
def test_span_is_the_greedy_schedules_end(host, slots, nx, tx, nw, tw):
    """each place takes the next workgroup when it is done"""
    free = [0.0] * slots
    for job in [tx] * nx + [tw] * nw:
        heapq.heapreplace(free, free[0] + job)
    # the additions' order differs: 2^-53 of the sum for each, and two more
    assert host.span(nx, tx, nw, tw, slots) == pytest.approx(max(free), rel=2.0 ** -53 * (nx + nw + 2))
