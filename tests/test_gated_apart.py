"""Gated products refuse outputs that meet each other or an input (csrc/gated.h): host arithmetic, compiled with g++ and checked
without a GPU."""
import ctypes as C
import os
import random
import subprocess

import pytest

from conftest import PKG, ROOT, sa3k

P = ("X", "Wg", "Wu", "dY", "G", "U", "Y", "Go", "Uo", "dX", "dWg", "dWu", "bg", "bu", "dbg", "dbu")
LD = ("x", "w", "dy", "z", "y", "dx", "dw")
M, N, K = 4, 24, 16
# each tensor in a place of its own
FWD = dict(X=1 << 12, Wg=2 << 12, Wu=3 << 12, Y=4 << 12, Go=5 << 12, Uo=6 << 12, bg=7 << 12, bu=8 << 12)
BWD = dict(X=1 << 12, Wg=2 << 12, Wu=3 << 12, dY=4 << 12, G=5 << 12, U=6 << 12, dX=7 << 12, dWg=8 << 12, dWu=9 << 12, dbg=10 << 12,
           dbu=11 << 12)


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("gated_apart") / "libgated_apart.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "gated_apart_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return C.CDLL(out)


def refused(host, at, m=M, dw_type=sa3k.TYPE_BF16, **ld):
    lds = dict(x=K, w=K, dy=N, z=N, y=N, dx=K, dw=K)
    lds.update(ld)
    r = host.apart(sa3k.TYPE_BF16, (C.c_int64 * 3)(m, N, K), (C.c_int64 * 16)(*[at.get(n, 0) for n in P]),
                   (C.c_int64 * 7)(*[lds[n] for n in LD]), dw_type, int("dY" in at))
    assert r in (0, 1), "refused by the other checks"
    return bool(r)


def test_tensors_of_their_own(host):
    assert not refused(host, FWD) and not refused(host, BWD)
    assert not refused(host, {k: FWD[k] for k in ("X", "Wg", "Wu", "Y")})
    assert not refused(host, dict(FWD, Wu=FWD["Wg"], bu=FWD["bg"]))   # inputs may be the same
    assert not refused(host, dict(BWD, dY=BWD["X"], G=BWD["X"], U=BWD["X"]))
    assert not refused(host, dict(FWD, Wu=FWD["Wg"] + 2 * N * K))     # halves of one
    assert not refused(host, BWD, m=0)


@pytest.mark.parametrize("out", ["Y", "Go", "Uo"])
def test_forward_refuses(host, out):
    for other in FWD:
        if {out, other} != {"Go", "Uo"} and out != other:
            assert refused(host, dict(FWD, **{out: FWD[other]})), other
            assert refused(host, dict(FWD, **{out: FWD[other] - 4})), other   # its second element on the other's first, or the third


@pytest.mark.parametrize("out", ["dX", "dWg", "dWu", "dbg", "dbu"])
def test_backward_refuses(host, out):
    for other in BWD:
        if out != other and {out, other} not in ({"dWg", "dWu"}, {"dbg", "dbu"}):
            assert refused(host, dict(BWD, **{out: BWD[other]})), other
            assert refused(host, dict(BWD, **{out: BWD[other] - 4})), other


def test_borders(host):
    """the last element of one and the first of the next; rows in turns of one buffer"""
    for step, want in ((0, False), (2, True)):
        assert refused(host, dict(FWD, Y=FWD["X"] + 2 * M * K - step)) == want
        assert refused(host, dict(FWD, Y=FWD["X"] - 2 * M * N + step)) == want
        assert refused(host, dict(BWD, dWg=BWD["dX"] + 2 * M * K - step)) == want
        assert refused(host, dict(BWD, dWg=1 << 20, dX=(1 << 20) + 4 * N * K - 2 * step), dw_type=sa3k.TYPE_F32) == want
    # g, u and Y beside each other, and X beside them
    row = 3 * N + K
    side = dict(FWD, Y=FWD["Go"] + 2 * 2 * N, Uo=FWD["Go"] + 2 * N, X=FWD["Go"] + 2 * 3 * N)
    assert not refused(host, side, z=row, y=row, x=row)
    assert refused(host, dict(side, Y=side["Y"] - 2), z=row, y=row, x=row)
    assert refused(host, dict(side, Y=side["Y"] + 2), z=row, y=row, x=row)
    assert refused(host, side, z=row, y=2 * row, x=row) is False      # every second row's place
    assert refused(host, side, z=row, y=row + 1, x=row)


def test_rows_meet_is_what_bytes_say(host):
    rng = random.Random(5)
    found = [0, 0]
    for _ in range(4000):
        x, y = ([rng.randint(0, 60), 0, rng.randint(1, 6), rng.randint(1, 9)] for _ in range(2))
        for r in (x, y):
            r[1] = r[3] + rng.randint(0, 12)
        if rng.random() < 0.5:
            y[1] = max(x[1], y[3])
            x[1] = max(y[1], x[3])
        x[0], y[0] = x[0] + 100, y[0] + 100
        of = lambda r: {r[0] + i * r[1] + k for i in range(r[2]) for k in range(r[3])}  # noqa: E731
        want = bool(of(x) & of(y))
        found[want] += 1
        assert bool(host.meet((C.c_int64 * 4)(*x), (C.c_int64 * 4)(*y))) == want, (x, y)
    assert min(found) > 500
