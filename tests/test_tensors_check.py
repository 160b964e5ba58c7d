"""The tensor lists' checks and their cut into pieces (csrc/tensors.h), which are host arithmetic: compiled with g++ and checked
without a GPU."""
import ctypes as C
import os
import random
import subprocess

import pytest

from conftest import PKG, ROOT, sa3k

INVALID, UNSUPPORTED = 1, 4
F32, F16, BF16 = sa3k.TYPE_F32, sa3k.TYPE_F16, sa3k.TYPE_BF16
BYTES = {F32: 4, F16: 2, BF16: 2}


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("tensors") / "libtensors.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "tensors_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    lib = C.CDLL(out)
    lib.tensors.argtypes = [C.POINTER(sa3k.TensorEntry), C.c_int64]
    lib.clip.argtypes = [C.c_int, C.c_float, C.c_int64]
    lib.pieces.argtypes = [C.POINTER(sa3k.TensorEntry), C.c_int64, C.POINTER(C.c_int64), C.c_int64]
    lib.pieces.restype = C.c_int64
    return lib


def entries(ts):
    """(address, elements, type, output or None, its type)"""
    return (sa3k.TensorEntry * max(1, len(ts)))(*[sa3k.TensorEntry(g, o, n, t, ot) for g, n, t, o, ot in ts])


def check(host, *ts):
    return host.tensors(entries(ts), len(ts))


def test_accepts(host):
    assert check(host) == 0
    assert check(host, (64, 10, F32, None, F32)) == 0 and check(host, (64, 10, BF16, 64, BF16)) == 0
    assert check(host, (64, 10, BF16, 200, F32), (84, 10, BF16, 240, F32)) == 0       # end to end
    assert check(host, (0, 0, F32, None, F32)) == 0                                    # an empty one
    assert check(host, (66, 3, F16, 128, F16)) == 0
    assert check(host, (64, 10, F32, 1000, F32), (64, 10, F32, 2000, F32)) == 0       # a gradient twice
    assert check(host, (64, 10, F32, 104, F32)) == 0                                   # its output right behind it


@pytest.mark.parametrize("want,ts", [
    (UNSUPPORTED, [(64, 4, sa3k.TYPE_Q8_0, None, sa3k.TYPE_Q8_0)]), (UNSUPPORTED, [(64, 4, BF16, 128, F16)]),
    (UNSUPPORTED, [(64, 4, F32, 128, BF16)]), (INVALID, [(64, -1, F32, None, F32)]), (INVALID, [(64, 1 << 40, F32, None, F32)]),
    (INVALID, [(0, 4, F32, None, F32)]), (INVALID, [(66, 4, F32, None, F32)]), (INVALID, [(65, 4, F16, None, F16)]),
    (INVALID, [(64, 4, BF16, 130, F32)]), (INVALID, [(64, 4, BF16, None, F32)]), (INVALID, [(64, 4, BF16, 64, F32)]),
    (INVALID, [(64, 4, F32, None, F32), (64, 4, F32, None, F32)]),      # scaled twice
    (INVALID, [(64, 10, F32, 100, F32)]),                               # partly over itself
    (INVALID, [(64, 10, F32, 60, F32)]),
    (INVALID, [(64, 10, F32, 200, F32), (400, 10, F32, 239 // 4 * 4, F32)]),
    (INVALID, [(64, 10, F32, 200, F32), (204, 1, F32, 300, F32)]),      # an output over another's gradient
    (INVALID, [(1000, 100, F32, None, F32), (1100, 2, F16, 64, F16)]),
    (INVALID, [(64, 10, F32, None, F32), (64, 10, F32, 200, F32)]),     # in place, and read elsewhere
])
def test_refuses(host, want, ts):
    assert check(host, *ts) == want


def test_refuses_lists_and_calls(host):
    assert host.tensors(None, 3) == INVALID and host.tensors(None, -1) == INVALID and host.tensors(None, 0) == 0
    assert host.clip(1, 1.0, 64) == 0 and host.clip(1, 0.0, 0) == 0 and host.clip(7, float("inf"), 0) == 0
    assert host.clip(0, 1.0, 0) == INVALID and host.clip(-1, 1.0, 0) == INVALID and host.clip(1, float("nan"), 0) == INVALID
    assert host.clip(1, 1.0, 4) == INVALID


def test_overlaps_by_every_byte(host):
    """against marks on every byte, for small random lists"""
    rng = random.Random(3)
    seen = [0, 0]
    for _ in range(3000):
        ts = []
        for _ in range(rng.randint(1, 4)):
            t = rng.choice([F32, BF16])
            ot = rng.choice([t, F32])
            g, n = rng.randrange(1, 40) * 4, rng.randint(0, 6)
            o = rng.choice([None, g, rng.randrange(1, 40) * 4])
            ts.append((g, n, t, o, t if o in (None, g) else ot))
        ok = True
        span = lambda a, n, t: set(range(a, a + n * BYTES[t]))  # noqa: E731
        outs = [span(g if o is None else o, n, t if o is None else ot) for g, n, t, o, ot in ts]
        for i, (g, n, t, o, ot) in enumerate(ts):
            mine = span(g, n, t)
            for j in range(len(ts)):
                if i != j and (outs[i] & outs[j] or mine & outs[j]):
                    ok = False
            if mine & outs[i] and not (o is None or (o == g and ot == t)):
                ok = False
        assert (check(host, *ts) == 0) == ok, ts
        seen[ok] += 1
    assert min(seen) > 300


def test_pieces_cover_every_element_once(host):
    ts = [(1 << 20, 20001, F32, None, F32), (1 << 22, 1, BF16, 1 << 23, F32), (1 << 24, 0, F16, None, F16),
          (1 << 25, 16384, F16, 1 << 26, F16), (1 << 27, 16385, BF16, 1 << 28, F32), (1 << 29, 8192, F32, 1 << 30, F32)]
    out = (C.c_int64 * 400)()
    n = host.pieces(entries(ts), len(ts), out, 100)
    got = [tuple(out[4 * i:4 * i + 4]) for i in range(n)]
    want = []
    for g, k, t, o, ot in ts:
        most = 32768 // BYTES[t]
        for at in range(0, k, most):
            want.append((g + at * BYTES[t], (g if o is None else o) + at * BYTES[ot], min(most, k - at),
                         {F32: 0, F16: 1, BF16: 2}[t] | (4 if ot == F32 else 0)))
    assert got == want
