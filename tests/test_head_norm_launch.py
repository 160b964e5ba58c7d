"""The head norms' angles and launch shapes (csrc/head_norm.h), which are host arithmetic, by their stated bounds: compiled with g++
and checked without a GPU."""
import ctypes as C
import os
import subprocess
from decimal import Decimal, getcontext

import pytest

from conftest import PKG, ROOT

getcontext().prec = 60
TURN = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
BASES = [1.0, 1.0000001, 1.01, 1.5, 2.0, 10.0, 777.7, 1e4, 500000.0, 1e30, 3e38]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("head_norm_launch") / "libhead_norm_launch.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "head_norm_launch_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    lib = C.CDLL(out)
    lib.turns.argtypes = [C.c_int, C.c_float, C.POINTER(C.c_uint64)]
    return lib


def fractions(dims, base):
    """turns a position of each pair makes, by 60-digit arithmetic"""
    b = Decimal(C.c_float(base).value)
    return [(b.ln() * Decimal(-2 * i) / Decimal(dims)).exp() / TURN for i in range(dims // 2)]


@pytest.mark.parametrize("dims", [0, 16, 32, 48, 64, 80, 128, 160, 240, 256])
@pytest.mark.parametrize("base", BASES)
def test_turns(host, dims, base):
    """within 4 units of 2^-64 turns, whatever the base and the pair"""
    out = (C.c_uint64 * 128)()
    host.turns(dims, base, out)
    for i, f in enumerate(fractions(dims, base)):
        assert abs(Decimal(out[i]) - f * (1 << 64)) <= 4, (i, out[i])


@pytest.mark.parametrize("pos", [0, 1, -1, 999983, 2 ** 30 + 7, 2 ** 31 - 1, -2 ** 31])
@pytest.mark.parametrize("base", BASES)
def test_angles_of_far_positions(host, base, pos):
    """pos times the fraction of a turn, modulo 2^64 and rounded to 32 bits behind the point as the kernel does, against the angle in 60
    digits: 4 x 2^31 units of 2^-64 and the rounding's 2^-33, below 2^-30 turns"""
    dims = 256
    out = (C.c_uint64 * 128)()
    host.turns(dims, base, out)
    for i, f in enumerate(fractions(dims, base)):
        t = ((pos * out[i] + (1 << 31)) % (1 << 64)) >> 32
        off = (Decimal(t) / (1 << 32) - pos * f) % 1
        off = min(abs(off), abs(1 - off), abs(1 + off))
        assert off < Decimal(2) ** -30, (i, float(off))


def test_every_head_has_a_wave(host):
    """a wave takes `groups` groups of 64 / lanes heads: the parts hold all heads, and none is empty"""
    for dim in range(8, 257, 8):
        n = host.lanes(dim)
        assert 64 % n == 0 and n * 8 >= dim and (n == 4 or n * 4 < dim)
        per = host.groups() * (64 // n)
        for heads in (1, 2, 3, 5, 6, 7, 12, 13, 16, 24, 25, 32, 48, 49, 128, 65535):
            parts = host.parts(heads, dim)
            assert (parts - 1) * per < heads <= parts * per, (dim, heads, parts)
