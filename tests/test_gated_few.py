"""Which gated products of up to 16 rows run on the kernel for few rows (csrc/gated.h): the faster side of each shape as measured on
MI355X. Host arithmetic, compiled with g++ and checked without a GPU."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import PKG, ROOT

# (M, N, K): us on the kernel for few rows, on tiles; bf16, weights that no cache holds
MEASURED = {
    (1, 64, 1024): (5.6, 9.6), (16, 1024, 1024): (6.5, 10.6), (1, 6144, 1536): (10.0, 15.1), (16, 6144, 1536): (11.7, 15.5),
    (16, 512, 2048): (10.8, 11.6), (16, 2048, 2560): (12.2, 14.1), (1, 2048, 4608): (13.5, 16.2), (1, 1024, 4096): (12.5, 13.3),
    (16, 4096, 4096): (18.0, 19.7), (16, 4096, 8192): (36.5, 40.1), (8, 8192, 8192): (57.9, 67.6), (1, 16384, 4096): (51.5, 64.3),
    (16, 8192, 2560): (21.7, 22.5),
    (1, 1024, 8192): (23.5, 16.9), (16, 1024, 8192): (30.1, 18.1), (1, 1024, 16384): (41.7, 23.4), (16, 1024, 16384): (55.1, 24.6),
    (1, 512, 7168): (20.1, 15.0), (16, 512, 7168): (25.4, 16.3), (8, 64, 5120): (16.9, 12.9), (16, 2048, 5120): (22.7, 17.3),
    (8, 1024, 6144): (18.8, 16.2), (1, 128, 8192): (21.0, 14.6), (16, 2048, 14336): (54.0, 29.3), (16, 16384, 5120): (86.5, 60.3),
    (16, 16384, 3584): (56.3, 44.2), (16, 28672, 4096): (106.1, 90.2), (16, 8192, 14336): (111.4, 83.9), (16, 32768, 8192): (243.6, 188.8),
    # operands off the 16-byte grid, which the tiles copy first
    (1, 2047, 2050): (10.9, 23.5), (16, 333, 2559): (15.4, 16.9), (1, 2048, 4099): (28.3, 31.5), (16, 4099, 8191): (58.9, 93.3),
    (16, 16000, 4099): (72.4, 163.2), (16, 8200, 8191): (113.4, 199.1),
    (16, 333, 3583): (21.3, 18.4), (1, 1001, 4095): (28.7, 25.2), (16, 1001, 5119): (36.8, 27.4), (1, 500, 6001): (37.7, 24.9),
    (1, 1001, 8191): (53.4, 35.9), (16, 1001, 8191): (53.3, 36.6),
}


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("gated_few") / "libgated_few.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "gated_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    lib = C.CDLL(out)
    lib.plans.argtypes = [C.c_int64] * 3 + [C.POINTER(C.c_int)]
    return lib


@pytest.mark.parametrize("shape", list(MEASURED), ids=lambda s: "x".join(map(str, s)))
def test_the_faster_kernel(host, shape):
    o = (C.c_int * 11)()
    host.plans(*shape, o)
    few, tiles = MEASURED[shape]
    assert (o[0] == 1) == (few < tiles), list(o)[:2]
