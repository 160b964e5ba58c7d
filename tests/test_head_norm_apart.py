"""Head norms refuse an output at the address of a tensor that it may not be (csrc/head_norm.h): host arithmetic, compiled with g++
and checked without a GPU."""
import ctypes as C
import os
import subprocess

import pytest

from conftest import PKG, ROOT

P = ("q", "k", "v", "dqo", "dko", "q_gain", "k_gain", "pos", "slot", "len", "qo", "ko", "vo", "dq_gain", "dk_gain")
PLACE = {n: (i + 1) << 16 for i, n in enumerate(P)}
FWD = {n: PLACE[n] for n in ("q", "k", "v", "q_gain", "k_gain", "pos", "len", "qo", "ko", "vo")}
BWD = {n: PLACE[n] for n in ("q", "k", "dqo", "dko", "q_gain", "k_gain", "pos", "len", "qo", "ko", "dq_gain", "dk_gain")}


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("head_norm_apart") / "libhead_norm_apart.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "head_norm_apart_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return C.CDLL(out)


def apart(host, at, tokens=10, cache=0, **change):
    at = dict(at, **{k: PLACE.get(v, v) for k, v in change.items()})
    return host.apart(tokens, cache, (C.c_int64 * 15)(*[at.get(n, 0) for n in P]), int("dqo" in at))


def test_tensors_of_their_own(host):
    assert apart(host, FWD) == 0 and apart(host, BWD) == 0
    assert apart(host, FWD, slot="slot", cache=16) == 0
    assert apart(host, FWD, k="q", v="q", k_gain="q_gain", len="pos") == 0        # inputs may be the same
    assert apart(host, FWD, qo="q", ko="k", vo="v") == 0                           # in place
    assert apart(host, BWD, qo="dqo", ko="dko") == 0 and apart(host, BWD, qo="q", ko="k") == 0


@pytest.mark.parametrize("out,own", [("qo", "q"), ("ko", "k"), ("vo", "v")])
def test_forward_refuses(host, out, own):
    for other in FWD:
        if other not in (out, own):
            assert apart(host, FWD, **{out: other}) != 0, other
    assert apart(host, FWD, slot="slot", cache=16, **{out: "slot"}) == 1
    assert apart(host, FWD, qo="q", k="q") == 1       # q in place while k still reads the same heads
    assert apart(host, FWD, tokens=0, ko="q") == 0    # nothing is read or written


@pytest.mark.parametrize("out,own", [("qo", ("q", "dqo")), ("ko", ("k", "dko"))])
def test_backward_refuses(host, out, own):
    for other in BWD:
        if other != out and other not in own:
            assert apart(host, BWD, **{out: other}) != 0, other
    assert apart(host, BWD, qo="dqo", dko="dqo") == 1   # dq over a gradient that k's heads read too
