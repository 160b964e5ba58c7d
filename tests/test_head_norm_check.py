"""The head norms' argument checks, angles and launch shapes (csrc/head_norm.h), which are host arithmetic: compiled with g++ and
checked without a GPU."""
import ctypes as C
import os
import subprocess
from fractions import Fraction

import pytest

from conftest import PKG, ROOT, sa3k

INVALID, UNSUPPORTED = 1, 4
I = ("type", "batch", "tokens", "heads", "kv_heads", "head_dim", "rope_dims", "neighbours", "cache_tokens")
P = ("q", "k", "v", "dqo", "dko", "q_gain", "k_gain", "pos", "slot", "len", "qo", "ko", "vo", "dq_gain", "dk_gain")
S = ("q", "k", "v", "qo", "ko", "vo")


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("head_norm") / "libhead_norm.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "head_norm_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return C.CDLL(out)


def check(host, bwd=False, eps=1e-6, base=1e4, accumulate=0, strides=None, **kw):
    i = dict(type=sa3k.TYPE_BF16, batch=2, tokens=10, heads=4, kv_heads=2, head_dim=64, rope_dims=32, neighbours=0, cache_tokens=0)
    at = dict(q=64, k=128, qo=1024, ko=2048)
    if bwd:
        at.update(dqo=512, dko=768)
    for n, v in kw.items():
        (i if n in i else at)[n] = v
    D, H, K, T, cache = i["head_dim"], i["heads"], i["kv_heads"], i["tokens"], i["cache_tokens"] or i["tokens"]
    dense = lambda n, h: (n * h * D, h * D, D)  # noqa: E731
    st = dict(q=dense(T, H), k=dense(T, K), v=dense(T, K), qo=dense(T, H), ko=dense(cache, K), vo=dense(cache, K))
    st.update(strides or {})
    host.head_norm.argtypes = [C.POINTER(C.c_int), C.c_float, C.c_float, C.POINTER(C.c_int64), C.POINTER(C.c_int64), C.c_int, C.c_int]
    return host.head_norm((C.c_int * 9)(*[i[n] for n in I]), eps, base, (C.c_int64 * 18)(*[x for t in S for x in st[t]]),
                          (C.c_int64 * 15)(*[at.get(n, 0) for n in P]), accumulate, int(bwd))


def test_accepts(host):
    assert check(host) == 0 and check(host, bwd=True) == 0
    assert check(host, q=0, qo=0) == 0 and check(host, k=0, ko=0) == 0            # either alone
    assert check(host, q=0, qo=0, k=0, ko=0, v=64, vo=512) == 0
    assert check(host, v=64, vo=512, slot=64, cache_tokens=5) == 0
    assert check(host, q=66, qo=1026) == 0                                          # any element may start a row
    assert check(host, qo=64) == 0                                                   # in place
    assert check(host, bwd=True, qo=512) == 0
    assert check(host, batch=0, q=0, k=0, qo=0, ko=0) == 0 and check(host, tokens=0, q=0, k=0, qo=0, ko=0) == 0
    assert check(host, bwd=True, tokens=0, q=0, k=0, qo=0, ko=0, dqo=0, dko=0, dq_gain=64) == 0
    assert check(host, rope_dims=0) == 0 and check(host, rope_dims=64) == 0 and check(host, head_dim=256, rope_dims=256) == 0
    assert check(host, head_dim=8, rope_dims=0) == 0 and check(host, eps=0.0) == 0 and check(host, base=1.0) == 0
    assert check(host, strides=dict(q=(0, 0, 0), k=(0, 64, 0))) == 0                 # inputs may repeat
    assert check(host, strides=dict(qo=(2600, 65, 650))) == 0                        # head-major, rows apart by an odd number
    assert check(host, bwd=True, q=0, qo=0, dqo=0) == 0
    assert check(host, k=0, ko=0, strides=dict(k=(2560, 256, 64), ko=(9999, 128, 64))) == 0   # of no tensor


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=sa3k.TYPE_Q8_0)), (UNSUPPORTED, dict(head_dim=264)), (UNSUPPORTED, dict(head_dim=60)),
    (UNSUPPORTED, dict(batch=60, tokens=1 << 20, heads=64)), (UNSUPPORTED, dict(head_dim=0)), (UNSUPPORTED, dict(head_dim=-8)), (UNSUPPORTED, dict(rope_dims=8)), (UNSUPPORTED, dict(rope_dims=40)),
    (INVALID, dict(rope_dims=80)), (INVALID, dict(rope_dims=-16)), (INVALID, dict(neighbours=2)), (INVALID, dict(batch=-1)),
    (INVALID, dict(batch=65536)), (INVALID, dict(tokens=-1)), (INVALID, dict(tokens=1 << 28)), (INVALID, dict(batch=60000, tokens=1 << 20)),
    (INVALID, dict(heads=0)), (INVALID, dict(kv_heads=0)), (INVALID, dict(heads=65536)), (INVALID, dict(eps=-1e-6)),
    (INVALID, dict(eps=float("nan"))), (INVALID, dict(eps=float("inf"))), (INVALID, dict(base=0.5)), (INVALID, dict(base=float("nan"))),
    (INVALID, dict(base=float("inf"))), (INVALID, dict(cache_tokens=-1)), (INVALID, dict(slot=64)), (INVALID, dict(pos=66)),
    (INVALID, dict(slot=66, cache_tokens=4)), (INVALID, dict(len=2)), (INVALID, dict(q_gain=66)), (INVALID, dict(k_gain=2)),
    (INVALID, dict(q=65)), (INVALID, dict(type=sa3k.TYPE_F32, ko=2050)), (INVALID, dict(qo=0)), (INVALID, dict(q=0)),
    (INVALID, dict(v=64)), (INVALID, dict(vo=64)), (INVALID, dict(q=0, k=0, qo=0, ko=0)), (INVALID, dict(strides=dict(q=(-1, 256, 64)))),
    (INVALID, dict(strides=dict(k=(1 << 40, 256, 64)))), (INVALID, dict(strides=dict(qo=(2560, 256, 56)))),
    (INVALID, dict(strides=dict(qo=(2560, 65, 650)))), (INVALID, dict(strides=dict(qo=(0, 256, 64)))), (INVALID, dict(qo=64, strides=dict(q=(2560, 512, 64)))),
    (INVALID, dict(ko=128, slot=64, cache_tokens=10)), (INVALID, dict(v=64, vo=64, slot=64, cache_tokens=10)),
    (INVALID, dict(slot=64, cache_tokens=12, strides=dict(ko=(1280, 128, 64)))),   # the samples' caches overlap
])
def test_forward_refuses(host, want, change):
    assert check(host, **change) == want


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=7)), (INVALID, dict(dqo=0)), (INVALID, dict(dko=0)), (INVALID, dict(qo=0)), (INVALID, dict(accumulate=2)),
    (INVALID, dict(dq_gain=66)), (INVALID, dict(dk_gain=2)), (INVALID, dict(dqo=513)), (INVALID, dict(q=0, qo=0, dq_gain=64)),
    (INVALID, dict(strides=dict(q=(0, 256, 64)))),                 # dq's rows overlap as q's do
    (INVALID, dict(qo=512, strides=dict(qo=(5120, 512, 64)))),
])
def test_backward_refuses(host, want, change):
    assert check(host, bwd=True, **change) == want


def test_outputs_are_each_their_own(host):
    for kw in (dict(ko=1024), dict(v=64, vo=1024), dict(v=64, vo=2048), dict(bwd=True, ko=1024),
               dict(bwd=True, dq_gain=4096, dk_gain=4096), dict(bwd=True, dq_gain=4096, dk_gain=4096 + 4 * 63),
               dict(bwd=True, dq_gain=4096, dk_gain=4096 - 4 * 63)):
        assert check(host, **kw) == INVALID, kw
    assert check(host, bwd=True, dq_gain=4096, dk_gain=4096 + 4 * 64) == 0
    assert check(host, q_gain=64, k_gain=64) == 0   # one gain for both


def test_null_shape(host):
    assert host.head_norm_null() == INVALID


@pytest.mark.parametrize("dims", [0, 16, 32, 48, 128, 256])
@pytest.mark.parametrize("base", [1.0, 1e4, 500000.0, 1e30])
def test_turns(host, dims, base):
    """base^(-2i / dims) / 2 pi to 64 bits behind the point: in integers, by 80-digit decimal arithmetic"""
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    pi = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
    out = (C.c_uint64 * max(1, dims // 2))()
    host.turns.argtypes = [C.c_int, C.c_float, C.POINTER(C.c_uint64)]
    host.turns(dims, base, out)
    b = Decimal(C.c_float(base).value)
    for i in range(dims // 2):
        want = (b.ln() * Decimal(-2 * i) / Decimal(dims)).exp() / (2 * pi) * (1 << 64)
        assert abs(Decimal(out[i]) - want) <= 1 + 130 * want / (Decimal(1 << 64)), (i, out[i], want)


def test_launch_shapes(host):
    for dim in range(8, 257, 8):
        n = host.lanes(dim)
        assert 64 % n == 0 and n * 8 >= dim
        for heads in (1, 2, 7, 24, 65535):
            assert heads <= host.parts(heads, dim) * (64 // n) * 4 and host.parts(heads, dim) <= 65535 // 2


def test_angles_are_exact_modulo_a_turn():
    """pos times the fraction, modulo 2^64, is the angle's fraction of a turn: pos * fraction is off by pos * 2^-65 turns"""
    frac = 0x28BE60DB9391054A   # 1 / 2 pi
    for pos in (0, 1, -1, 999983, 2 ** 31 - 1, -2 ** 31):
        t = (pos % (1 << 64)) * frac % (1 << 64)
        exact = (Fraction(pos) * Fraction(frac, 1 << 64)) % 1
        assert Fraction(t, 1 << 64) == exact
