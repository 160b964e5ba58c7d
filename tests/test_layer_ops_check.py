"""The layer operators' argument checks and the rules that pick a variant (csrc/layer_ops.h), which are host
arithmetic: compiled with g++ and checked without a GPU."""
import ctypes as C
import os
import random
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


ATTN_I = ("type", "batch", "heads", "kv_heads", "head_dim", "q_tokens", "k_tokens", "left", "right", "sinks", "causal")
ATTN_P = ("q", "k", "v", "o", "dO", "lse", "q_len", "k_len", "dq", "dk", "dv")


def attn(host, bwd=False, scale=0.125, strides=None, **kw):
    i = dict(type=sa3k.TYPE_BF16, batch=2, heads=4, kv_heads=2, head_dim=64, q_tokens=10, k_tokens=20, left=3, right=0,
             sinks=1, causal=0)
    at = dict(q=64, k=64, v=64, o=64)
    if bwd:
        at.update(dO=64, lse=64, dq=64, dk=64, dv=64)
    for n, v in kw.items():
        (i if n in i else at)[n] = v
    D, H, K = i["head_dim"], i["heads"], i["kv_heads"]
    st = dict(q=(i["q_tokens"] * H * D, H * D, D), k=(i["k_tokens"] * K * D, K * D, D), v=(i["k_tokens"] * K * D, K * D, D),
              o=(i["q_tokens"] * H * D, H * D, D))
    st.update(strides or {})
    host.attn.argtypes = [C.POINTER(C.c_int), C.c_float, C.POINTER(C.c_int64), C.POINTER(C.c_int64), C.c_int]
    return host.attn((C.c_int * 11)(*[i[n] for n in ATTN_I]), scale,
                     (C.c_int64 * 12)(*[x for t in "qkvo" for x in st[t]]),
                     (C.c_int64 * 11)(*[at.get(n, 0) for n in ATTN_P]), int(bwd))


def test_attn_accepts(host):
    assert attn(host) == 0 and attn(host, bwd=True) == 0
    assert attn(host, batch=0, q=0, k=0, v=0, o=0) == 0
    assert attn(host, q_tokens=0, q=0, o=0) == 0 and attn(host, bwd=True, q_tokens=0, q=0, o=0, dO=0, lse=0, dq=0) == 0
    assert attn(host, k_tokens=0, k=0, v=0) == 0
    assert attn(host, left=-1, right=-1, sinks=1 << 30) == 0
    assert attn(host, strides=dict(k=(0, 128, 0), v=(0, 64, 0))) == 0           # shared keys, for reading
    assert attn(host, strides=dict(q=(8, 5120, 64))) == 0                        # samples interleaved, for reading
    assert attn(host, bwd=True, strides=dict(q=(64 * 10 * 4, 64, 640))) == 0    # head-major


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=sa3k.TYPE_F32)), (UNSUPPORTED, dict(head_dim=96)), (INVALID, dict(heads=3)),
    (INVALID, dict(kv_heads=0)), (INVALID, dict(heads=0)), (INVALID, dict(batch=-1)), (INVALID, dict(batch=65536)),
    (INVALID, dict(q_tokens=-1)), (INVALID, dict(k_tokens=1 << 28)), (INVALID, dict(sinks=-1)), (INVALID, dict(causal=2)),
    (INVALID, dict(scale=0.0)), (INVALID, dict(scale=-1.0)), (INVALID, dict(scale=float("nan"))),
    (INVALID, dict(scale=float("inf"))), (INVALID, dict(strides=dict(q=(2560, 260, 64)))),
    (INVALID, dict(strides=dict(k=(-2560, 128, 64)))), (INVALID, dict(strides=dict(k=(2560, 56, 64)))),
    (INVALID, dict(strides=dict(v=(2560, 1 << 24, 64)))), (INVALID, dict(strides=dict(k=(1 << 40, 128, 64)))),
    (INVALID, dict(strides=dict(o=(2560, 256, 0)))), (INVALID, dict(strides=dict(o=(2552, 256, 64)))),
    (INVALID, dict(q=0)), (INVALID, dict(o=0)), (INVALID, dict(k=0)), (INVALID, dict(v=0)), (INVALID, dict(k=72)),
    (INVALID, dict(lse=66)), (INVALID, dict(q_len=65)), (INVALID, dict(k_len=2)),
    (UNSUPPORTED, dict(batch=65535, heads=64, q_tokens=4096)),
])
def test_attn_refuses(host, want, change):
    assert attn(host, **change) == want


@pytest.mark.parametrize("change", [
    dict(dO=0), dict(lse=0), dict(dq=0), dict(dk=0), dict(dv=0), dict(dq=72), dict(strides=dict(k=(0, 128, 64))),
    dict(strides=dict(v=(2560, 128, 0))), dict(strides=dict(q=(8, 5120, 64))), dict(o=0),
])
def test_attn_backward_refuses(host, change):
    assert attn(host, bwd=True, **change) == INVALID


def test_attn_null_shape(host):
    assert host.attn_null() == INVALID


FAR = 1 << 29


def sees(p, j, nk, left, right, sinks, causal):
    """the definition"""
    return 0 <= j < nk and (not causal or j <= p) and (j < sinks or p - left <= j <= p + right)


def windows(r):
    causal = r.randint(0, 1)
    return (r.choice([0, 1, 5, 40, 200, FAR]), 0 if causal else r.choice([0, 1, 5, 40, 200, FAR]), r.choice([0, 1, 4, 30, 70]),
            causal)


def test_seen_keys(host):
    """lo, n and first of a query's keys against the definition"""
    r = random.Random(1)
    out = (C.c_int * 3)()
    for _ in range(400):
        nk, w = r.randint(0, 90), windows(r)
        w = w[:2] + (min(w[2], nk),) + w[3:]
        for p in (r.randint(-20, nk), nk - 1, 0):
            if p >= nk:
                continue
            host.seen(p, nk, (C.c_int * 4)(*w), out)
            got = {j for j in range(nk) if out[0] <= j < out[0] + out[1] or j < out[2]}
            assert got == {j for j in range(nk) if sees(p, j, nk, *w)}, (p, nk, w)


def test_key_blocks(host):
    """every block with a visible key, once, in order, and none far from any"""
    r = random.Random(2)
    out = (C.c_int * 64)()
    for _ in range(600):
        nk, w, blk = r.randint(0, 260), windows(r), r.choice([8, 32, 64])
        w = w[:2] + (min(w[2], nk),) + w[3:]
        pa = r.randint(-30, max(nk - 1, 0))
        pb = min(pa + r.randint(0, 40), nk - 1)
        if pb < pa:
            continue
        n = host.blocks(pa, pb, nk, (C.c_int * 4)(*w), blk, out, 64)
        got = list(out[:n])
        assert got == sorted(set(got)) and all(0 <= b and b * blk < nk for b in got)
        need = {j // blk for p in range(pa, pb + 1) for j in range(nk) if sees(p, j, nk, *w)}
        assert need <= set(got), (pa, pb, nk, w, blk)
        assert set(got) - need <= set(range(min(got), max(got) + 1)) if need else True
        assert len(set(got) - need) <= 1 or w[0] < 0, (pa, pb, nk, w, blk, got, need)


def test_seen_from(host):
    """the queries that see a key exactly; those of a run of keys at least"""
    r = random.Random(3)
    out = (C.c_int * 2)()
    for _ in range(600):
        nq, nk, w = r.randint(1, 80), r.randint(1, 80), windows(r)
        w = w[:2] + (min(w[2], nk),) + w[3:]
        off = nk - nq
        k0 = r.randint(0, nk - 1)
        host.__getattr__("from")(k0, k0, nq, off, (C.c_int * 4)(*w), out)
        assert set(range(out[0], out[1] + 1)) == {i for i in range(nq) if sees(i + off, k0, nk, *w)}, (k0, nq, nk, w)
        k1 = min(nk - 1, k0 + r.randint(0, 50))
        host.__getattr__("from")(k0, k1, nq, off, (C.c_int * 4)(*w), out)
        need = {i for i in range(nq) for k in range(k0, k1 + 1) if sees(i + off, k, nk, *w)}
        assert need <= set(range(out[0], out[1] + 1)) and out[0] >= 0 and out[1] < nq


def test_key_items(host):
    """every tile of keys, with its shares one after another; no more workgroups than a launch takes"""
    r = random.Random(4)
    for _ in range(300):
        K, G = r.choice([1, 2, 8]), r.choice([1, 2, 8])
        sq, sk = r.randint(1, 9000), r.randint(1, 9000)
        i = (sa3k.TYPE_BF16, r.randint(1, 8), K * G, K, 64, sq, sk, r.choice([-1, 0, 100, 2000]), r.choice([-1, 0, 100]),
             r.choice([0, 4, 200, 9000]), r.randint(0, 1))
        out, few = (C.c_int * (3 * 40000))(), C.c_int()
        n = host.items((C.c_int * 11)(*i), (C.c_int64 * 12)(*[8] * 12), out, 40000, C.byref(few))
        assert 0 < n < 40000 and i[1] * K * n * 256 < 1 << 32
        got = [tuple(out[3 * k:3 * k + 3]) for k in range(n)]
        want = []
        for t in range(-(-sk // 128)):
            s = [g[2] for g in got if g[0] == t]
            assert len(set(s)) == 1 and len(s) == s[0] <= 256
            want += [(t, k, s[0]) for k in range(s[0])]
        assert got == want
        assert 1 <= few.value <= 512


def test_split_keys(host):
    """the rule that picks the forward's kernel, and that the widened cases of the attention's tests run by tiles"""
    from window_attn_ref import CASES, widened

    def split(c):
        i = (sa3k.TYPE_BF16, c["batch"], c["heads"], c["kv"], c["dim"], c["sq"], c["sk"], c["left"], c["right"], c["sinks"],
             int(c["causal"]))
        return host.split_keys((C.c_int * 11)(*i), (C.c_int64 * 12)(*[8] * 12))

    base = dict(batch=1, heads=32, kv=8, dim=128, sq=1, sk=100, left=-1, right=-1, sinks=0, causal=True)
    assert split(base) == 1 and split(dict(base, sq=512)) == 1 and split(dict(base, sq=513)) == 0
    assert split(dict(base, batch=8, sq=8)) == 1 and split(dict(base, batch=8, sq=9)) == 0
    assert split(dict(base, batch=8, sq=32, sk=1025)) == 1 and split(dict(base, batch=8, sq=33, sk=1025)) == 0
    wide = [w for w in map(widened, CASES) if w]
    assert len(wide) > 15 and not any(split(w) for w in wide)
    assert any(split(c) for c in CASES)


PROD_P = ("x", "w", "r", "dy", "z", "y", "zo", "dx", "dw", "bias", "db")


def prod(host, bwd=False, type=sa3k.TYPE_BF16, act=sa3k.ACT_GELU, M=10, N=24, K=40, dw_type=None, accumulate=0, ld=None, **p):
    at = dict(x=64, w=64, y=64) if not bwd else dict(x=64, w=64, dy=64, z=64, dx=64, dw=64, db=64)
    at.update(p)
    lds = dict(x=K, w=K, r=N, dy=N, z=N, y=N, dx=K, dw=K)
    lds.update(ld or {})
    I64 = C.POINTER(C.c_int64)
    host.prod.argtypes = [C.c_int, C.c_int, I64, I64, I64, C.c_int, C.c_int, C.c_int]
    return host.prod(type, act, (C.c_int64 * 3)(M, N, K), (C.c_int64 * 11)(*[at.get(n, 0) for n in PROD_P]),
                     (C.c_int64 * 8)(*[lds[n] for n in ("x", "w", "r", "dy", "z", "y", "dx", "dw")]),
                     type if dw_type is None else dw_type, accumulate, int(bwd))


def test_prod_accepts(host):
    assert prod(host) == 0 and prod(host, bwd=True) == 0
    assert prod(host, r=64, zo=64, bias=64) == 0 and prod(host, M=1, N=1, K=1) == 0
    assert prod(host, x=66, w=34, y=2, ld=dict(x=41, w=43, y=25)) == 0      # any element may start a row
    assert prod(host, M=0, x=0, y=0) == 0
    assert prod(host, bwd=True, M=0, dy=0, z=0, x=0) == 0
    assert prod(host, bwd=True, act=sa3k.ACT_NONE, z=0) == 0
    assert prod(host, bwd=True, dx=0, w=0) == 0 and prod(host, bwd=True, dw=0, x=0) == 0
    assert prod(host, bwd=True, dx=0, dw=0, w=0, x=0) == 0
    assert prod(host, bwd=True, dw_type=sa3k.TYPE_F32, accumulate=1) == 0


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=sa3k.TYPE_F32)), (INVALID, dict(act=5)), (INVALID, dict(act=-1)), (INVALID, dict(M=-1)),
    (INVALID, dict(N=0)), (INVALID, dict(K=0)), (INVALID, dict(K=1 << 22)), (INVALID, dict(M=1 << 31)), (INVALID, dict(w=0)),
    (INVALID, dict(x=0)), (INVALID, dict(y=0)), (INVALID, dict(ld=dict(x=39))), (INVALID, dict(ld=dict(w=1 << 22))),
    (INVALID, dict(ld=dict(y=23))), (INVALID, dict(x=65)), (INVALID, dict(y=33)), (INVALID, dict(bias=66)),
    (INVALID, dict(r=64, ld=dict(r=23))), (UNSUPPORTED, dict(M=1 << 27, N=1 << 14)),
])
def test_prod_forward_refuses(host, want, change):
    assert prod(host, **change) == want


@pytest.mark.parametrize("want,change", [
    (UNSUPPORTED, dict(type=8)), (INVALID, dict(dy=0)), (INVALID, dict(z=0)), (INVALID, dict(x=0)), (INVALID, dict(w=0)),
    (INVALID, dict(accumulate=2)), (INVALID, dict(accumulate=1)), (INVALID, dict(dw_type=sa3k.TYPE_F16)),
    (INVALID, dict(dw_type=sa3k.TYPE_F32, dw=66)), (INVALID, dict(db=2)), (INVALID, dict(ld=dict(dx=39))),
    (INVALID, dict(ld=dict(dw=39))), (INVALID, dict(ld=dict(dy=23))), (INVALID, dict(ld=dict(z=23))),
])
def test_prod_backward_refuses(host, want, change):
    assert prod(host, bwd=True, **change) == want


def test_prod_plan(host):
    """the splits cover K, none is empty, their sums fit"""
    r = random.Random(5)
    out = (C.c_int * 3)()
    host.plan.argtypes = [C.c_int64, C.c_int64, C.c_int64, C.POINTER(C.c_int)]
    seen = set()
    for _ in range(3000):
        M, N, K = (int(2 ** r.uniform(0, 14)) for _ in range(3))
        host.plan(M, N, K, out)
        edge, splits, per = out
        kt = -(-K // 64)
        assert edge in (128, 256) and splits * per >= kt and (splits - 1) * per < kt
        assert splits == 1 or splits * M * (N + 8) <= 1 << 26
        seen.add((edge, splits > 1))
    assert len(seen) == 4   # both tiles, split and not


def test_prod_pair(host):
    """as the plan of one product; together only on tiles of 128"""
    r = random.Random(6)
    out, I = (C.c_int * 7)(), C.c_int64 * 3
    seen = set()
    for _ in range(2000):
        M, N, K = (int(2 ** r.uniform(0, 13)) for _ in range(3))
        host.pair(I(M, K, N), I(N, K, M), out)
        for (edge, splits, per), (m, n, k) in ((out[1:4], (M, K, N)), (out[4:7], (N, K, M))):
            kt = -(-k // 64)
            assert edge == 128 or (edge == 256 and not out[0])
            assert splits * per >= kt and (splits - 1) * per < kt and (splits == 1 or splits * m * (n + 8) <= 1 << 26)
        seen.add(out[0])
    assert seen == {0, 1}
