"""What the layer operators' launches take (csrc/layer_ops.h, host arithmetic): the scratch of shared key tiles, and that the GPU
tests' shapes reach the variants that they are there for."""
import ctypes as C
import os
import random
import subprocess

import pytest

from conftest import PKG, ROOT, sa3k
from layer_ops_shapes import BACKWARD, FIRST_SHARED, FORWARD


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("layer_ops_plans") / "liblayer_ops_plans.so")
    cmd = ["g++", "-std=c++17", "-O2", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror", "-I", os.path.join(ROOT, "include"),
           "-I", os.path.join(PKG, "csrc"), os.path.join(ROOT, "tests", "host", "layer_ops_plan_shim.cpp"), "-o", out]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-4000:]
    return C.CDLL(out)


def shares(host, batch, heads, kv, dim, sq, sk, left=-1, right=-1, sinks=0, causal=True):
    """tiles, tiles with first tokens, shares of those, shares of the others, workgroups, places in the scratch"""
    out = (C.c_int * 6)()
    host.key_shares((C.c_int * 11)(sa3k.TYPE_BF16, batch, heads, kv, dim, sq, sk, left, right, sinks, int(causal)), out)
    return tuple(out)


def test_scratch_holds_the_shares_and_no_more(host):
    """a place for every workgroup of a tile that more than one takes, in the order of the workgroups, none for the others"""
    r = random.Random(1)
    seen = set()
    for _ in range(3000):
        K, s = r.choice([1, 2, 8]), int(2 ** r.uniform(0, 14))
        tiles, first_tiles, first, rest, wgs, places = shares(
            host, r.randint(1, 4), K * r.choice([1, 4]), K, r.choice([64, 128]), s, s, r.choice([-1, 16, 500, 4000]),
            r.choice([-1, 16, 500]), r.choice([0, 4, 200]), r.random() < 0.5)
        assert wgs == first_tiles * first + (tiles - first_tiles) * rest
        split = [n > 1 for t in range(tiles) for n in [first if t < first_tiles else rest] for _ in range(n)]
        assert places == sum(split) and all(split[:places])
        seen.add((first_tiles > 0, first > 1, rest > 1))
    assert {(True, True, False), (True, True, True), (False, False, True), (False, False, False)} <= seen


@pytest.mark.parametrize("batch,s,left,most", [(2, 8192, 1023, 2), (4, 32768, 127, 3), (4, 131072, 127, 3)])
def test_long_windows_with_first_tokens_take_little_scratch(host, batch, s, left, most):
    """32 on 8 heads of 128, 4 first tokens: only their tile is shared out, whatever the length"""
    tiles, first_tiles, first, rest, wgs, places = shares(host, batch, 32, 8, 128, s, s, left, 0, 4)
    assert (first_tiles, rest) == (1, 1) and wgs >= s // 128 and places == first and 1 < places <= most


@pytest.mark.parametrize("c", FIRST_SHARED, ids=[c["name"] for c in FIRST_SHARED])
def test_shapes_share_first_tokens_only(host, c):
    tiles, first_tiles, first, rest, _, _ = shares(host, c["batch"], c["heads"], c["kv"], c["dim"], c["sq"], c["sk"], c["left"],
                                                   c["right"], c["sinks"], c["causal"])
    assert first > 1 and rest == 1 and tiles > first_tiles > 0


def search(host, batch, heads, kv, dim, sq, sk, left=-1, right=-1, sinks=0, causal=True):
    """(shares of tiles with first tokens, of the others) as chosen, the plans priced for that, and the cheapest of all plans"""
    out = (C.c_int * 5)()
    host.key_search((C.c_int * 11)(sa3k.TYPE_BF16, batch, heads, kv, dim, sq, sk, left, right, sinks, int(causal)), out)
    return (out[0], out[1]), out[2], (out[3], out[4])


def test_key_split_finds_the_cheapest_plan(host):
    r = random.Random(2)
    for _ in range(4000):
        K, sq = r.choice([1, 2, 4, 8]), int(2 ** r.uniform(0, 16))
        sk = sq if r.random() < 0.7 else int(2 ** r.uniform(0, 16))
        args = (r.randint(1, 8), K * r.choice([1, 2, 4, 8, 32]), K, r.choice([64, 128]), sq, sk, r.choice([-1, 0, 16, 1000]),
                r.choice([-1, 0, 16, 500]), r.choice([0, 1, 4, 64, 200, 5000, 1 << 20]), r.random() < 0.5)
        chosen, _, best = search(host, *args)
        assert chosen == best, args


@pytest.mark.parametrize("args", [(3, 16, 2, 128, 2049, 2049, 511, 0, 4), (1, 32, 8, 128, 8192, 8192, 1023, 0, 4),
                                  (1, 32, 8, 128, 32768, 32768, 1023, 0, 4), (1, 32, 1, 64, 1024, 1024, -1, -1, 4),
                                  (1, 16, 2, 128, 8192, 8192, 4095, 0, 4), (2, 24, 24, 64, 1088, 1088, 128, 128, 64, False)])
def test_key_split_prices_few_plans(host, args):
    """each call of the backward chooses anew: a plan takes about 8 ns to price, so that 64 of them are half a microsecond"""
    assert search(host, *args)[1] <= 64


def product(host, M, N, K):
    """edge of the tiles, splits of K"""
    out, I = (C.c_int * 2)(), C.c_int64
    host.product(I(M), I(N), I(K), out)
    return tuple(out)


def backward(host, M, N, K):
    """dX and dW together, edge and splits of dX, of dW"""
    out, I = (C.c_int * 5)(), C.c_int64
    host.backward(I(M), I(N), I(K), out)
    return tuple(out)


@pytest.mark.parametrize("shape", list(FORWARD))
def test_forward_shapes_reach_their_tiles(host, shape):
    M, N, K = shape
    for k in (K, -(-K // 8) * 8):   # as they are, and in padded rows
        edge, splits = product(host, M, N, k)
        assert (edge, splits > 1) == FORWARD[shape]
    assert -(-K // 64) >= 6 or shape == (7563, 1048, 16)


@pytest.mark.parametrize("shape", list(BACKWARD))
def test_backward_shapes_reach_their_tiles(host, shape):
    together, ex, sx, ew, sw = backward(host, *shape)
    assert (bool(together), ex, sx > 1, ew, sw > 1) == BACKWARD[shape]


def test_shapes_cover_every_variant(host):
    """those of 4000 drawn shapes, of up to 2^13 rows, columns and length"""
    assert set(FORWARD.values()) == {(128, False), (128, True), (256, False), (256, True)}
    r, seen = random.Random(3), set()
    for _ in range(4000):
        together, ex, sx, ew, sw = backward(host, *(int(2 ** r.uniform(4, 13.2)) for _ in range(3)))
        seen.add((bool(together), ex, sx > 1, ew, sw > 1))
    assert seen <= set(BACKWARD.values()), seen - set(BACKWARD.values())
    M, N, K = 1313, 1739, 9179   # its single gradients are there on 256 x 256 tiles, too
    assert product(host, M, K, N)[0] == product(host, N, K, M)[0] == 256
