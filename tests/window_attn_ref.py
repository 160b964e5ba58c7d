"""Windowed attention in 64 bits, and the cases that its tests share."""
import torch


def visible(c, ql, kl):
    """[Sq][Sk] of one sample with ql queries and kl keys"""
    i, j = torch.arange(c["sq"])[:, None], torch.arange(c["sk"])[None, :]
    p = i + kl - ql
    ok = (i < ql) & (j < kl)
    if c["causal"]:
        ok &= j <= p
    near = torch.ones_like(ok)
    if c["left"] >= 0:
        near &= j >= p - c["left"]
    if c["right"] >= 0 and not c["causal"]:
        near &= j <= p + c["right"]
    return ok & (near | (j < c["sinks"]))


def forward(c, q, k, v):
    """q [B][Sq][H][D], k, v [B][Sk][K][D] f64 -> o, lse (natural units of the weights p too, and |p| |v|)"""
    g = c["heads"] // c["kv"]
    ok = torch.stack([visible(c, ql, kl) for ql, kl in zip(c["ql"], c["kl"])])[:, None]
    k, v = (t.transpose(1, 2).repeat_interleave(g, 1) for t in (k, v))
    # whatever lies past a sample's length is not read
    there = torch.stack([torch.arange(c["sk"]) < n for n in c["kl"]])[:, None, :, None]
    k, v = torch.where(there, k, torch.zeros_like(k)), torch.where(there, v, torch.zeros_like(v))
    rows = torch.stack([torch.arange(c["sq"]) < n for n in c["ql"]])[:, None, :, None]
    q = torch.where(rows, q.transpose(1, 2), torch.zeros_like(q.transpose(1, 2)))
    s = (q @ k.transpose(2, 3)) * c["scale"]
    s = s.masked_fill(~ok, float("-inf"))
    m = s.amax(3, keepdim=True) if c["sk"] else torch.full(s.shape[:3] + (1,), float("-inf"), dtype=s.dtype)
    e = torch.exp(s - m.masked_fill(m == float("-inf"), 0))
    l = e.sum(3, keepdim=True)
    p = e / l.masked_fill(l == 0, 1)
    lse = (m + torch.log(l))[..., 0] * 1.4426950408889634
    return dict(p=p, ok=ok, q=q, k=k, v=v, o=p @ v, lse=lse, rows=rows, absv=p @ v.abs(),
                allv=(ok.to(v.dtype) @ v.abs()), s_abs=((q.abs() @ k.abs().transpose(2, 3)) * c["scale"] * ok))


def case(name, b=1, h=2, kv=None, d=64, sq=1, sk=None, left=-1, right=-1, sinks=0, causal=False, ql=None, kl=None,
         layout="packed", scale=None):
    sk = sq if sk is None else sk
    return dict(name=name, batch=b, heads=h, kv=kv or h, dim=d, sq=sq, sk=sk, left=left, right=right, sinks=sinks,
                causal=causal, ql=[sq] * b if ql is None else ql, kl=[sk] * b if kl is None else kl, lens=ql is not None or
                kl is not None, layout=layout, scale=scale or d ** -0.5)


def widened(c):
    """the case with so many heads that it runs by tiles of 128 queries; None where it never does"""
    g = c["heads"] // c["kv"]
    if c["sq"] * g <= 32 or (c["sq"] <= 32 and c["sk"] > 1024):
        return None
    f = 128 // (c["batch"] * c["heads"] * -(-c["sq"] // 128)) + 1
    return dict(c, name=c["name"] + ", many heads", heads=c["heads"] * f, kv=c["kv"] * f)


CASES = [
    case("one token", h=3),
    case("a few tokens", h=2, kv=1, sq=5),
    case("one tile and a key", sq=65, d=128),
    case("two workgroups, dense", b=2, h=2, sq=200, ql=[200, 77], kl=[200, 77]),
    case("window both ways, first tokens", b=2, h=4, kv=2, sq=200, left=16, right=16, sinks=3, ql=[200, 131], kl=[200, 131]),
    case("window of the token itself", sq=130, left=0, right=0),
    case("window of the token itself, first tokens, causal", sq=130, left=0, sinks=2, causal=True, d=128),
    case("causal groups of four", h=8, kv=2, d=128, sq=333, left=64, sinks=4, causal=True),
    case("causal, no window", h=4, kv=4, sq=257, causal=True),
    case("one-sided bound ahead", sq=190, left=-1, right=5),
    case("one-sided bound behind", sq=190, left=7, right=-1, d=128),
    case("first tokens past a tile, far window", h=2, kv=1, d=128, sq=700, left=32, sinks=70, causal=True),
    case("first tokens ahead of the window", h=2, sq=300, left=8, right=8, sinks=100),
    case("more first tokens than keys", sq=90, left=3, right=3, sinks=500),
    case("other keys than queries", h=2, sq=100, sk=37, layout="split"),
    case("fewer keys than queries, causal: empty rows", b=2, sq=150, sk=90, causal=True, sinks=3, left=20, layout="split"),
    case("no keys, no queries", b=4, sq=70, sk=70, ql=[0, 70, 33, 70], kl=[70, 0, 5, 1], left=9, right=9, sinks=2),
    case("lengths out of range are clamped", b=2, sq=40, sk=70, ql=[40, 40], kl=[70, 0], layout="split"),
    case("step over a cache", b=2, h=8, kv=2, d=128, sq=1, sk=1000, causal=True, layout="cache", ql=[1, 1], kl=[1000, 517]),
    case("step, window and first tokens", b=3, h=4, kv=2, d=64, sq=1, sk=3000, left=255, right=0, sinks=4, causal=True,
         layout="cache", ql=[1, 1, 1], kl=[3000, 200, 1]),
    case("five new tokens, two chunks of rows", b=1, h=16, kv=2, d=128, sq=5, sk=777, left=100, sinks=64, causal=True,
         layout="cache"),
    case("32 queries, keys split", h=2, kv=2, sq=32, sk=2500, causal=True, layout="cache"),
    case("33 queries, keys split", h=4, kv=2, sq=33, sk=2500, causal=True, layout="cache", ql=[33], kl=[2441]),
    case("33 queries, few keys", h=2, kv=2, sq=33, sk=1500, causal=True, layout="cache"),
    case("many heads, few keys", b=3, h=96, kv=2, sq=2, sk=70, causal=True, layout="cache", ql=[2, 1, 2], kl=[70, 3, 66]),
    case("200 queries over many keys, split", h=2, kv=1, d=128, sq=200, sk=3500, left=3000, causal=True, sinks=4, layout="cache"),
    case("split over many workgroups", h=1, sq=3, sk=20000, layout="cache", d=128),
    case("small scale", sq=80, scale=0.01),
]
