"""Shapes of the layer operators that take one certain variant; that they do is checked on the CPU, what it computes on the GPU."""
from window_attn_ref import case

# backward passes whose key tiles with first tokens are shared out over workgroups, and the others are not
FIRST_SHARED = [
    case("a tile of first tokens in shares", h=1, d=64, sq=457, left=16, sinks=4, causal=True),
    case("two tiles of first tokens in shares", h=1, d=64, sq=461, left=8, sinks=130, causal=True),
    case("first tokens in shares, ragged", b=2, h=2, kv=2, d=128, sq=559, left=64, sinks=4, causal=True, ql=[559, 300],
         kl=[559, 300]),
    case("first tokens in shares, groups", b=2, h=4, kv=2, d=64, sq=1669, left=64, sinks=4, causal=True),
    case("first tokens in shares, both ways", b=1, h=2, kv=2, d=128, sq=559, left=8, right=8, sinks=130),
]
