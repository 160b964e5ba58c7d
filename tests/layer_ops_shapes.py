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

# products (M, N, K) forward: (edge of the tiles, whether K is split) that they run on, all but the first with six tiles of K or more
FORWARD = {
    (7563, 1048, 16): (256, False), (8364, 952, 324): (256, False), (8259, 129, 7722): (256, True), (40, 24, 1540): (128, True),
    (1500, 1030, 390): (128, False),
}
# backward: (dX and dW in one launch, edge of dX's tiles, whether its contraction is split, the same of dW)
BACKWARD = {
    (1313, 1739, 9179): (False, 256, False, 256, False), (8229, 133, 9050): (False, 256, False, 256, True),
    (142, 7556, 8508): (False, 256, True, 256, False), (654, 4043, 3894): (False, 128, False, 256, False),
    (16, 8431, 908): (False, 128, True, 256, False), (1922, 921, 7851): (False, 256, False, 128, False),
    (8360, 16, 938): (False, 256, False, 128, True), (8257, 16, 403): (False, 128, False, 128, True),
    (16, 7474, 406): (False, 128, True, 128, False), (528, 929, 16): (True, 128, True, 128, True),
    (2000, 130, 200): (True, 128, False, 128, True), (300, 2049, 700): (True, 128, True, 128, False),
    (2049, 2056, 1300): (True, 128, False, 128, False),
}
