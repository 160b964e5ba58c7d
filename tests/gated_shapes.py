"""Shapes of gated products that take one certain variant; that they do is checked on the CPU, what it computes on the GPU."""

# (M, N, K) forward: (edge of the tiles, or blocks of few rows; whether K is split)
FORWARD = {
    (417, 8435, 316): (256, False), (33, 82, 302): (128, False), (35, 80, 516): (128, True), (156, 8820, 3596): (256, True),
    (513, 6632, 325): (256, False), (155, 8511, 4009): (256, True), (396, 9688, 16): (256, False), (300, 520, 1000): (128, True), (17, 82, 302): (2, False), (19, 80, 516): (2, False),
    (32, 8192, 40): (2, False), (31, 8193, 40): (128, False), (32, 40, 1024): (2, False), (17, 40, 1032): (128, True),
    (17, 40, 1025): (2, False), (21, 40, 2049): (128, True), (32, 2048, 2049): (2, False), (29, 8200, 250): (2, False),
    (16, 33, 2000): (1, False),
}
# backward, both products: (dX and dW in one launch, edge of dX's tiles, whether its contraction is split, the same of dW)
BACKWARD = {
    (139, 141, 158): (True, 128, False, 128, False), (421, 1503, 5364): (True, 128, False, 128, False),
    (16, 195, 16): (True, 128, True, 128, False), (142, 8768, 409): (True, 128, True, 128, False),
    (644, 18, 16): (True, 128, False, 128, True), (7375, 144, 6594): (True, 128, False, 128, True),
    (158, 278, 130): (True, 128, True, 128, True), (858, 141, 132): (True, 128, True, 128, True),
    (1310, 446, 132): (True, 128, True, 128, True), (1728, 745, 8765): (True, 256, False, 256, False),
    (131, 3914, 8405): (True, 256, True, 256, False), (131, 8117, 149): (False, 128, True, 128, False),
    (9766, 16, 672): (False, 128, False, 128, True), (1775, 1098, 4583): (False, 128, False, 256, False),
    (16, 11997, 276): (False, 128, True, 256, False), (2728, 685, 5560): (False, 256, False, 128, False),
    (12111, 18, 1153): (False, 256, False, 128, True), (2321, 2250, 1695): (False, 256, True, 128, False),
}
# a backward product by itself: (edge of its tiles, whether its contraction is split)
DX_ALONE = {(17, 267, 48): (128, True), (17, 16, 200): (128, False), (4609, 16, 1700): (256, False), (136, 3538, 8222): (256, True)}
DW_ALONE = {(589, 20, 136): (128, True), (17, 64, 1000): (128, False), (16, 8830, 392): (256, False), (3073, 8899, 135): (256, True)}
