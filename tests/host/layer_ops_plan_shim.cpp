// The sizes of the layer operators' launches and scratch (csrc/layer_ops.h) for the CPU tests.
#include "layer_ops.h"

using namespace sa3k;

extern "C" {

// i: type, batch, heads, kv_heads, head_dim, q_tokens, k_tokens, left, right, sinks, causal
static AttnShape shape(const int* i) {
    sa3k_window_attn d{};
    d.type = i[0]; d.batch = i[1]; d.heads = i[2]; d.kv_heads = i[3]; d.head_dim = i[4]; d.q_tokens = i[5];
    d.k_tokens = i[6]; d.left = i[7]; d.right = i[8]; d.sinks = i[9]; d.causal = i[10];
    return attn_shape(d, nullptr, nullptr);
}
// out: tiles, tiles with first tokens, shares of those, shares of the others, workgroups, workgroups with a place in the scratch
void key_shares(const int* i, int* out) {
    const KeySplit k = key_split(shape(i));
    out[0] = k.tiles; out[1] = k.first_tiles; out[2] = k.first; out[3] = k.rest;
    out[4] = k.items(); out[5] = k.shares();
}

// out: the shares that key_split chooses, how many plans it priced, and the cheapest of all plans priced one by one
void key_search(const int* i, int* out) {
    const AttnShape s = shape(i);
    const KeySplit k = key_split(s, &out[2]);
    out[0] = k.first; out[1] = k.rest;
    const int64_t all = s.Sq > 0 ? (s.Sq + 63) / 64 : 1, band = ((int64_t)kKeyTile + s.left + s.right + 62) / 64 + 1;
    const int64_t most = s.G * all, usual = s.G * (band < all ? band : all), pairs = (int64_t)s.B * s.K;
    const int64_t later = k.tiles - k.first_tiles, q_wgs = (int64_t)s.B * s.H * ((s.Sq + 127) / 128), k_all = (s.Sk + 63) / 64;
    const int64_t k_band = ((int64_t)128 + s.left + s.right + 62) / 64 + 1 + (s.sinks + 63) / 64;
    const double block = s.D == 64 ? 0.9 : 1.95, share = 2.0 * kKeyTile * s.D * 4 * 2 / 4e6;
    const double by_query = 0.85 * (double)q_wgs * (double)((k_band < k_all ? k_band : k_all) + 2);
    double least = 1e300;
    for (int64_t n = 1; n <= 64 && (n == 1 || usual / n >= 4); ++n)
        for (int64_t f = k.first_tiles > 0 ? n : 1; f <= (k.first_tiles > 0 ? 256 : 1); ++f) {
            if (f != n && f != 1 && most / f < 4) break;
            const int64_t len = (usual + n - 1) / n, flen = k.first_tiles > 0 ? (most + f - 1) / f : 0;
            const int64_t longest = later > 0 && len > flen ? len : k.first_tiles > 0 ? flen : (most + f - 1) / f;
            const int64_t wgs = pairs * (k.first_tiles * f + later * n);
            const double work = (double)pairs * (double)(k.first_tiles * most + later * usual) + 2.0 * (double)wgs + by_query;
            const double last = (double)(longest + 2) * block * (wgs + q_wgs <= 256 ? 1.35 : 2.0);
            double t = work * block / 256.0 > last ? work * block / 256.0 : last;
            const int64_t summed = n > 1 ? wgs : f > 1 ? pairs * k.first_tiles * f : 0;
            if (summed > 0 || n > 1) t += 4.0 + (double)summed * share;
            if (t < least) {
                least = t;
                out[3] = (int)f; out[4] = (int)n;
            }
        }
}

// out: edge and splits of a product of M x N x K
void product(int64_t M, int64_t N, int64_t K, int* out) {
    const ProdPlan p = prod_plan(M, N, K);
    out[0] = p.edge; out[1] = p.splits;
}
// a backward's dX [M][K] and dW [N][K]; out: together, then edge and splits of each
void backward(int64_t M, int64_t N, int64_t K, int* out) {
    const int64_t x[3] = {M, K, N}, w[3] = {N, K, M};
    const ProdPair p = prod_pair(x, w);
    out[0] = p.together;
    out[1] = p.a.edge; out[2] = p.a.splits; out[3] = p.b.edge; out[4] = p.b.splits;
}

}  // extern "C"
