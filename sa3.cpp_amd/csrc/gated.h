// Host-side arithmetic of the gated products: their backward's plan and the checks of their arguments. No HIP in here: compiled
// with g++ in the CPU tests too.
#pragma once

#include "layer_ops.h"

namespace sa3k {

struct GatedArgs {
    int type = 0, act = 0;
    int64_t M = 0, N = 0, K = 0;
    const void *X = nullptr, *Wg = nullptr, *Wu = nullptr, *dY = nullptr, *G = nullptr, *U = nullptr;
    void *Y = nullptr, *Go = nullptr, *Uo = nullptr, *dX = nullptr, *dWg = nullptr, *dWu = nullptr;   // Go, Uo: the forward's g and u
    int64_t ldx = 0, ldw = 0, lddy = 0, ldz = 0, ldy = 0, lddx = 0, lddw = 0;
    const float *bg = nullptr, *bu = nullptr;
    float *dbg = nullptr, *dbu = nullptr;
    int dw_type = 0, accumulate = 0;
};

// gate's and up's gradients lie side by side, each padded to whole tiles of 64
inline int64_t gated_half(int64_t N) { return (N + 63) / 64 * 64; }

// The blocks of 16 rows that the kernel for few rows takes (0: tiles). A workgroup of it reads 16 columns' weights whole, so long rows (K)
// on fewer workgroups (N / 16) than CUs wait for memory where the tiles split K, and x, read again for every 16 columns, takes
// over with more than 8 rows of large weights. Measured on MI355X, bf16, us (few / tiles), 1 and 16 rows: 1536 -> 6144 10.0 / 15.1 and 11.7 /
// 15.5, 4608 -> 2048 13.5 / 16.2 and 16.8 / 16.4, 4608 -> 64 11.1 / 12.9 and 14.2 / 12.8, 5120 -> 2048 18.7 / 17.1 and 22.7 / 17.3, 8192 ->
// 1024 23.5 / 16.9 and 30.1 / 18.1, 16384 -> 1024 41.7 / 23.4 and 55.1 / 24.6, 8192 -> 4096 32.4 / 39.5 and 36.5 / 40.1, 3584 -> 16384
// 47.0 / 44.4 and 56.3 / 44.2, 5120 -> 16384 70.1 / 59.8 and 86.5 / 60.3, 8192 -> 8192 54.4 / 67.7 and 63.2 / 67.5.
// A second block pays while the weights are one round of loads (K) on one round of workgroups (N): 32 rows 1024 -> 4096 7.5 / 12.8, 512 ->
// 1024 6.8 / 9.7, 768 -> 8192 9.7 / 12.2, 128 -> 512 7.1 / 7.2; past that 1536 -> 6144 16.0 / 15.1, 256 -> 20000 18.0 / 10.7, 8192 -> 1024
// 30.3 / 17.5. Operands off the tiles' 16-byte grid, which those copy first (padded), run here unless few workgroups have long rows to
// read: 1 row 2559 -> 333 15.0 / 16.5, 4095 -> 1001 28.7 / 25.2, 8191 -> 1001 53.4 / 35.9, 8191 -> 4099 56.9 / 92.5, 16 rows 4099 -> 16000 72 /
// 163, 32 rows 4100 -> 11008 47 / 123, 1535 -> 6144 20.6 / 31.5, 255 -> 20000 22.5 / 24.6, 4095 -> 256 20.9 / 18.5, 8191 -> 1024 47 / 32.
inline int few_blocks(int64_t M, int64_t N, int64_t K, bool padded) {
    if (M > 2 * kFewRows) return 0;
    if (M > kFewRows) return (padded ? N >= 2048 || K <= 2048 : K <= 1024 && N <= 8192) ? 2 : 0;
    if (padded) return N >= 2048 || K <= 2560 ? 1 : 0;
    return (N >= 4096 || K <= 4608) && (M <= 8 || N * K <= 40000000) ? 1 : 0;
}

// tiles of an M x N result that an XCD takes of a launch, and how many its 32 CUs hold at a time
inline int64_t xcd_tiles(int edge, int64_t M, int64_t N) { return ((M + edge - 1) / edge * ((N + edge - 1) / edge) + 7) / 8; }
inline int64_t xcd_slots(int edge) { return edge == 256 ? 32 : 64; }

// The forward's plan: rounds of workgroups on an XCD, and the split sums. The times are fitted to whole calls on MI355X at 136 shapes of
// 17 to 8191 rows, 128 and 256 wide tiles, 1 to 16 splits, 9% off them; the plan chosen is 0.6% above the best of them on average and
// 11% at most (prod_plan 2.8% and 26%). bf16, us (M x K -> N: prod_plan's / this one's): 1836 x 384 -> 4433 45 / 34 (128 whole), 56 x
// 3768 -> 1045 19.4 / 16.3 (128, six splits), 17 x 1536 -> 6144 16.5 / 14.8 (128, two).
inline ProdPlan gated_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t kt = (K + 63) / 64;
    ProdPlan best{128, 1, (int)kt, 1e300};
    for (int edge = 256; edge >= 128; edge /= 2) {
        const int64_t tiles = xcd_tiles(edge, M, 2 * N), slots = xcd_slots(edge);
        for (int64_t n = 1; n <= 16; ++n) {
            if (!split_fits(n, kt, M, 2 * N)) continue;
            const int64_t per = (kt + n - 1) / n, wgs = tiles * n;
            const double wg = edge == 256 ? 1.6 * (double)per + 8.1 : (wgs <= 32 ? 0.44 : 0.98) * (double)per + 5.8;
            const double sums = n > 1 ? 0.6 + 0.3 * (double)n + 16.0 * (double)n * (double)M * (double)N / 4.5e6 : 0.0;
            const double t = (double)((wgs + slots - 1) / slots) * wg + sums;
            if (t < best.us) best = ProdPlan{edge, (int)n, (int)per, t};
        }
    }
    return best;
}

// The backward products' plan: one after the other, or both in one launch of 128 x 128 or 256 x 256 tiles, dX's workgroups first. A
// launch ends with its last workgroup: each XCD takes every eighth; its 32 CUs hold 64 of the small tiles or 32 of the large, and
// after the last full round of dX's, nx % slots of those start dW's later than the rest (pair_span). The times below are fitted to
// whole calls on MI355X at 160 shapes of 16 to 40000 rows and at all their splits, 9% off them; the plan chosen is 1.6% above the
// best of them on average and 13% at most (with the other products' plan, prod_pair, 6.8%). The large tiles' dW stays whole: in two
// splits it lost on every shape tried. bf16, us (M x K -> N: prod_pair's plan / this one): 2176 x 1536 -> 6144 212 / 194 (256, dX in
// four splits), 8192 x 1536 -> 6144 769 / 626 (256, whole), 4096 x 2048 -> 2048 155 / 137 (256, whole), 512 x 4096 -> 11008 280 / 260
// (256, three), 1031 x 1001 -> 2731 63.5 / 55 (256, six), 1500 x 1024 -> 2048 60 / 47 (128, two), 2982 x 304 -> 1496 54 / 42 (128,
// three and three), 784 x 760 -> 1848 32 (128, five, as before).
inline double pair_span(int64_t nx, double tx, int64_t nw, double tw, int64_t slots) {
    const int64_t late = nx % slots;
    const double early_from = (double)(nx / slots) * tx, late_from = early_from + tx;
    // no end is before the work shared evenly, nor before the last of dX's
    const double shared = ((double)nx * tx + (double)nw * tw) / (double)slots, least = late && late_from > shared ? late_from : shared;
    double best = 1e300;
    for (int side = 0; side < 2; ++side) {   // the last end lies whole workgroups of dW after one of both starts
        const double from = side ? early_from : late_from;
        for (int64_t k = least > from ? (int64_t)((least - from) / tw) : 0;; ++k) {
            const double end = from + (double)k * tw;
            if (late && end < late_from) continue;
            const int64_t by_late = late ? (int64_t)((end - late_from) / tw + 1e-9) * late : 0;
            if (by_late + (int64_t)((end - early_from) / tw + 1e-9) * (slots - late) < nw) continue;
            if (end < best) best = end;
            break;
        }
    }
    return best;
}
// Microseconds of a workgroup with `per` tiles of 64 along K, of a launch that gives each XCD `wgs` workgroups; of the pass over
// the split sums of M x N; and of a product in a launch of its own.
inline double pair_wg_us(int edge, int64_t wgs, int64_t per) {
    return edge == 256 ? 1.43 * (double)per + 7.4 : (wgs <= 32 ? 0.74 : 0.94) * (double)per + 3.7;
}
inline double pair_sum_us(int64_t n, int64_t M, int64_t N) { return n > 1 ? 8.0 * (double)n * (double)M * (double)N / 6.7e6 : 0.0; }
constexpr double kPairSums = 4.6;   // a launch that adds splits up
inline double alone_us(const ProdPlan& p, int64_t M, int64_t N) {
    const int64_t n = xcd_tiles(p.edge, M, N) * p.splits, slots = xcd_slots(p.edge);
    const double sums = p.splits > 1 ? pair_sum_us(p.splits, M, N) + kPairSums : 0.0;
    return (double)((n + slots - 1) / slots) * pair_wg_us(p.edge, n, p.per) + sums;
}
inline ProdPair gated_pair(int64_t M, int64_t N, int64_t K, const ProdPlan& x, const ProdPlan& w) {
    const int64_t cols = 2 * gated_half(N), kx = cols / 64, kw = (M + 63) / 64;
    ProdPair best{false, x, w};
    double least = alone_us(x, M, K) + alone_us(w, cols, K) + 9.4;
    constexpr int kMost = 8;     // splits
    int64_t per[2][kMost + 1];   // tiles of 64 along K that a split of dX, of dW takes; 0: not one to try
    double sums[2][kMost + 1];
    for (int64_t n = 1; n <= kMost; ++n) {
        per[0][n] = split_fits(n, kx, M, K) ? (kx + n - 1) / n : 0;
        per[1][n] = split_fits(n, kw, cols, K) ? (kw + n - 1) / n : 0;
        sums[0][n] = pair_sum_us(n, M, K);
        sums[1][n] = pair_sum_us(n, cols, K);
    }
    for (int edge = 128; edge <= 256; edge *= 2) {
        const int64_t slots = xcd_slots(edge), tiles_x = xcd_tiles(edge, M, K), tiles_w = xcd_tiles(edge, cols, K);
        for (int n = 1; n <= kMost; ++n)
            for (int m = 1; m <= (edge == 256 ? 1 : kMost); m += m < 4 ? 1 : 2) {
                if (!per[0][n] || !per[1][m]) continue;
                const int64_t nx = tiles_x * n, nw = tiles_w * m;
                const double tx = pair_wg_us(edge, nx + nw, per[0][n]), tw = pair_wg_us(edge, nx + nw, per[1][m]);
                const double rest = sums[0][n] + sums[1][m] + (n > 1 || m > 1 ? kPairSums : 0.0) + (edge == 256 ? 1.6 : 0.0);
                if (((double)nx * tx + (double)nw * tw) / (double)slots + rest >= least) continue;   // no span is below that
                const double t = pair_span(nx, tx, nw, tw, slots) + rest;
                if (t >= least) continue;
                least = t;
                best = ProdPair{true, ProdPlan{edge, n, (int)per[0][n], t}, ProdPlan{edge, m, (int)per[1][m], t}};
            }
    }
    return best;
}

// Rows in memory, in bytes. (A pitch is no shorter than its rows, but where there is one row.)
struct Rows {
    uintptr_t at;
    int64_t ld, n, width;
};
inline Rows rows_of(const void* p, int64_t ld, int64_t n, int64_t cols, int bytes) {
    return Rows{reinterpret_cast<uintptr_t>(p), ld * bytes, p && n > 0 ? n : 0, cols * bytes};
}
// whether a byte is of both: rows that take turns in one buffer have none
inline bool rows_meet(const Rows& x, const Rows& y) {
    if (x.n == 0 || y.n == 0) return false;
    auto end = [](const Rows& r) { return r.at + (uintptr_t)((r.n - 1) * r.ld + r.width); };
    if (end(x) <= y.at || end(y) <= x.at) return false;
    if (x.n > 1 && y.n > 1 && x.ld == y.ld) {   // the higher one's rows begin r behind rows q, q + 1, .. of the lower one
        const Rows &lo = x.at < y.at ? x : y, &hi = x.at < y.at ? y : x;
        const int64_t d = (int64_t)(hi.at - lo.at), q = d / lo.ld, r = d % lo.ld;
        return (q < lo.n && r < lo.width) || (q + 1 < lo.n && lo.ld - r < hi.width);
    }
    // Other pitches within one range of addresses: row by row of the one with fewer
    const Rows &a = x.n <= y.n ? x : y, &b = x.n <= y.n ? y : x;
    for (int64_t i = 0; i < a.n; ++i) {
        const int64_t from = (int64_t)(a.at - b.at) + i * a.ld;   // from b's first row on
        const int64_t j = from < b.width ? 0 : (from - b.width) / b.ld + 1;   // the first of b's rows that ends behind it
        if (j < b.n && j * b.ld < from + a.width) return true;
    }
    return false;
}

inline const char* gated_check(const GatedArgs& a, bool bwd, int* code) {
    *code = SA3K_ERR_INVALID;
    if (a.type != SA3K_TYPE_BF16 && a.type != SA3K_TYPE_F16) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "type must be bf16 or f16";
    }
    if (a.act < SA3K_ACT_NONE || a.act > SA3K_ACT_GELU_TANH) return "unknown activation";
    if (a.M < 0 || a.M >= kMaxExtent) return "M out of range";
    if (a.N <= 0 || a.K <= 0 || 2 * gated_half(a.N) >= kProdMaxPitch || a.K >= kProdMaxPitch) return "N or K out of range";
    if (bwd && a.accumulate != 0 && a.accumulate != 1) return "accumulate must be 0 or 1";
    if (bwd && !a.dWg != !a.dWu) return "the gradients of both weights, or of neither";
    if (bwd && a.dWg && a.dw_type != a.type && a.dw_type != SA3K_TYPE_F32) return "dw_type must be f32 or type";
    if (bwd && a.dWg && a.accumulate && a.dw_type != SA3K_TYPE_F32) return "only an f32 dW can be added to";
    const void* p[12] = {a.X, a.Wg, a.Wu, a.dY, a.G, a.U, a.Y, a.Go, a.Uo, a.dX, a.dWg, a.dWu};
    const int64_t ld[12] = {a.ldx, a.ldw, a.ldw, a.lddy, a.ldz, a.ldz, a.ldy, a.ldz, a.ldz, a.lddx, a.lddw, a.lddw};
    const int64_t w[12] = {a.K, a.K, a.K, a.N, a.N, a.N, a.N, a.N, a.N, a.K, a.K, a.K};
    for (int i = 0; i < 12; ++i) {
        if (!p[i]) continue;
        if (ld[i] < w[i] || ld[i] >= kProdMaxPitch) return "a row pitch is smaller than its rows or out of range";
        if (!elem_aligned(p[i], i >= 10 ? elem_bytes(a.dw_type) : 2)) return "a tensor is not aligned to its elements";
    }
    const void* f[4] = {a.bg, a.bu, a.dbg, a.dbu};
    for (const void* x : f)
        if (!elem_aligned(x, 4)) return "an f32 vector is not 4-byte aligned";
    // a launch has fewer than 2^24 workgroups: tiles of 64 x 64 at the least, and the split sums' 2048 values
    const int64_t cols = 2 * gated_half(a.N);
    if (((a.M + 63) / 64) * ((cols > a.K ? cols : a.K) / 64 + 1) >= ((int64_t)1 << 23)) {
        *code = SA3K_ERR_UNSUPPORTED;
        return "M x N is too large for one launch";
    }
    const int wb = elem_bytes(a.dw_type);
    if (rows_meet(rows_of(a.Go, a.ldz, a.M, a.N, 2), rows_of(a.Uo, a.ldz, a.M, a.N, 2)) ||
        rows_meet(rows_of(a.dWg, a.lddw, a.N, a.K, wb), rows_of(a.dWu, a.lddw, a.N, a.K, wb)) ||
        rows_meet(rows_of(a.dbg, a.N, 1, a.N, 4), rows_of(a.dbu, a.N, 1, a.N, 4)))
        return "gate's output meets up's";
    if (!bwd) {
        if (!a.Wg || !a.Wu) return "the weights must not be null";
        if (a.M > 0 && (!a.X || !a.Y)) return "X and Y must not be null";
    } else {
        if (a.M > 0 && (!a.dY || !a.G || !a.U)) return "dY, G and U must not be null";
        if (a.M > 0 && a.dWg && !a.X) return "dW needs X";
        if (a.dX && (!a.Wg || !a.Wu)) return "dX needs the weights";
    }
    return nullptr;
}

// What gated_check found in order, taken two by two: an output that meets another output would be written over (Y over the kept g
// leaves a wrong g behind), one that meets an input is written while other workgroups still read that.
inline const char* gated_apart(const GatedArgs& a, bool bwd) {
    const int wb = bwd ? elem_bytes(a.dw_type) : 2;
    auto vec = [&](const void* p) { return rows_of(p, a.N, 1, a.N, 4); };
    const Rows out[8] = {rows_of(a.Y, a.ldy, a.M, a.N, 2), rows_of(a.Go, a.ldz, a.M, a.N, 2), rows_of(a.Uo, a.ldz, a.M, a.N, 2),
                         rows_of(a.dX, a.lddx, a.M, a.K, 2), rows_of(a.dWg, a.lddw, a.N, a.K, wb),
                         rows_of(a.dWu, a.lddw, a.N, a.K, wb), vec(a.dbg), vec(a.dbu)};
    const Rows in[8] = {rows_of(a.X, a.ldx, a.M, a.K, 2), rows_of(a.Wg, a.ldw, a.N, a.K, 2), rows_of(a.Wu, a.ldw, a.N, a.K, 2),
                        rows_of(a.dY, a.lddy, a.M, a.N, 2), rows_of(a.G, a.ldz, a.M, a.N, 2), rows_of(a.U, a.ldz, a.M, a.N, 2),
                        vec(a.bg), vec(a.bu)};
    for (int i = 0; i < 8; ++i) {
        for (int j = 0; j < i; ++j)
            if (rows_meet(out[i], out[j])) return "an output meets another";
        for (const Rows& r : in)
            if (rows_meet(out[i], r)) return "an output meets an input";
    }
    return nullptr;
}

}  // namespace sa3k
